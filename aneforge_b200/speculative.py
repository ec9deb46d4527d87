"""Greedy speculative decoding on the device (the reference's `aneforge/speculative.py:131-165`,
`spec_generate`): a small draft model proposes `n_draft` tokens, the target checks all of them in
ONE multi-token verify step over its resident cache, and the matching prefix plus one corrected (or
bonus) token are emitted. Greedy speculative decoding is exact: it emits the target's greedy tokens.

B200 form:
  * the draft's proposals are `n_draft` back-to-back replays of its decode program with the token
    fed back on the device (no host round trip between them), read once from its token history;
  * the target's verify is the decode step over Kq = n_draft + 1 rows that are consecutive tokens of
    one sequence sharing one cache (`LlamaPrefill._verifier`): each row appends its K / V first and
    attends up to its own position, the head's greedy argmax gives the target's token after each;
  * both caches are seeded by their batched prefill; rejected draft positions are overwritten in the
    next round (the reference's incremental scheme), the target's too (the next verify rewrites from
    the first unconfirmed position on before any row reads it).
"""
from __future__ import annotations

import numpy as np

import torch

from .llm import LlamaPrefill


def _argmax_rows(target: LlamaPrefill, ver) -> list:
  """The target's greedy token after each verify row: the device argmax when the head is exactly fp16
  (it then equals the host fp32 head's argmax), else the host logits with the reference's tie-margin
  recheck on each row."""
  prog = ver["prog"]
  if target._head_exact:
    return [int(t) for t in prog.read_output("tok_out")]
  hid = prog.read_output("hid")
  return [int(np.argmax(target._decode_logits(h, None, True))) for h in hid]


def spec_generate(target: LlamaPrefill, draft: LlamaPrefill, token_ids, max_new_tokens=40, eos_id=None,
                  max_len=None, n_draft=4, on_token=None, stats: dict | None = None):
  """Greedy speculative decoding (reference signature): the same tokens as `target.generate(...)`,
  with the target run once per accepted run of draft tokens. `stats`, when given, receives the
  number of verify steps and of accepted draft tokens."""
  prompt = [int(t) for t in token_ids]
  target._check_ids(prompt)
  P = len(prompt)
  M = int(max_len or P + max_new_tokens)
  Kq = int(n_draft) + 1
  eos = {int(eos_id)} if isinstance(eos_id, int) else {int(e) for e in (eos_id or ())}
  ver = target._verifier(M, Kq)
  dec = draft._decoder(M, 1)
  vprog, dprog = ver["prog"], dec["prog"]
  with torch.cuda.device(target.device):
    torch.cuda.synchronize()
    target._reset_state(ver)
  with torch.cuda.device(draft.device):
    draft._reset_state(dec)
  # both caches from their batched prefills; the first token is the target's greedy choice
  pre, real, _ = target._prefill_hidden(prompt)
  hid = pre["prog"].read_output("hid")
  cur = int(np.argmax(target._decode_logits(hid[real - 1], None, True)))
  with torch.cuda.device(target.device):
    target._seed_cache(ver, pre, real)
    torch.cuda.synchronize()
  dpre, dreal, _ = draft._prefill_hidden(prompt)
  with torch.cuda.device(draft.device):
    draft._seed_cache(dec, dpre, dreal)
    torch.cuda.synchronize()
  out = [cur]
  n_verify = n_accept = 0
  if cur in eos:
    return out
  if on_token is not None:
    on_token(cur)
  p = P                                                       # position of `cur`
  while len(out) < max_new_tokens and p + Kq < M:
    # the draft proposes n_draft tokens from cur (device-resident feedback)
    dprog.set_input("tok", np.array([cur], np.int32))
    dprog.set_input("pos", np.array([p], np.int32))
    for _ in range(n_draft):
      dprog.execute_async()
    dprog.sync()
    drafts = [int(t) for t in dprog.read_output("hist")[0][p:p + n_draft]]
    # one verify step over cur + drafts at positions p .. p + n_draft
    vprog.set_input("tok", np.array([cur] + drafts, np.int32))
    vprog.set_input("pos", np.arange(p, p + Kq, dtype=np.int32))
    vprog.execute()
    n_verify += 1
    g = _argmax_rows(target, ver)
    a = 0
    while a < n_draft and g[a] == drafts[a]:
      a += 1
    n_accept += a
    if a == n_draft:
      # every draft accepted: give the draft's cache the last proposal too (row p + n_draft)
      dprog.set_input("tok", np.array([drafts[-1]], np.int32))
      dprog.set_input("pos", np.array([p + n_draft], np.int32))
      dprog.execute()
    emit = drafts[:a] + [g[a]]
    for t in emit:
      if len(out) >= max_new_tokens:
        break
      out.append(t)
      if t in eos:
        break
      if on_token is not None:
        on_token(t)
    if out[-1] in eos:
      break
    cur, p = emit[-1], p + a + 1
  if stats is not None:
    stats.update(verify_steps=n_verify, accepted=n_accept)
  return out[:max_new_tokens]


def tree_parents(branches):
  """Parents of a tree with a root and branches[d] children of every node of level d, level by level."""
  parents, level = [-1], [0]
  for b in branches:
    if int(b) < 1:
      raise ValueError("branches must be positive")
    parents += [p for p in level for _ in range(int(b))]
    level = list(range(len(parents) - len(level) * int(b), len(parents)))
  return parents


def tree_generate(target: LlamaPrefill, draft: LlamaPrefill, token_ids, max_new_tokens=40, eos_id=None, branches=(3, 2, 1),
                  temperature=0.0, top_p=1.0, top_k=0, min_p=0.0, seed=None, page=64, on_token=None,
                  stats: dict | None = None):
  """Speculative decoding with a drafted tree: every round the draft proposes its branches[d] best tokens after
  each node of level d, the target runs the last token and the whole tree in one step and draws its own token
  after every node, the matching path is kept in both caches and its tokens and one more are emitted. The head's
  logits are the device's. A model with a learned position table needs len(branches) positions past the last token.
  `stats` gets the number of target steps and of accepted draft tokens."""
  from .paged import PagedKV, TreeStep, _stops
  prompt = [int(t) for t in token_ids]
  target._check_ids(prompt)
  parents = tree_parents(branches)
  T, depth = len(parents), len(branches)
  if T > 256:
    raise ValueError("a tree has at most 256 nodes")
  if draft.device != target.device or draft.cfg.vocab != target.cfg.vocab:
    raise ValueError("draft and target must share a vocabulary and a device")
  if not prompt or max_new_tokens < 1:
    return []
  eos, P = _stops(eos_id), len(prompt)
  children = [[] for _ in parents]
  for t, p in enumerate(parents):
    if p >= 0:
      children[p].append(t)
  rows = P + max_new_tokens + T
  dev = torch.device("cuda", target.device)
  rng = np.random.default_rng(seed)
  kvt, kvd = (PagedKV(m.cfg, 1, rows, page=page, device=m.device) for m in (target, draft))
  last = P + max_new_tokens + depth                          # positions of drafted nodes stay below
  big = TreeStep(target, kvt, 1, parents, last, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
  small = None
  try:
    small = TreeStep(draft, kvd, 1, parents, last)
    logits = None
    for model, kv, step in ((draft, kvd, small), (target, kvt, big)):
      pre, real, _ = model._prefill_hidden(prompt)
      with torch.cuda.stream(step.stream):
        kv.seed(0, pre, real)
      if model is target:
        logits = model._logits(pre["prog"].read_output("hid")[real - 1])
      torch.cuda.synchronize(dev)
    from . import kernels
    with torch.cuda.stream(big.stream):
      first, _ = kernels.sample(torch.from_numpy(np.ascontiguousarray(logits, np.float32)).to(dev)[None],
                                torch.from_numpy(rng.random(1, np.float32)).to(dev), temperature, top_k, top_p, min_p)
      cur = int(first[0])
    out, n_steps, n_accept = [cur], 0, 0
    if on_token is not None and cur not in eos:
      on_token(cur)
    slot, grow = (torch.tensor([v], dtype=torch.int32, device=dev) for v in (0, T))
    path_host = np.zeros((1, depth + 1), np.int32)
    while len(out) < max_new_tokens and out[-1] not in eos:
      with torch.cuda.stream(small.stream):
        # level by level: the draft runs the nodes that it has, the best tokens after the last level's are the next
        kvd.reserve(slot, grow)
        small.tok[0, 0] = cur
        lo, hi = 0, 1
        for b in branches:
          small.nodes.fill_(hi)
          small.run()
          best = small.logits[0, lo:hi].topk(int(b), dim=1).indices
          lo, hi = hi, hi + best.numel()
          small.tok[0, lo:hi] = best.reshape(-1).to(torch.int32)
      with torch.cuda.stream(big.stream):
        big.stream.wait_stream(small.stream)
        kvt.reserve(slot, grow)
        big.tok.copy_(small.tok)
        big.u.copy_(torch.from_numpy(rng.random((1, T), np.float32)))
        big.run()
        toks, drawn = torch.stack((big.tok[0], big.out[0])).tolist()
      n_steps += 1
      path = [0]
      while True:
        nxt = next((c for c in children[path[-1]] if toks[c] == drawn[path[-1]]), None)
        if nxt is None:
          break
        path.append(nxt)
      n_accept += len(path) - 1
      path_host[0, :len(path)] = path
      with torch.cuda.stream(small.stream):
        if len(path) == depth + 1:                           # a leaf: its row is not in the draft's cache yet
          small.nodes.fill_(T)
          small.run()
        kvd.compact(slot, torch.from_numpy(path_host).to(dev), [len(path)])
      with torch.cuda.stream(big.stream):
        kvt.compact(slot, torch.from_numpy(path_host).to(dev), [len(path)])
      for t in (drawn[p] for p in path):
        out.append(t)
        if t in eos:
          break
        if on_token is not None:
          on_token(t)
        if len(out) >= max_new_tokens:
          break
      cur = out[-1]
    small.check()
    big.check()
  finally:
    big.release()
    if small is not None:
      small.release()
  if stats is not None:
    stats.update(verify_steps=n_steps, accepted=n_accept)
  return out
