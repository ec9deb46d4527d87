"""The operators of tree-speculative and sampled decoding over a paged cache, as they are measured: each case once in
plain torch (32 bits) and once through the package's own entry points, with the same inputs and the same outputs.

  sample   tokens drawn from rows of logits: temperature, top-k, top-p, min-p, one given uniform number a row
  tree     attention of a tree of drafted tokens over a paged cache: the nodes' rows are appended and attended
           (a tree of one node is the ordinary decode step)
  fork     sequences forked from others (their pages shared), then made writable: shared tail pages are copied
  compact  the rows of a tree's accepted path moved together behind the prefix, in every layer's pages

The definitions that the two forms share:

  sample: l the logits as fp32 (NaN counts as -inf), z = l / temperature, e = exp(z - max z), the weight of a token
  w = floor(e * 2^40) as an integer, so that sums do not depend on their order. Kept are the tokens with l at least the
  k-th largest l (ties stay); of these, in the order of falling l (ties: lowest index first), the tokens whose weight
  sum before them is under ceil(top_p * total); and of these the ones with e >= min_p. The token is the first, in the
  order of the vocabulary, whose running sum of kept weights passes floor(u * kept total). A temperature that is not
  over 0 takes the first largest logit. logp is the token's log-probability among the kept.

  tree: node t of sequence b sits in cache row lens[b] + t, at position lens[b] + depth[b, t]; it sees the rows before
  lens[b] and the nodes whose bit is set in mask[b, t] (32 nodes a word).
"""
import math

import torch

own = False

SCALE = float(1 << 40)


# ---------------------------------------------------------------------------------------------------------- cases

def listed():
  return [
    # one chat stream, the usual settings, the headline model's vocabulary: the smallest call, where latency counts
    dict(name="sample 1x128256", op="sample", rows=1, vocab=128256, dtype="float32", mode="chat"),
    # a serving batch with settings of its own for every request, 152064 words
    dict(name="sample 16x152064 mixed", op="sample", rows=16, vocab=152064, dtype="float32", mode="mixed"),
    # the verify rows of a large batch, nucleus only: no top-k bounds the candidates
    dict(name="sample 256x128256 top-p", op="sample", rows=256, vocab=128256, dtype="float32", mode="nucleus"),
    # an odd vocabulary in 16 bits (GPT-2's), temperature and min-p only
    dict(name="sample 96x50257 f16", op="sample", rows=96, vocab=50257, dtype="float16", mode="min-p"),
    # single tokens, one short sequence (the 8B shape's heads): the smallest call
    dict(name="tree 1x1 at 576", op="tree", batch=1, nodes=1, heads=32, kv_heads=8, dh=128, length=576, page=64, ragged=False),
    # one user's verify step with a tree of 24 nodes, an odd length
    dict(name="tree 1x24 at 4001", op="tree", batch=1, nodes=24, heads=32, kv_heads=8, dh=128, length=4001, page=64, ragged=False),
    # a batch of trees over ragged lengths, the 72B shape's heads (group of 8), small pages
    dict(name="tree 12x16 ragged 8000", op="tree", batch=12, nodes=16, heads=64, kv_heads=8, dh=128, length=8000, page=16, ragged=True),
    # long contexts, 64 drafted nodes each: the largest
    dict(name="tree 8x64 at 32768", op="tree", batch=8, nodes=64, heads=32, kv_heads=8, dh=128, length=32768, page=128, ragged=False),
    # four samples of one prompt: three forks
    dict(name="fork 1 to 4", op="fork", prompts=1, copies=3, layers=32, kv_heads=8, dh=128, length=545, page=64),
    # eight prompts, eight samples each
    dict(name="fork 8 to 64", op="fork", prompts=8, copies=7, layers=32, kv_heads=8, dh=128, length=1077, page=64),
    # one user's accepted path, after each verify step
    dict(name="compact 1x5", op="compact", batch=1, nodes=24, accept=5, layers=32, kv_heads=8, dh=128, length=4001, page=64),
    # a batch's accepted paths, the 72B shape's 80 layers
    dict(name="compact 48x7", op="compact", batch=48, nodes=64, accept=7, layers=80, kv_heads=8, dh=128, length=300, page=32),
  ]


def _log(rng, lo, hi):
  return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
  op = rng.choice(["sample", "sample", "tree", "tree", "tree", "fork", "compact"])
  if op == "sample":
    rows = _log(rng, 1, 256)
    return dict(op=op, rows=rows, vocab=_log(rng, 997, 128256 if rows > 200 else 152064),
                dtype=rng.choice(["float32", "float32", "float16", "bfloat16"]),
                mode=rng.choice(["chat", "mixed", "nucleus", "min-p"]))
  if op == "tree":
    kv_heads = rng.choice([1, 2, 8, 8])
    group = rng.choice([1, 2, 4, 8])
    dh = rng.choice([64, 128, 128])
    nodes = _log(rng, 1, 64)
    length = _log(rng, 1, 32768)
    # the largest listed case reads 8 x 32768 rows for 64 x 4 query rows of each of 8 heads
    most = min(8 * 32768 * 8 // kv_heads, 8 * 32768 * 8 * 256 // (kv_heads * group * nodes))
    batch = _log(rng, 1, max(1, min(64, most // (length + nodes))))
    return dict(op=op, batch=batch, nodes=nodes, heads=kv_heads * group, kv_heads=kv_heads, dh=dh, length=length,
                page=rng.choice([16, 32, 64, 100, 128, 256]), ragged=rng.random() < 0.5)
  if op == "fork":
    prompts = _log(rng, 1, 8)
    return dict(op=op, prompts=prompts, copies=_log(rng, 1, 7), layers=_log(rng, 2, 32), kv_heads=rng.choice([1, 2, 8]),
                dh=rng.choice([64, 128]), length=_log(rng, 1, 1077), page=rng.choice([16, 32, 64, 64]))
  nodes = _log(rng, 2, 64)
  return dict(op=op, batch=_log(rng, 1, 48), nodes=nodes, accept=_log(rng, 1, min(nodes, 7)), layers=_log(rng, 2, 80),
              kv_heads=rng.choice([1, 2, 8]), dh=rng.choice([64, 128]), length=_log(rng, 1, 300), page=rng.choice([16, 32, 64, 100]))


def _lengths(case):
  """Prefix rows of each sequence: all the same, or spread between a sixteenth of the length and all of it."""
  n, B = case["length"], case["batch"]
  if not case.get("ragged"):
    return [n] * B
  return [max(1, n * (1 + (b * 7) % 16) // 16) for b in range(B)]


def _copied_rows(case):
  """Rows that a fork's copies hold in shared tail pages: every sharer but one of each prompt copies its tail."""
  return case["prompts"] * case["copies"] * (case["length"] % case["page"])


def work(case):
  if case["op"] == "sample":
    size = 4 if case["dtype"] == "float32" else 2
    n = case["rows"] * case["vocab"]
    return dict(bytes=n * size + case["rows"] * 28, flops=4 * n)      # scale, subtract, exponential, sum
  if case["op"] == "tree":
    B, T, H, KV, dh = (case[k] for k in ("batch", "nodes", "heads", "kv_heads", "dh"))
    keys = sum(_lengths(case))
    rows = B * T
    return dict(bytes=4 * keys * KV * dh                            # K and V of the prefix, 16 bits each
                + rows * (4 * (H + 2 * KV) * dh                     # qkv in 32 bits
                          + 4 * KV * dh + 2 * H * dh),              # the appended rows, the output
                flops=4 * dh * H * T * (keys + B * (T + 1) // 2))
  row = 2 * 2 * case["layers"] * case["kv_heads"] * case["dh"]      # K and V of one cache row in every layer
  if case["op"] == "fork":
    S = case["prompts"] * (1 + case["copies"])
    return dict(bytes=2 * row * _copied_rows(case) + 16 * S * (case["length"] // case["page"] + 2), flops=0)
  return dict(bytes=2 * row * case["batch"] * case["accept"] + 16 * case["batch"] * case["accept"], flops=0)


# ---------------------------------------------------------------------------------------------------------- inputs

def _gen(seed):
  g = torch.Generator(device="cuda")
  g.manual_seed(seed)
  return g


# settings (temperature, top-k, top-p, min-p) that the rows of a case go through in turn
MODES = {
  "chat": [(0.8, 50, 0.95, 0.0)],
  "nucleus": [(1.0, 0, 0.9, 0.0)],
  "min-p": [(1.1, 0, 1.0, 0.05)],
  "mixed": [(0.7, 40, 0.9, 0.0), (1.0, 0, 0.95, 0.0), (0.0, 0, 1.0, 0.0), (1.3, 0, 1.0, 0.02), (0.9, 1000, 0.99, 0.01),
            (1.0, 0, 1.0, 0.0)],
}


def _prepare_sample(case, seed):
  g = _gen(seed)
  R, V = case["rows"], case["vocab"]
  # a bulk of unlikely words and some that stand out, as a language model's rows have
  l = torch.randn((R, V), generator=g, device="cuda") * 2.0
  hot = torch.randint(0, V, (R, 64), generator=g, device="cuda")
  l.scatter_add_(1, hot, 5.0 + 7.0 * torch.rand((R, 64), generator=g, device="cuda"))
  sets = [MODES[case["mode"]][r % len(MODES[case["mode"]])] for r in range(R)]
  col = lambda k, dt: torch.tensor([s[k] for s in sets], dtype=dt, device="cuda")
  return dict(op="sample", logits=l.to(getattr(torch, case["dtype"])), u=torch.rand((R,), generator=g, device="cuda"),
              temperature=col(0, torch.float32), top_k=col(1, torch.int32), top_p=col(2, torch.float32),
              min_p=col(3, torch.float32))


def _tables(g, B, pages_each, extra):
  """A table of distinct random pages for each of B sequences, and the page count."""
  n = B * pages_each + extra
  perm = torch.randperm(n, generator=g, device="cuda").to(torch.int32)
  return perm[:B * pages_each].view(B, pages_each).contiguous(), n


def _prepare_tree(case, seed):
  g = _gen(seed)
  B, T, H, KV, dh, page = (case[k] for k in ("batch", "nodes", "heads", "kv_heads", "dh", "page"))
  lens = _lengths(case)
  W = -(-(max(lens) + T) // page)
  table, P = _tables(g, B, W, 1)
  half = lambda *s: torch.randn(s, generator=g, device="cuda", dtype=torch.float16)
  # each node hangs on one of the few before it; a node's ancestors are the powers of that relation
  node = torch.arange(T, device="cuda")
  parent = node - torch.minimum(torch.randint(1, 7, (B, T), generator=g, device="cuda"), node)
  anc = torch.eye(T, device="cuda") + (parent[:, :, None] == node) * (node > 0)[:, None]
  anc = torch.matrix_power(anc, max(1, T - 1)) > 0
  bits = torch.zeros((B, T, -(-T // 32) * 32), dtype=torch.int64, device="cuda")
  bits[:, :, :T] = anc
  m = (bits.view(B, T, -1, 32) << torch.arange(32, device="cuda")).sum(-1)
  mask = torch.where(m >= 1 << 31, m - (1 << 32), m).to(torch.int32)
  depth = (anc.sum(-1) - 1).to(torch.int32)
  M = W * page
  ang = torch.outer(torch.arange(M, dtype=torch.float64, device="cuda"),
                    500000.0 ** (-torch.arange(0, dh, 2, dtype=torch.float64, device="cuda") / dh))
  return dict(op="tree", H=H, KV=KV, dh=dh, T=T, scale=dh ** -0.5,
              qkv=torch.randn((B * T, (H + 2 * KV) * dh), generator=g, device="cuda"),
              kc=half(P, KV, page, dh), vc=half(P, KV, page, dh), table=table,
              lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
              depth=depth, mask=mask,
              cos=torch.cat([ang.cos(), ang.cos()], 1).half(), sin=torch.cat([ang.sin(), ang.sin()], 1).half())


def _pool(g, layers, P, KV, page, dh):
  return torch.empty((layers, 2, P, KV, page, dh), dtype=torch.float16, device="cuda").normal_(generator=g)


def _prepare_fork(case, seed):
  g = _gen(seed)
  n, c, page, length = case["prompts"], case["copies"], case["page"], case["length"]
  S, used = n * (1 + c), -(-length // page)
  W = -(-(length + 1) // page) + 1
  # pages for every prompt, and for every sequence a copied tail and the next page
  P = n * used + 2 * S
  perm = torch.randperm(P, generator=g, device="cuda").to(torch.int32)
  table = torch.full((S, W), -1, dtype=torch.int32, device="cuda")
  table[:n, :used] = perm[:n * used].view(n, used)
  refs = torch.zeros((P,), dtype=torch.int32, device="cuda")
  refs[perm[:n * used].long()] = 1
  lens = torch.zeros((S,), dtype=torch.int32, device="cuda")
  lens[:n] = length
  src = torch.arange(n, dtype=torch.int32, device="cuda").repeat_interleave(c)
  dst = torch.arange(n, S, dtype=torch.int32, device="cuda")
  return dict(op="fork", pool=_pool(g, case["layers"], P, case["kv_heads"], page, case["dh"]), table=table, refs=refs,
              lens=lens, src=src, dst=dst, slots=torch.arange(S, dtype=torch.int32, device="cuda"),
              rows=torch.ones((S,), dtype=torch.int32, device="cuda"), err=torch.zeros((1,), dtype=torch.int32, device="cuda"))


def _prepare_compact(case, seed):
  g = _gen(seed)
  B, T, D, page = case["batch"], case["nodes"], case["accept"], case["page"]
  W = -(-(case["length"] + T) // page)
  table, P = _tables(g, B, W, 0)
  # the accepted nodes of each tree, parents before children; the root is always node 0
  path = torch.sort(torch.rand((B, T - 1), generator=g, device="cuda").argsort(1)[:, :D - 1] + 1, 1).values
  path = torch.cat([torch.zeros((B, 1), dtype=path.dtype, device="cuda"), path], 1)
  n = 1 + torch.randint(0, D, (B,), generator=g, device="cuda")
  n[0] = D
  return dict(op="compact", pool=_pool(g, case["layers"], P, case["kv_heads"], page, case["dh"]), table=table,
              lens=torch.full((B,), case["length"], dtype=torch.int32, device="cuda"),
              slots=torch.arange(B, dtype=torch.int32, device="cuda"), path=path.to(torch.int32).contiguous(),
              n=n.to(torch.int32), lens_out=torch.zeros((B,), dtype=torch.int32, device="cuda"),
              err=torch.zeros((1,), dtype=torch.int32, device="cuda"))


def prepare(case, seed):
  return {"sample": _prepare_sample, "tree": _prepare_tree, "fork": _prepare_fork, "compact": _prepare_compact}[case["op"]](case, seed)


# ---------------------------------------------------------------------------------------------------------- plain forms

def _plain_sample(s):
  l = s["logits"].float()
  l = torch.where(torch.isnan(l), -math.inf, l)
  V = l.shape[1]
  ok = s["temperature"] > 0
  temp = torch.where(ok, s["temperature"], 1.0)[:, None]
  lmax, first = l.max(1, keepdim=True).values, (l == l.max(1, keepdim=True).values).to(torch.int32).argmax(1)
  z, zmax = l / temp, lmax / temp
  e = torch.where(l == lmax, 1.0, torch.exp(z - zmax))
  w = (e * SCALE).to(torch.int64)
  by, order = torch.sort(l, dim=1, descending=True, stable=True)
  k = torch.where((s["top_k"] > 0) & (s["top_k"] < V), s["top_k"], V).long()
  in_k = by >= by.gather(1, k[:, None] - 1)
  ws = torch.where(in_k, w.gather(1, order), 0)
  before = ws.cumsum(1) - ws
  total = ws.sum(1)
  limit = torch.ceil(s["top_p"].double() * total.double()).to(torch.int64)
  nucleus = (s["top_p"] > 0) & (s["top_p"] < 1)
  in_p = torch.where(nucleus[:, None], before < limit[:, None], True)
  kept = torch.zeros_like(in_k).scatter(1, order, in_k & in_p) & (e >= s["min_p"].clamp(max=1.0)[:, None])
  wk = torch.where(kept, w, 0)
  run_sum = wk.cumsum(1)
  total = run_sum[:, -1]
  t = torch.floor(s["u"].double() * total.double()).to(torch.int64)
  t = torch.minimum(t.clamp(min=0), total - 1)
  tok = (run_sum <= t[:, None]).sum(1).clamp(max=V - 1)
  logp = (z.gather(1, tok[:, None]) - zmax)[:, 0] - torch.log(total.float() / SCALE)
  tok, logp = torch.where(ok, tok, first), torch.where(ok, logp, 0.0)
  none = lmax[:, 0] == -math.inf
  return torch.where(none, -1, tok).to(torch.int32), torch.where(none, -math.inf, logp)


def _turn(x, cos, sin):
  """Rotary position of head vectors [..., heads, dh] with factors [..., 1, dh]."""
  h = x.shape[-1] // 2
  return x * cos + torch.cat([-x[..., h:], x[..., :h]], -1) * sin


def _plain_tree(s):
  H, KV, dh, T, table = s["H"], s["KV"], s["dh"], s["T"], s["table"].long()
  B, W = table.shape
  page = s["kc"].shape[2]
  N, G = W * page, H // KV
  qkv = s["qkv"].float().view(B, T, H + 2 * KV, dh)
  row = s["lens"].long()[:, None] + torch.arange(T, device="cuda")
  at = s["lens"].long()[:, None] + s["depth"].long()
  cos, sin = s["cos"][at].float()[:, :, None], s["sin"][at].float()[:, :, None]
  q = _turn(qkv[:, :, :H], cos, sin).half().float()
  where = table.gather(1, row // page)
  s["kc"][where, :, row % page] = _turn(qkv[:, :, H:H + KV], cos, sin).half()
  s["vc"][where, :, row % page] = qkv[:, :, H + KV:].half()
  k = s["kc"][table].permute(0, 2, 1, 3, 4).reshape(B, KV, N, dh).float()
  v = s["vc"][table].permute(0, 2, 1, 3, 4).reshape(B, KV, N, dh).float()
  q = q.view(B, T, KV, G, dh).permute(0, 2, 3, 1, 4).reshape(B, KV, G * T, dh)
  j = torch.arange(N, device="cuda") - s["lens"].long()[:, None]                    # node number of each row, < 0: prefix
  c = j.clamp(0, T - 1)
  words = s["mask"].long().gather(2, (c // 32)[:, None, :].expand(B, T, N))
  sees = torch.where((j >= 0)[:, None], ((words >> (c % 32)[:, None]) & 1).bool() & (j < T)[:, None], True)
  sc = (q @ k.transpose(2, 3)).view(B, KV, G, T, N) * s["scale"]
  sc = torch.where(sees[:, None, None], sc, -math.inf)
  e = torch.exp(sc - sc.amax(-1, keepdim=True).clamp(min=-3.0e38))
  o = (e.view(B, KV, G * T, N) @ v) / e.sum(-1).view(B, KV, G * T, 1).clamp(min=1e-30)
  o = o.view(B, KV, G, T, dh).permute(0, 3, 1, 2, 4).reshape(B * T, H * dh)
  return o.half(), s["kc"], s["vc"]


def _plain_fork(s):
  pool, table, refs, lens, src, dst = (s[k] for k in ("pool", "table", "refs", "lens", "src", "dst"))
  src, dst, slots = src.long(), dst.long(), s["slots"].long()
  S, W = table.shape
  P, page = pool.shape[2], pool.shape[4]
  count = lambda t, sign: refs.index_add_(0, t.clamp(min=0).view(-1).long(), torch.where(t >= 0, sign, 0).to(torch.int32).view(-1))
  # what the forked slots held goes back; then they share the pages their source fills
  count(table[dst], -1)
  full = (lens[src] + page - 1) // page
  shared = torch.where(torch.arange(W, device="cuda") < full[:, None], table[src], -1)
  table[dst] = shared
  lens[dst] = lens[src]
  count(shared, 1)
  # writable rows [len, len + rows): of the sharers of a tail page all but the last listed take a copy
  ln, need = lens[slots], s["rows"][:, None]
  tail = torch.where(ln % page != 0, table[slots].gather(1, (ln // page).clamp(max=W - 1).long()[:, None])[:, 0], -1)
  same = (tail[:, None] == tail[None, :]) & (tail >= 0)[:, None]
  rank = torch.tril(same, -1).sum(1)
  copies = (tail >= 0) & (refs[tail.clamp(min=0).long()] - rank > 1)
  col = torch.arange(W, device="cuda")
  wanted = (col >= (ln // page)[:, None]) & (col < ((ln[:, None] + need + page - 1) // page))
  fresh = wanted & ((table[slots] < 0) | (copies[:, None] & (col == (ln // page)[:, None])))
  order = torch.argsort((refs != 0).to(torch.int32), stable=True)                     # free pages first, lowest first
  number = fresh.view(-1).long().cumsum(0).view(S, W) - 1
  given = torch.where(fresh, order[number.clamp(0, P - 1)].to(torch.int32), table[slots])
  count(torch.where(copies, tail, -1), -1)
  count(torch.where(fresh, given, -1), 1)
  table[slots] = given
  new = given.gather(1, (ln // page).clamp(max=W - 1).long()[:, None])[:, 0]
  old, new, fill = tail[copies].long(), new[copies].long(), (ln % page)[copies]
  rows = (torch.arange(page, device="cuda") < fill[:, None])[None, None, :, None, :, None]
  pool[:, :, new] = torch.where(rows, pool[:, :, old], pool[:, :, new])
  return table, lens, refs, pool


def _plain_compact(s):
  pool, table, lens = s["pool"], s["table"].long(), s["lens"].long()
  page, D = pool.shape[4], s["path"].shape[1]
  slots = s["slots"].long()
  j = torch.arange(D, device="cuda")
  live = j < s["n"].long()[:, None]
  a = (lens[slots][:, None] + s["path"].long())[live]
  b = (lens[slots][:, None] + j)[live]
  who = slots[:, None].expand(-1, D)[live]
  moved = pool[:, :, table[who, a // page], :, a % page]
  pool[:, :, table[who, b // page], :, b % page] = moved
  s["lens_out"].copy_(s["lens"])
  s["lens_out"][slots] = (lens[slots] + s["n"]).to(torch.int32)
  return s["lens_out"], pool


# ---------------------------------------------------------------------------------------------------------- the package

def _own(s):
  from aneforge_b200 import kernels as K
  if s["op"] == "sample":
    return K.sample(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
  if s["op"] == "tree":
    if "scratch" not in s:                                   # a program keeps its workspace
      s["scratch"] = K.attn_tree_scratch(s["table"].shape[0], s["T"], s["H"], s["KV"], s["dh"], device=s["qkv"].device)
    out = K.attn_tree(s["qkv"], s["kc"], s["vc"], s["table"], s["lens"], s["cos"], s["sin"], s["H"], s["KV"], s["dh"],
                      s["scale"], mask=s["mask"], depth=s["depth"], scratch=s["scratch"])
    return out, s["kc"], s["vc"]
  if s["op"] == "fork":
    K.kv_fork(s["table"], s["lens"], s["refs"], s["src"], s["dst"], s["pool"].shape[4], err=s["err"])
    K.kv_reserve(s["pool"], s["table"], s["lens"], s["refs"], s["slots"], s["rows"], err=s["err"])
    return s["table"], s["lens"], s["refs"], s["pool"]
  K.kv_compact(s["pool"], s["table"], s["lens"], s["slots"], s["path"], s["n"], lens_out=s["lens_out"], err=s["err"])
  return s["lens_out"], s["pool"]


def run(state):
  if own:
    return _own(state)
  return {"sample": _plain_sample, "tree": _plain_tree, "fork": _plain_fork, "compact": _plain_compact}[state["op"]](state)


# ---------------------------------------------------------------------------------------------------------- 64 bits

def exact(case, seed):
  def sample(s):
    """Row by row, straight from the definition: sorted candidates, their weights in 64 bits."""
    logps = []
    for r in range(s["logits"].shape[0]):
      l, temp, u = s["logits"][r].double(), float(s["temperature"][r]), float(s["u"][r])
      if not temp > 0:
        logps.append(0.0)
        continue
      p = torch.softmax(l / temp, 0)
      k, top_p, min_p = int(s["top_k"][r]), float(s["top_p"][r]), float(s["min_p"][r])
      alive = torch.ones_like(p, dtype=torch.bool)
      if 0 < k < p.numel():
        alive &= l >= torch.topk(l, k).values[-1]
      if 0 < top_p < 1:
        desc = torch.argsort(torch.where(alive, l, -math.inf), descending=True, stable=True)
        mass = torch.where(alive, p, 0.0)[desc]
        mass = mass / mass.sum()
        alive &= torch.zeros_like(alive).scatter(0, desc, mass.cumsum(0) - mass < top_p)
      alive &= p >= min_p * p.max()
      mass = torch.where(alive, p, 0.0)
      mass = mass / mass.sum()
      tok = int(torch.searchsorted(mass.cumsum(0), torch.tensor([u], dtype=torch.float64, device="cuda"), right=True))
      logps.append(math.log(float(mass[min(tok, p.numel() - 1)])))
    return None, torch.tensor(logps, dtype=torch.float64, device="cuda")

  def tree(s):
    H, KV, dh, T = s["H"], s["KV"], s["dh"], s["T"]
    page, G, B = s["kc"].shape[2], H // KV, s["table"].shape[0]
    kc, vc, out = s["kc"].double(), s["vc"].double(), []
    lens, table, words = s["lens"].tolist(), s["table"].tolist(), s["mask"].tolist()
    half = dh // 2
    for b in range(B):
      n = lens[b]
      x = s["qkv"][b * T:(b + 1) * T].double().view(T, H + 2 * KV, dh)
      at = n + s["depth"][b].long()
      cos, sin = s["cos"][at].double()[:, None], s["sin"][at].double()[:, None]
      rot = x * cos + torch.stack([-x[..., half:], x[..., :half]], -2).flatten(-2) * sin
      for t in range(T):
        p, r = table[b][(n + t) // page], (n + t) % page
        kc[p, :, r], vc[p, :, r] = rot[t, H:H + KV], x[t, H + KV:]
      rows = torch.arange(n + T, device="cuda")
      pg = s["table"][b].long()[rows // page]
      sees = torch.ones((T, n + T), dtype=torch.bool)
      sees[:, n:] = torch.tensor([[bool(words[b][t][j // 32] >> (j % 32) & 1) for j in range(T)] for t in range(T)])
      sees = sees.cuda()
      res = []
      for h in range(KV):
        K, V = kc[pg, h, rows % page], vc[pg, h, rows % page]
        for g in range(G):
          sc = rot[:, h * G + g] @ K.T * s["scale"]
          res.append(torch.softmax(sc.masked_fill(~sees, -math.inf), 1) @ V)
      out.append(torch.stack(res, 1).reshape(T, H * dh))
    return torch.cat(out), kc, vc

  if case["op"] == "sample":
    return sample(prepare(case, seed))
  if case["op"] == "tree":
    return tree(prepare(case, seed))
  return None                                               # rows and page numbers are moved, not computed
