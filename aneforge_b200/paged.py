"""Sequences whose key / value rows lie in pages of one pool, and the model step that decodes them.

The runner's own decode program keeps one cache block per sequence. Here the rows of all sequences lie in
pages of one pool, a sequence is a row of the page table, and so
  * many samples of one prompt share the prompt's pages (`PagedKV.fork`; a shared page is copied when a
    sequence comes to append to it) - `sample_generate`;
  * a step may carry a tree of drafted tokens per sequence: every node attends to the prefix and to its own
    ancestors, and the accepted path is moved behind the prefix (`PagedKV.compact`) -
    `aneforge_b200.speculative.tree_generate`;
  * the next token of every row is drawn on the device (temperature, top-k, top-p, min-p).

`TreeStep` is the step as one program: embedding -> layers with tree attention over the pages -> head ->
sampling. A plain decode step is a tree of one node. The table and the lengths stay on the device: a
generation loop only launches, and reads its tokens when it wants them.
"""
from __future__ import annotations

import numpy as np

import torch

from . import _runtime as R
from . import kernels
from .llm import (DECODE_MIXERS, DECODE_MLPS, PREFILL_MLPS, LlamaPrefill, _emit_embedding, _emit_final_norm, is_graph_builder,
                  plan_gemv_chains, plan_l2_prefetch, rope_tables)
from .plan import PlanBuilder


class PagedKV:
  """`slots` sequences of at most `max_len` cache rows in `pages` pages of `page` rows each (default: enough for
  every slot to be full), for a model of cfg.n_layers layers. pool [L, 2, pages, KV, page, dh] fp16, table
  [slots, width] int32 (-1: no page), lens [slots], refs [pages]: all on the device, changed by kernels in the
  order of the current stream. Slots and counts are lists or int32 tensors on the device. Take a `page` of a multiple
  of 8 rows, best 64 or 128: with others (and with head dims 16 and 32) attention runs without the tensor cores and
  takes ten times as long and more."""

  def __init__(self, cfg, slots: int, max_len: int, pages: int | None = None, page: int = 64, device: int = 0):
    self.slots, self.page = int(slots), int(page)
    if self.slots < 1 or self.page < 1 or max_len < 1:
      raise ValueError("slots, page and max_len must be positive")
    self.width = -(-int(max_len) // self.page)
    self.pages = int(pages) if pages is not None else self.slots * self.width
    if self.pages < 1:
      raise ValueError("a cache needs a page")
    self.device = torch.device("cuda", int(device))
    i32 = dict(dtype=torch.int32, device=self.device)
    self.pool = torch.zeros((cfg.n_layers, 2, self.pages, cfg.n_kv_heads, self.page, cfg.dh), dtype=torch.float16,
                            device=self.device)
    self.table = torch.full((self.slots, self.width), -1, **i32)
    self.lens = torch.zeros((self.slots,), **i32)
    self.refs = torch.zeros((self.pages,), **i32)
    self.err = torch.zeros((1,), **i32)
    self._lens_next = torch.zeros_like(self.lens)

  def _i32(self, x):
    if isinstance(x, torch.Tensor):
      return x
    return torch.tensor([int(v) for v in x], dtype=torch.int32, device=self.device)

  def fork(self, src, dst) -> None:
    """Slots `dst` become copies of slots `src` (their pages are shared until one of them appends)."""
    kernels.kv_fork(self.table, self.lens, self.refs, self._i32(src), self._i32(dst), self.page, err=self.err)

  def reserve(self, slots, rows) -> None:
    """Gives each slot pages of its own for `rows` more rows (a step writes them; lens is left as it is)."""
    kernels.kv_reserve(self.pool, self.table, self.lens, self.refs, self._i32(slots), self._i32(rows), err=self.err)

  def compact(self, slots, path, n_path) -> None:
    """Keeps the accepted path of each slot's last tree: node numbers path [n, D], the first n_path of each."""
    kernels.kv_compact(self.pool, self.table, self.lens, self._i32(slots), path, self._i32(n_path),
                       lens_out=self._lens_next, err=self.err)
    self.lens.copy_(self._lens_next)

  def free(self, slots, keep=None) -> None:
    """Gives back the pages past `keep` rows of each slot (default: all of them)."""
    kernels.kv_free(self.table, self.lens, self.refs, self._i32(slots), self.page, None if keep is None else self._i32(keep),
                    err=self.err)

  def check(self) -> None:
    """Raises if a call since the last check found no free pages, or a slot or path that cannot be."""
    code = int(self.err.item())
    if code:
      self.err.zero_()
      what = {4: "cache pages exhausted", 5: "bad cache slot or path"}.get(code, f"error {code}")
      raise RuntimeError(f"paged cache: {what}")

  def seed(self, slot: int, pre, real: int) -> None:
    """An empty slot gets the first `real` rows of a batched prefill (`LlamaPrefill._prefill_hidden`), device to
    device."""
    L, _, _, KV, page, dh = self.pool.shape
    self.free([slot])
    self.reserve([slot], [real])
    self.check()
    full, rest = divmod(real, page)
    pages = self.table[slot, :full + (rest > 0)].long()
    for li in range(L):
      for i, nm in enumerate(("K", "V")):
        src = pre["prog"].tensor(f"L{li}.{nm}", (KV, pre["seq"], dh))
        if full:
          self.pool[li, i].index_copy_(0, pages[:full], src[:, :full * page].view(KV, full, page, dh).transpose(0, 1).contiguous())
        if rest:
          self.pool[li, i, pages[full], :, :rest] = src[:, full * page:real]
    self.lens[slot] = real


class TreeStep:
  """One step of `model` over slots [0, B) of `kv`, a tree of T tokens each (`parents`, see
  `kernels.tree_layout`; None: T = 1, the plain decode step), as a program on a stream of its own.

  The caller fills `tok` [B, T] and `u` [B, T] (and the settings temperature, top_k, top_p, min_p, each [B, T]),
  reserves T rows in `kv`, and calls `run()` - all in the order of `stream`. Positions go up to `max_pos` (default:
  what the cache holds). The step writes the nodes' K and V,
  and gives `out` [B, T] (the token drawn after each node), `logp` and `logits` [B, T, V]. `nodes` [B] may be
  lowered to run the first nodes of the tree only. With feed=True (T = 1) `out` is `tok`: each step's token is
  the next one's input."""

  def __init__(self, model: LlamaPrefill, kv: PagedKV, B: int, parents=None, max_pos: int | None = None,
               temperature: float = 0.0, top_k: int = 0, top_p: float = 1.0, min_p: float = 0.0, feed: bool = False):
    cfg, d = model.cfg, model._load()
    parents = [-1] if parents is None else [int(p) for p in parents]
    B, T = int(B), len(parents)
    if not 1 <= B <= kv.slots:
      raise ValueError(f"the cache has {kv.slots} slots")
    if feed and T != 1:
      raise ValueError("feed=True needs a tree of one node")
    if model.tp is not None or any(
        model._spec(i).mixer != "attention" or is_graph_builder(DECODE_MIXERS["attention"]) for i in range(cfg.n_layers)):
      raise NotImplementedError("the paged step needs the fused attention mixer on one GPU")
    if kv.device.index != model.device or tuple(kv.pool.shape[i] for i in (0, 3, 5)) != (cfg.n_layers, cfg.n_kv_heads, cfg.dh):
      raise ValueError("the cache is for another model or device")
    # the GQA expansion factor of int8 / int4 models rounds back to the same fp16 value for every normal number
    # as long as it is within a quarter of a unit in the last place of 1
    if abs(d["kvc"] - 1.0) >= 2.0 ** -12:
      raise NotImplementedError("a GQA expansion factor this far from 1")
    rows = int(max_pos or kv.width * kv.page)
    model._check_positions(rows)
    self.model, self.kv, self.B, self.T = model, kv, B, T
    depth, mask = kernels.tree_layout(parents)
    n, D, H, KV, dh, V = B * T, cfg.dim, cfg.n_heads, cfg.n_kv_heads, cfg.dh, cfg.vocab
    ctx = model._ctx(n, rows)
    ctx["tree"] = dict(b=B, t=T, p=kv.pages, page=kv.page, w=kv.width, rows=rows)
    pb = PlanBuilder()
    for name in ("tok", "topk", "pos", "depth"):
      pb.buf(name, 4 * n, "state")
    for name in ("u", "temp", "topp", "minp"):
      pb.buf(name, 4 * n, "state")
    pb.buf("nodes", 4 * B, "state"); pb.buf("mask", 4 * n * ((T + 31) // 32), "state")
    pb.buf("tok_out", 4 * n, "out"); pb.buf("logp", 4 * n, "out")
    pb.buf("hid", 2 * n * D, "out"); pb.buf("logits", 4 * n * V, "out")
    pb.buf("h", 4 * n * D, "tmp"); pb.buf("xn", 2 * n * D, "tmp"); pb.buf("qkv", 4 * n * (H + 2 * KV) * dh, "tmp")
    pb.buf("att", 2 * n * H * dh, "tmp")
    F = max([l["gu"].N // 2 for l in d["layers"] if "gu" in l] + [l["experts"].F for l in d["layers"] if "experts" in l]
            + [l["shgu"].N // 2 for l in d["layers"] if "shgu" in l] + [1])
    pb.buf("act", 2 * n * F, "tmp")
    pb.buf("tree.scr", max(1, R.load_library().af_attn_tree_scratch_bytes(B, T, H, KV, dh)), "scratch")
    pb.buf("embed", 2 * V * D, "weight"); pb.buf("lm_head", 2 * V * D, "weight"); pb.buf("final_g", 2 * D, "weight")
    if cfg.norm_type == "layer":
      pb.buf("final_b", 2 * D, "weight")
    if cfg.rope:
      pb.buf("rope.cos", 2 * rows * dh, "weight"); pb.buf("rope.sin", 2 * rows * dh, "weight")
    pb.buf("kv.table", 4 * B * kv.width, "ext"); pb.buf("kv.lens", 4 * B, "ext")
    plane = kv.pool[0, 0].numel() * 2
    for li in range(cfg.n_layers):
      model._declare_layer_weights(pb, li, d["layers"][li])
    self._planes = {f"L{li}.{nm}": kv.pool[li, i] for li in range(cfg.n_layers) for i, nm in enumerate(("K", "V"))}
    for name in self._planes:
      pb.buf(name, plane, "ext")
    self._learned_pos = "wpe" in d
    _emit_embedding(pb, cfg, d, n, "pos")
    lows = []
    for li in range(cfg.n_layers):
      ls = model._spec(li)
      DECODE_MIXERS[ls.mixer](pb, ctx, li, d["layers"][li], cfg, ls)
      mlp = DECODE_MLPS[ls.mlp]
      if is_graph_builder(mlp):
        model._lower_graph_mlp(pb, li, PREFILL_MLPS.get(ls.mlp, mlp), n, lows, "tree")     # the form for several rows
      else:
        mlp(pb, ctx, li, d["layers"][li], cfg, ls)
    _emit_final_norm(pb, cfg, d, n)
    pb.op("gemv", wf="f16", epi="f32", x="hid", w="lm_head", y="logits", nb=n, n=V, k=D)
    pb.op("sample", logits="logits", nb=n, v=V, u="u", temp="temp", topk="topk", topp="topp", minp="minp", tok="tok_out",
          logp="logp")
    plan_gemv_chains(pb)
    plan_l2_prefetch(pb)
    prog = R.Program.from_text(pb.text(), {"tok": (n,), "u": (n,)}, {"tok_out": (n,), "logits": (n, V)}, model.device,
                               {"tok": "int32", "u": "fp32", "tok_out": "int32", "logits": "fp32"})
    self.prog = prog
    if feed:
      prog.share_buffer(0, "tok_out", 0, "tok")
    prog.bind("embed", d["embed"]); prog.bind("lm_head", d["lm_head"])
    model._bind_globals(prog)
    if cfg.rope:
      cos_t, sin_t = rope_tables(rows, dh, cfg.rope_base, cfg.rotary_dim, cfg.rope_interleaved, cfg.rope_scaling)
      prog.upload("rope.cos", cos_t); prog.upload("rope.sin", sin_t)
    for li in range(cfg.n_layers):
      model._bind_layer(prog, li, d["layers"][li])
    for name, t in self._planes.items():
      prog.bind(name, t)
    for low in lows:
      low.finish(prog)
    self._lows = lows                                       # own the weights of lowered MLPs
    prog.bind("kv.table", kv.table); prog.bind("kv.lens", kv.lens)
    view = lambda name, dt="int32", shape=(B, T): prog.tensor(name, shape, dt)     # noqa: E731
    self.out, self.logp, self.logits = view("tok_out"), view("logp", "fp32"), view("logits", "fp32", (B, T, V))
    self.tok = self.out if feed else view("tok")
    self.u, self.nodes = view("u", "fp32"), view("nodes", shape=(B,))
    self.temperature, self.top_k = view("temp", "fp32"), view("topk")
    self.top_p, self.min_p = view("topp", "fp32"), view("minp", "fp32")
    self._pos, self._depth = view("pos"), view("depth")
    self.stream = torch.cuda.ExternalStream(prog.stream(), device=kv.device)
    with torch.cuda.device(kv.device):
      self._depth.copy_(torch.from_numpy(depth).expand(B, T))
      view("mask", shape=(B, T, mask.shape[1])).copy_(torch.from_numpy(mask).expand(B, T, -1))
      self.nodes.fill_(T)
      for t, v in ((self.temperature, temperature), (self.top_k, top_k), (self.top_p, top_p), (self.min_p, min_p)):
        t.fill_(v)
      torch.cuda.synchronize()

  def run(self) -> None:
    """Launches the step (call inside `torch.cuda.stream(self.stream)`)."""
    if self._learned_pos:
      torch.add(self.kv.lens[:self.B, None], self._depth, out=self._pos)
    self.prog.execute_async()

  def check(self) -> None:
    """Waits for the step and raises on an error that its kernels or the cache's recorded."""
    self.prog.sync()
    with torch.cuda.stream(self.stream):
      self.kv.check()

  def release(self) -> None:
    self.prog.release()


def _stops(eos_id):
  return {int(eos_id)} if isinstance(eos_id, int) else {int(e) for e in (eos_id or ())}


def sample_generate(model: LlamaPrefill, token_ids, n: int, max_new_tokens: int = 40, eos_id=None, temperature: float = 1.0,
                    top_p: float = 1.0, top_k: int = 0, min_p: float = 0.0, seed: int | None = None, page: int = 64,
                    stats: dict | None = None):
  """`n` continuations of one prompt, drawn independently: the prompt is prefilled once, its pages are shared by
  all sequences, and every step decodes one token of each and draws the next on the device. Returns n token
  lists, each ended by a stop token or max_new_tokens. `seed` fixes the random numbers. `stats` gets the pages
  in use at the end."""
  prompt = [int(t) for t in token_ids]
  model._check_ids(prompt)
  n, steps = int(n), int(max_new_tokens)
  if n < 1 or not prompt:
    raise ValueError("sample_generate needs a prompt and at least one sample")
  if steps < 1:
    return [[] for _ in range(n)]
  P, eos = len(prompt), _stops(eos_id)
  own = -(-(P + steps) // page) - P // page                  # pages that a sequence does not share
  kv = PagedKV(model.cfg, n, P + steps, pages=-(-P // page) + n * own, page=page, device=model.device)
  step = TreeStep(model, kv, n, max_pos=P + steps, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p,
                  feed=True)
  try:
    pre, real, _ = model._prefill_hidden(prompt)
    logits = model._logits(pre["prog"].read_output("hid")[real - 1])
    u = np.random.default_rng(seed).random((steps, n), np.float32)
    with torch.cuda.stream(step.stream):
      u = torch.from_numpy(u).to(kv.device)
      kv.seed(0, pre, real)
      if n > 1:
        kv.fork([0] * (n - 1), range(1, n))
      first = torch.from_numpy(np.ascontiguousarray(logits, np.float32)).to(kv.device).expand(n, -1).contiguous()
      hist = torch.empty((steps, n), dtype=torch.int32, device=kv.device)
      kernels.sample(first, u[0], temperature, top_k, top_p, min_p, out=(step.out.view(n), step.logp.view(n)))
      hist[0].copy_(step.out.view(n))
      every, one = torch.arange(n, dtype=torch.int32, device=kv.device), torch.ones((n,), dtype=torch.int32, device=kv.device)
      group = max(1, int(model.eos_check_every)) if eos else steps
      stop = torch.tensor(sorted(eos), dtype=torch.int32, device=kv.device)
      done = 1
      while done < steps:
        if eos and bool(torch.isin(hist[:done], stop).any(0).all()):
          break
        for i in range(done, min(done + group, steps)):
          kv.reserve(every, one)
          step.u.copy_(u[i].view(n, 1))
          step.run()
          kv.lens.add_(one)
          hist[i].copy_(step.out.view(n))
        done = min(done + group, steps)
      step.check()
      tokens = hist[:done].t().cpu().numpy()
      if stats is not None:
        stats.update(pages=int((kv.refs > 0).sum()))
  finally:
    step.release()
  out = []
  for row in tokens.tolist():
    end = next((i + 1 for i, t in enumerate(row) if t in eos), len(row))
    out.append(row[:end])
  return out
