"""Python wrappers of the kernel-level C ABI (include/af_cuda.h). Tensors are torch CUDA tensors used
only as device memory; every call goes through libaf_cuda.so on torch's current stream and raises on
a non-zero return code. No CPU path exists."""
from __future__ import annotations

import ctypes

import numpy as np

import torch

from . import _runtime as R


def _stream(t) -> int:
  dev = t.get_device()
  if dev < 0:                                              # the raw call would take -1 for the current device
    raise ValueError(f"a CUDA tensor is wanted, not one on {t.device}")
  return torch._C._cuda_getCurrentRawStream(dev)                  # a twentieth of current_stream(...).cuda_stream


def _p(t) -> int:
  return 0 if t is None else t.data_ptr()


def _need(cond, msg):
  if not cond:
    raise ValueError(msg)


def quantize_per_row_i8(W):
  """Per-row int8 codes [N,K] + fp16 scales [N] (bit-exact to the reference numpy encoder)."""
  import torch
  _need(W.is_cuda and W.dim() == 2 and W.is_contiguous(), "W must be a contiguous 2-D CUDA tensor")
  _need(W.dtype in (torch.float16, torch.float32), "W must be fp16 or fp32")
  N, K = W.shape
  q = torch.empty((N, K), dtype=torch.int8, device=W.device)
  s = torch.empty((N,), dtype=torch.float16, device=W.device)
  R.check(R.lib().af_quantize_per_row_i8(_p(W), int(W.dtype == torch.float16), N, K, _p(q), _p(s), _stream(W)),
          "af_quantize_per_row_i8")
  return q, s


def quantize_g32_i4(W):
  """Group-32 int4: packed [N, K/2] uint8 + fp16 scales [N, K/32]."""
  import torch
  _need(W.is_cuda and W.dim() == 2 and W.is_contiguous(), "W must be a contiguous 2-D CUDA tensor")
  N, K = W.shape
  _need(K % 32 == 0, "K must be a multiple of 32")
  p = torch.empty((N, K // 2), dtype=torch.uint8, device=W.device)
  s = torch.empty((N, K // 32), dtype=torch.float16, device=W.device)
  R.check(R.lib().af_quantize_g32_i4(_p(W), int(W.dtype == torch.float16), N, K, _p(p), _p(s), _stream(W)),
          "af_quantize_g32_i4")
  return p, s


def gemv(x, w, scales=None, bias=None, wf=R.W_I8, epi=R.EPI_F32, y=None, n_out=None):
  """y = epi(scales (.) (x . W^T) + bias). x [NB, K] fp16; w rows [N, ...]."""
  import torch
  _need(x.is_cuda and x.dtype == torch.float16 and x.dim() == 2, "x must be [NB, K] fp16 CUDA")
  NB, K = x.shape
  N = w.shape[0]
  cols = N // 2 if epi == R.EPI_SWIGLU else N
  if y is None:
    dt = torch.float16 if epi in (R.EPI_F16, R.EPI_SWIGLU) else torch.float32
    y = torch.zeros((NB, cols), dtype=dt, device=x.device)
  R.check(R.lib().af_gemv(wf, epi, _p(x), x.stride(0), _p(w), _p(scales), _p(bias), _p(y), y.stride(0), NB, N, K,
                          _stream(x)), "af_gemv")
  return y


def lm_head_argmax(x, w, scales=None, wf=R.W_F16, logits=True, pos=None, scratch=None, out=None):
  """Greedy token per row of x [NB, K] fp16 against head rows w [V, K]; optional fp32 logits.
  `scratch` (zeroed, left zeroed) may be reused across calls of one shape; `out` = (tok, logits)
  preallocated outputs."""
  import torch
  NB, K = x.shape
  V = w.shape[0]
  L = R.lib()
  nbytes = ctypes.c_size_t()
  R.check(L.af_lm_head_argmax_scratch(wf, V, K, NB, ctypes.byref(nbytes)), "scratch")
  if scratch is None:
    scratch = torch.zeros((nbytes.value,), dtype=torch.uint8, device=x.device)
  _need(scratch.numel() >= nbytes.value, "lm_head scratch too small")
  if out is not None:
    tok, lg = out
  else:
    tok = torch.zeros((NB,), dtype=torch.int32, device=x.device)
    lg = torch.zeros((NB, V), dtype=torch.float32, device=x.device) if logits else None
  R.check(L.af_lm_head_argmax(wf, _p(x), x.stride(0), _p(w), _p(scales), _p(lg), NB, V, K, _p(tok), _p(pos),
                              _p(scratch), scratch.numel(), _stream(x)), "af_lm_head_argmax")
  return tok, lg


def rmsnorm(x, g, floor):
  import torch
  NB, D = x.shape
  out = torch.empty((NB, D), dtype=torch.float16, device=x.device)
  R.check(R.lib().af_rmsnorm(_p(x), int(x.dtype == torch.float16), x.stride(0), _p(g), float(floor), _p(out),
                             out.stride(0), NB, D, _stream(x)), "af_rmsnorm")
  return out


def attn_decode_scratch_bytes(nb, kv, n_split, g, dh) -> int:
  n = ctypes.c_size_t()
  R.check(R.load_library().af_attn_decode_scratch(nb, kv, n_split, g, dh, ctypes.byref(n)), "scratch")
  return n.value


def attn_decode(qkv, kc, vc, pos, cos_t, sin_t, H, KV, dh, scale, kv_c=1.0, expand=False, n_split=1, scratch=None,
                err=None, out=None):
  """Decode attention; updates kc/vc at pos in place; returns fp16 [NB, H*dh]."""
  import torch
  NB = qkv.shape[0]
  M = kc.shape[2]
  if out is None:
    out = torch.zeros((NB, H * dh), dtype=torch.float16, device=qkv.device)
  if n_split > 1 and scratch is None:
    scratch = torch.zeros((attn_decode_scratch_bytes(NB, KV, n_split, H // KV, dh),), dtype=torch.uint8,
                          device=qkv.device)
  nbytes = 0 if scratch is None else scratch.numel()
  R.check(R.lib().af_attn_decode(_p(qkv), qkv.stride(0), _p(kc), _p(vc), _p(pos), _p(cos_t), _p(sin_t), _p(out),
                                 out.stride(0), NB, H, KV, dh, M, n_split, float(scale), float(kv_c), int(expand),
                                 _p(scratch), nbytes, _p(err), _stream(qkv)), "af_attn_decode")
  return out


def pack_i8_tiles(q):
  """Per-row int8 codes [N, K] -> the tensor-core fragment-tile layout (uint8, flat)."""
  import torch
  N, K = q.shape
  L = R.lib()
  out = torch.empty((L.af_pack_i8_tiles_bytes(N, K),), dtype=torch.uint8, device=q.device)
  R.check(L.af_pack_i8_tiles(_p(q), N, K, _p(out), _stream(q)), "af_pack_i8_tiles")
  return out


def gemv_tc_scratch(N, K, NB, device):
  import torch
  n = R.load_library().af_gemv_tc_scratch_bytes(N, K, NB)
  return torch.zeros((max(n, 1),), dtype=torch.uint8, device=device), n


def pack_i4_tiles(packed, scales, N, K):
  """Group-32 int4 (packed [N, K/2] + scales [N, K/32]) -> tensor-core tiles with the scales inside."""
  import torch
  L = R.lib()
  out = torch.empty((L.af_pack_i4_tiles_bytes(N, K),), dtype=torch.uint8, device=packed.device)
  R.check(L.af_pack_i4_tiles(_p(packed), _p(scales), N, K, _p(out), _stream(packed)), "af_pack_i4_tiles")
  return out


def gemv_tc_i4(x, tiles, N, K, bias=None, epi=R.EPI_F32, y=None, scratch=None):
  """Tensor-core group-32 int4 GEMV over pack_i4_tiles output. x [NB, K] fp16."""
  import torch
  NB = x.shape[0]
  cols = N // 2 if epi == R.EPI_SWIGLU else N
  if y is None:
    dt = torch.float16 if epi in (R.EPI_F16, R.EPI_SWIGLU) else torch.float32
    y = torch.zeros((NB, cols), dtype=dt, device=x.device)
  if scratch is None:
    scratch, nbytes = gemv_tc_scratch(N, K, NB, x.device)
  else:
    nbytes = scratch.numel()
  R.check(R.lib().af_gemv_tc_i4(epi, _p(x), x.stride(0), _p(tiles), _p(bias), _p(y), y.stride(0), NB, N, K,
                                _p(scratch), nbytes, _stream(x)), "af_gemv_tc_i4")
  return y


def gemv_tc(x, tiles, scales, N, K, bias=None, epi=R.EPI_F32, y=None, scratch=None):
  """Tensor-core int8 GEMV over packed tiles. x [NB, K] fp16."""
  import torch
  NB = x.shape[0]
  cols = N // 2 if epi == R.EPI_SWIGLU else N
  if y is None:
    dt = torch.float16 if epi in (R.EPI_F16, R.EPI_SWIGLU) else torch.float32
    y = torch.zeros((NB, cols), dtype=dt, device=x.device)
  if scratch is None:
    scratch, nbytes = gemv_tc_scratch(N, K, NB, x.device)
  else:
    nbytes = scratch.numel()
  R.check(R.lib().af_gemv_tc(epi, _p(x), x.stride(0), _p(tiles), _p(scales), _p(bias), _p(y), y.stride(0), NB, N, K,
                             _p(scratch), nbytes, _stream(x)), "af_gemv_tc")
  return y


def attn_decode_noalloc(qkv, kc, vc, pos, cos_t, sin_t, H, KV, dh, scale, kv_c=1.0, expand=False, n_split=1, err=None):
  """Decode attention using the library's built-in scratch (no allocation by the entry point).
  Returns (rc, out); rc != 0 means the shape was rejected (reason in _runtime.last_error())."""
  import torch
  NB = qkv.shape[0]
  M = kc.shape[2]
  out = torch.zeros((NB, H * dh), dtype=torch.float16, device=qkv.device)
  rc = R.lib().af_attn_decode_noalloc(_p(qkv), qkv.stride(0), _p(kc), _p(vc), _p(pos), _p(cos_t), _p(sin_t),
                                      _p(out), out.stride(0), NB, H, KV, dh, M, n_split, float(scale), float(kv_c),
                                      int(expand), _p(err), _stream(qkv))
  return rc, out


def moe_gate(logits, k, renorm=True):
  """Router logits [NB, E] fp32 -> (gw [NB, E] fp32, sel [NB, k] int32) on the device."""
  import torch
  NB, E = logits.shape
  gw = torch.zeros((NB, E), dtype=torch.float32, device=logits.device)
  sel = torch.zeros((NB, k), dtype=torch.int32, device=logits.device)
  R.check(R.lib().af_moe_gate(_p(logits), logits.stride(0), NB, E, k, int(renorm), _p(gw), _p(sel), _stream(logits)),
          "af_moe_gate")
  return gw, sel


def gemv_tc_expert(x, tiles, scales, N, K, E, wf=R.W_I8, epi=R.EPI_F32, y=None, sel=None, slot=0, fixed_e=0, rw=None,
                   scratch=None):
  """Tensor-core GEMV over E experts' tiles stored back to back; expert = sel[slot] or fixed_e."""
  import torch
  if sel is None and not 0 <= fixed_e < E:
    raise ValueError(f"fixed_e={fixed_e} outside the {E} experts of these tiles")
  NB = x.shape[0]
  cols = N // 2 if epi == R.EPI_SWIGLU else N
  if y is None:
    dt = torch.float16 if epi in (R.EPI_F16, R.EPI_SWIGLU) else torch.float32
    y = torch.zeros((NB, cols), dtype=dt, device=x.device)
  if scratch is None:
    scratch, nbytes = gemv_tc_scratch(N, K, NB, x.device)
  else:
    nbytes = scratch.numel()
  stride = tiles.numel() // E
  R.check(R.lib().af_gemv_tc_expert(wf, epi, _p(x), x.stride(0), _p(tiles), _p(scales), _p(y), y.stride(0), NB, N, K,
                                    _p(sel), slot, fixed_e, stride, N if scales is not None else 0, _p(rw), E,
                                    _p(scratch), nbytes, _stream(x)), "af_gemv_tc_expert")
  return y


def gemm_tc(x, tiles, scales, N, K, wf=R.W_I8, bias=None, epi=R.EPI_F32, y=None):
  """Prefill GEMM on tcgen05 over packed tiles: x [M, K] fp16 -> y [M, N] (or [M, N/2] for SWIGLU)."""
  import torch
  M = x.shape[0]
  cols = N // 2 if epi == R.EPI_SWIGLU else N
  if y is None:
    dt = torch.float16 if epi in (R.EPI_F16, R.EPI_SWIGLU) else torch.float32
    y = torch.zeros((M, cols), dtype=dt, device=x.device)
  R.check(R.lib().af_gemm_tc(wf, epi, _p(x), x.stride(0), _p(tiles), _p(scales), _p(bias), _p(y), y.stride(0), M, N, K,
                             _stream(x)), "af_gemm_tc")
  return y


def _i32(t, shape, name, dev):
  if not (t.dtype == torch.int32 and t.get_device() == dev and dev >= 0 and t.is_contiguous() and t.shape == shape):
    raise ValueError(f"{name} must be a contiguous int32 tensor of shape {tuple(shape)} on the call's CUDA device")
  return t.data_ptr()


def _entry(name, dev):
  """The C entry `name`, which runs on GPU `dev` whichever one is current; its last argument is dev's stream."""
  fn = getattr(R.lib(), name)
  if dev == torch._C._cuda_getDevice():
    return fn

  def there(*args):
    with torch.cuda.device(dev):
      return fn(*args)

  return there


def _err(t, dev):
  """The caller's error word, or none."""
  if t is None:
    return 0
  if not (t.get_device() == dev and t.dtype == torch.int32 and t.numel() >= 1):
    raise ValueError("err must be int32 [1] on the call's CUDA device")
  return t.data_ptr()


def _scratch(t, dev):
  """Pointer and bytes of a workspace."""
  if not (t.get_device() == dev and t.is_contiguous()):
    raise ValueError("scratch must be a contiguous tensor on the call's CUDA device")
  return t.data_ptr(), t.numel() * t.element_size()


_SAMPLE_DT = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _per_row(x, name, dtype, rows, dev):
  """A setting as (pointer of its row values, 0) or (0, the number for all rows)."""
  if hasattr(x, "data_ptr"):
    if not (x.get_device() == dev and x.dtype == dtype and x.shape == rows and x.is_contiguous()):
      raise ValueError(f"{name} must be a number or a contiguous {dtype} tensor [R] on the logits' device")
    return x.data_ptr(), 0
  _need(x == x and abs(x) != float("inf"), f"{name} must be finite")
  return 0, (max(-1, min(int(x), 0x7fffffff)) if name == "top_k" else x)


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, out=None):
  """One token per row of logits [R, V] (fp32, fp16 or bf16, rows any stride apart), drawn with the uniform numbers
  u [R] in [0, 1): temperature, then the top_k largest logits (ties with the last stay), of these the most
  probable until their mass reaches top_p (ties: lowest index first), of these the ones at least min_p as
  probable as the best; one draw in the order of the vocabulary. Each setting is a number or a CUDA tensor [R]
  (fp32; top_k int32); 0 (or top_p 1) turns it off, temperature 0 takes the first largest logit. Returns
  (tokens int32 [R], log-probabilities among the kept tokens fp32 [R]); -1 and -inf for a row that is all -inf
  or NaN. `out` = the two outputs, preallocated."""
  dev = logits.get_device()
  if not (dev >= 0 and logits.dim() == 2 and logits.dtype in _SAMPLE_DT):
    raise ValueError("logits must be a 2-D CUDA tensor of fp32, fp16 or bf16")
  n, V = logits.shape
  ld, col = logits.stride()
  _need(1 <= V < 1 << 24 and (col == 1 or V == 1), "logits must have contiguous rows of 1 to 2^24 - 1 values")
  if n <= 1:
    ld = V
  _need(ld >= V, "rows of logits must not overlap")
  rows = (n,)
  _need(u.get_device() == dev and u.dtype == torch.float32 and u.shape == rows and u.is_contiguous(),
        "u must be fp32 [R] on the logits' device")
  pt, st = _per_row(temperature, "temperature", torch.float32, rows, dev)
  pk, sk = _per_row(top_k, "top_k", torch.int32, rows, dev)
  pp, sp = _per_row(top_p, "top_p", torch.float32, rows, dev)
  pm, sm = _per_row(min_p, "min_p", torch.float32, rows, dev)
  if out is None:
    tok, logp = torch.empty_like(u, dtype=torch.int32), torch.empty_like(u)
  else:
    tok, logp = out
    _need(tok.dtype == torch.int32 and logp.dtype == torch.float32
          and all(o.get_device() == dev and o.shape == rows and o.is_contiguous() for o in out),
          "out must be (int32 [R], fp32 [R]) on the logits' device")
  rc = _entry("af_sample", dev)(logits.data_ptr(), _SAMPLE_DT[logits.dtype], ld, n, V, u.data_ptr(), pt, pk, pp, pm, st, sk, sp, sm,
                                tok.data_ptr(), logp.data_ptr(), torch._C._cuda_getCurrentRawStream(dev))
  if rc:
    R.check(rc, "af_sample")
  return tok, logp


def tree_layout(parents):
  """Depths [T] and visibility masks [T, ceil(T / 32)] (int32, bit u of word w: node 32 w + u) of a tree given by
  each node's parent (-1: hangs on the prefix; parents come before their children), as numpy arrays."""
  T = len(parents)
  depth = np.zeros(T, np.int32)
  mask = np.zeros((T, -(-T // 32)), np.uint32)
  for t, p in enumerate(parents):
    _need(-1 <= p < t, f"node {t}: parent {p} must be -1 or an earlier node")
    if p >= 0:
      depth[t] = depth[p] + 1
      mask[t] = mask[p]
    mask[t, t >> 5] |= np.uint32(1 << (t & 31))
  return depth, mask.view(np.int32)


def attn_tree_scratch(B, T, H, KV, dh, device=None):
  """Workspace of `attn_tree` for these sizes; it may serve any number of calls of one stream."""
  return torch.zeros((max(1, R.load_library().af_attn_tree_scratch_bytes(B, T, H, KV, dh)),), dtype=torch.uint8,
                     device=device or "cuda")


def attn_tree(qkv, kc, vc, table, lens, cos_t, sin_t, H, KV, dh, scale, mask=None, depth=None, nodes=None, qn=None, kn=None,
              qn_floor=0.0, kn_floor=0.0, scratch=None, err=None, out=None):
  """Attention of T drafted tokens (nodes of a tree) for each of B sequences over a paged cache. qkv [B * T,
  (H + 2 KV) dh] fp32; kc / vc [P, KV, page, dh] fp16 (pages any stride apart); table [B, W] int32: the page of
  each run of `page` rows; lens [B] int32: the rows before the tree. Node t becomes cache row lens + t (k and v
  are written there), its rotary position is lens + depth[b, t] (default t); it sees the rows before lens and the
  nodes set in mask [B, T, ceil(T / 32)] (int32 bits, see `tree_layout`; default: a chain). T = 1 is the ordinary
  decode step. nodes [B]: live nodes of each sequence. lens is left as it is (`kv_compact` advances it). Returns
  fp16 [B * T, H * dh], zeros for nodes that see nothing or are not live. err: int32 [1], zero: gets the device
  error code of a node without a page or rotary position. Head dims 64 and 128 with pages of a multiple of 8 rows (or
  W = 1) run on the tensor cores, the rest takes ten times as long and more."""
  f16 = torch.float16
  dev = qkv.get_device()
  if not (dev >= 0 and qkv.dtype == torch.float32 and qkv.dim() == 2 and table.dim() == 2):
    raise ValueError("qkv must be fp32 [B * T, cols] on the GPU and table int32 [B, W]")
  (n, cols), (ld, one), (B, W) = qkv.shape, qkv.stride(), table.shape
  if not (one == 1 and KV >= 1 and H % KV == 0 and cols >= (H + 2 * KV) * dh):
    raise ValueError("qkv needs contiguous rows of (H + 2 KV) dh columns, H a multiple of KV")
  if not (B >= 1 and n >= B and n % B == 0 and n <= 256 * B):
    raise ValueError("qkv needs the same number of rows, 1 to 256, for each sequence of the table")
  T = n // B
  if dh not in (16, 32, 64, 128):
    raise ValueError("head dims 16, 32, 64 and 128")
  shape, strides = kc.shape, kc.stride()
  if not (kc.dtype == f16 and vc.dtype == f16 and kc.get_device() == dev and vc.get_device() == dev and vc.shape == shape
          and len(shape) == 4 and shape[1] == KV and shape[3] == dh):
    raise ValueError("kc / vc must be fp16 [P, KV, page, dh] on qkv's device")
  P, _, page, _ = shape
  ps = strides[0] if P > 1 else KV * page * dh
  if not (strides[1:] == (page * dh, dh, 1) and vc.stride() == strides and ps >= KV * page * dh and ps % 8 == 0):
    raise ValueError("kc / vc pages must be contiguous, and alike")
  words = (T + 31) // 32
  rows = 0
  if cos_t is not None:
    rows = cos_t.shape[0]
    if not (cos_t.shape == (rows, dh) and sin_t.shape == (rows, dh) and cos_t.dtype == f16 and sin_t.dtype == f16
            and cos_t.is_contiguous() and sin_t.is_contiguous() and cos_t.get_device() == dev and sin_t.get_device() == dev):
      raise ValueError("cos_t / sin_t must be fp16 [rows, dh] on qkv's device")
  for g, name in ((qn, "qn"), (kn, "kn")):
    if g is not None and not (g.get_device() == dev and g.dtype == f16 and g.shape == (dh,) and g.is_contiguous()):
      raise ValueError(f"{name} must be fp16 [dh] on qkv's device")
  if out is None:
    out = qkv.new_empty((n, H * dh), dtype=f16)
    ldo = H * dh
  else:
    if not (out.get_device() == dev and out.dtype == f16 and out.shape == (n, H * dh) and out.stride(1) == 1):
      raise ValueError("out must be fp16 [B * T, H * dh] on qkv's device")
    ldo = out.stride(0)
  if scratch is None:
    scratch = attn_tree_scratch(B, T, H, KV, dh, qkv.device)
  scr, scr_bytes = _scratch(scratch, dev)
  rc = _entry("af_attn_tree", dev)(
      qkv.data_ptr(), ld, kc.data_ptr(), vc.data_ptr(), ps, P, page, _i32(table, (B, W), "table", dev), W,
      _i32(lens, (B,), "lens", dev), 0 if nodes is None else _i32(nodes, (B,), "nodes", dev),
      0 if depth is None else _i32(depth, (B, T), "depth", dev), 0 if mask is None else _i32(mask, (B, T, words), "mask", dev),
      words, _p(cos_t), _p(sin_t), rows, _p(qn), _p(kn), qn_floor, kn_floor, out.data_ptr(), ldo, B, T, H, KV, dh, scale, scr,
      scr_bytes, _err(err, dev), torch._C._cuda_getCurrentRawStream(dev))
  if rc:
    R.check(rc, "af_attn_tree")
  return out


def _book(table, lens, refs, slots):
  if not (table.dim() == 2 and lens.dim() == 1 and slots.dim() == 1 and (refs is None or refs.dim() == 1)):
    raise ValueError("table [S, W], lens [S], refs [P] and slots [n] are wanted")
  S, W = table.shape
  n = slots.shape[0]
  if n > 1024:
    raise ValueError("at most 1024 slots a call")
  dev = table.get_device()
  return (_i32(table, (S, W), "table", dev), S, W, _i32(lens, (S,), "lens", dev),
          0 if refs is None else _i32(refs, refs.shape, "refs", dev), _i32(slots, (n,), "slots", dev), n, dev)


def _pool(pool, dev):
  if not (pool.get_device() == dev and pool.dim() == 6 and pool.is_contiguous() and pool.element_size() == 2):
    raise ValueError("pool must be a contiguous 16-bit tensor [layers, 2, P, KV, page, dh] on the table's device")
  L, two, P, KV, page, dh = pool.shape
  if two != 2 or dh % 8:
    raise ValueError("pool must be [layers, 2, P, KV, page, dh], dh a multiple of 8")
  return L, P, KV, page, 2 * dh


def kv_fork(table, lens, refs, src, dst, page, err=None):
  """Slots dst[i] become copies of slots src[i]: they give back the pages they hold and share the ones that src
  fills (counted in refs [P]); no row moves until `kv_reserve` makes a shared page writable. All int32 on the GPU;
  table [S, W], lens [S]. The dst are distinct and none is a src."""
  pt, S, W, pl, pr, pd, n, dev = _book(table, lens, refs, dst)
  _need(page >= 1, "page must be positive")
  R.check(_entry("af_kv_fork", dev)(pt, S, W, pl, pr, refs.shape[0], page, _i32(src, (n,), "src", dev), pd, n, _err(err, dev),
                                    _stream(table)), "af_kv_fork")


def kv_reserve(pool, table, lens, refs, slots, rows, err=None, scratch=None):
  """Rows [lens, lens + rows[i]) of each slot get pages of the slot's own: free ones, lowest number first, and
  copies (in every layer of pool [layers, 2, P, KV, page, dh]) of a shared page that rows are appended to."""
  pt, S, W, pl, pr, ps, n, dev = _book(table, lens, refs, slots)
  L, P, KV, page, rb = _pool(pool, dev)
  _need(refs.shape[0] == P, "refs must have an entry for each page of the pool")
  if scratch is None:
    scratch = refs.new_empty((R.lib().af_kv_reserve_scratch_bytes(n, P) // 4 + 1,))               # int32
  scr, scr_bytes = _scratch(scratch, dev)
  R.check(_entry("af_kv_reserve", dev)(pool.data_ptr(), L, KV, rb, pt, S, W, pl, pr, P, page, ps, _i32(rows, (n,), "rows", dev), n,
                                       scr, scr_bytes, _err(err, dev), _stream(table)), "af_kv_reserve")


def kv_free(table, lens, refs, slots, page, keep=None, err=None):
  """Gives back what the slots hold past keep[i] rows (default: everything)."""
  pt, S, W, pl, pr, ps, n, dev = _book(table, lens, refs, slots)
  _need(page >= 1, "page must be positive")
  R.check(_entry("af_kv_free", dev)(pt, S, W, pl, pr, refs.shape[0], page, ps, 0 if keep is None else _i32(keep, (n,), "keep", dev),
                                    n, _err(err, dev), _stream(table)), "af_kv_free")


def kv_compact(pool, table, lens, slots, path, n_path, lens_out=None, err=None):
  """The rows lens + path[i, j], j < n_path[i], of each slot move to lens + j in every layer's K and V: the accepted
  path [n, D] through a drafted tree (node numbers, rising) becomes part of the prefix. Returns the new lengths:
  lens with n_path added to the listed slots (a new tensor, or lens_out)."""
  pt, S, W, pl, _, ps, n, dev = _book(table, lens, None, slots)
  L, P, KV, page, rb = _pool(pool, dev)
  _need(path.dim() == 2, "path must be int32 [n, D]")
  D = path.shape[1]
  if lens_out is None:
    lens_out = lens.new_empty(lens.shape)
  _need(lens_out.data_ptr() != lens.data_ptr(), "lens_out must be another buffer than lens")
  R.check(_entry("af_kv_compact", dev)(pool.data_ptr(), L, KV, rb, P, page, pt, S, W, pl, ps, _i32(path, (n, D), "path", dev), D,
                                       _i32(n_path, (n,), "n_path", dev), n, _i32(lens_out, (S,), "lens_out", dev), _err(err, dev),
                                       _stream(table)), "af_kv_compact")
  return lens_out
