"""Refusals of the sampling, tree-attention and cache-page entry points, and the tree helper (no GPU)."""
import ctypes

import numpy as np
import pytest
import torch

from aneforge_b200 import kernels as K


def test_tree_layout():
  depth, mask = K.tree_layout([-1, 0, 0, 1, -1])
  assert depth.tolist() == [0, 1, 1, 2, 0]
  assert mask[:, 0].tolist() == [0b1, 0b11, 0b101, 0b1011, 0b10000]
  depth, mask = K.tree_layout(list(range(-1, 69)))
  assert depth[-1] == 69 and mask.shape == (70, 3) and mask.dtype == np.int32
  assert mask.view(np.uint32)[63].tolist() == [0xFFFFFFFF, 0xFFFFFFFF, 0] and mask.view(np.uint32)[69, 2] == 0b111111
  for bad in ([0], [-1, 1], [-2], [-1, 0, 5]):
    with pytest.raises(ValueError):
      K.tree_layout(bad)


def test_host_tensors_are_refused():
  f, i = torch.zeros(2, 8), torch.zeros(2, dtype=torch.int32)
  with pytest.raises(ValueError):
    K.sample(f, torch.zeros(2))
  with pytest.raises(ValueError):
    K.attn_tree(torch.zeros(2, 3 * 64), torch.zeros(4, 1, 8, 64).half(), torch.zeros(4, 1, 8, 64).half(), i.view(2, 1), i, None,
                None, 1, 1, 64, 1.0)
  with pytest.raises(ValueError):
    K.kv_fork(i.view(2, 1), i, i, i, i, 8)
  with pytest.raises(ValueError):
    K.kv_free(i.view(2, 1), i, i, i, 8)
  with pytest.raises(ValueError):
    K.kv_reserve(torch.zeros(1, 2, 2, 1, 8, 8).half(), i.view(2, 1), i, i, i, i)
  with pytest.raises(ValueError):
    K.kv_compact(torch.zeros(1, 2, 2, 1, 8, 8).half(), i.view(2, 1), i, i, i.view(2, 1), i)


def test_native_entries_refuse_before_they_launch():
  """Bad arguments give -1 and a message; none of these calls reaches the device."""
  from aneforge_b200 import build
  L = ctypes.CDLL(str(build.build()))
  from aneforge_b200 import _runtime as R
  for name, res, args in R.SIGNATURES:
    getattr(L, name).restype, getattr(L, name).argtypes = res, args
  p = 1 << 20                                              # never read
  sample = lambda **k: L.af_sample(*[dict(dict(l=p, dt=0, ld=8, r=1, v=8, u=p, tok=p), **k)[x] for x in ("l", "dt", "ld", "r", "v", "u")],
                                   None, None, None, None, 1.0, 0, 1.0, 0.0, dict(dict(tok=p), **k)["tok"], None, None)
  for bad in (dict(l=None), dict(u=None), dict(tok=None), dict(v=0), dict(ld=7), dict(r=-1), dict(dt=3), dict(v=(1 << 24) + 1, ld=1 << 25)):
    assert sample(**bad) == -1, bad
    assert b"af_sample" in L.af_last_error()
  base = dict(qkv=p, ld=192, kc=p, vc=p, ps=512, P=4, page=8, table=p, W=1, lens=p, words=1, rows=0, out=p, ldo=64, b=1, t=1, h=1,
              kv=1, dh=64, scr=p, nb=1 << 30, cos=None, sin=None, mask=None)

  def tree(**k):
    a = dict(base, **k)
    return L.af_attn_tree(a["qkv"], a["ld"], a["kc"], a["vc"], a["ps"], a["P"], a["page"], a["table"], a["W"], a["lens"], None, None,
                          a["mask"], a["words"], a["cos"], a["sin"], a["rows"], None, None, 0.0, 0.0, a["out"], a["ldo"], a["b"],
                          a["t"], a["h"], a["kv"], a["dh"], 1.0, a["scr"], a["nb"], None, None)

  for bad in (dict(qkv=None), dict(kc=None), dict(kc=p + 2), dict(vc=p + 8), dict(table=None), dict(lens=None), dict(out=None), dict(scr=None),
              dict(nb=3), dict(ld=191), dict(ldo=63), dict(ps=511), dict(ps=516), dict(P=0), dict(page=0), dict(W=0), dict(b=-1), dict(t=0),
              dict(t=257), dict(h=0), dict(kv=0), dict(h=3, kv=2), dict(dh=48), dict(dh=256, ps=1 << 20, ld=1 << 12, ldo=1 << 12),
              dict(cos=p), dict(cos=p, sin=p, rows=0), dict(mask=p, t=33, words=1)):
    assert tree(**bad) == -1, bad
  for n in (-1, 1025):
    assert L.af_kv_fork(p, 4, 4, p, p, 8, 8, p, p, n, None, None) == -1
    assert L.af_kv_free(p, 4, 4, p, p, 8, 8, p, None, n, None, None) == -1
    assert L.af_kv_reserve(p, 1, 1, 128, p, 4, 4, p, p, 8, 8, p, p, n, p, 1 << 30, None, None) == -1
  assert L.af_kv_fork(p, 4, 4, p, None, 8, 8, p, p, 1, None, None) == -1
  assert L.af_kv_reserve(p, 1, 1, 120, p, 4, 4, p, p, 8, 8, p, p, 1, p, 1 << 30, None, None) == -1
  assert L.af_kv_reserve(p, 1, 1, 128, p, 4, 4, p, p, 8, 8, p, p, 1, p, 8, None, None) == -1
  assert L.af_kv_reserve(p + 2, 1, 1, 128, p, 4, 4, p, p, 8, 8, p, p, 1, p, 1 << 30, None, None) == -1
  assert L.af_kv_compact(p, 1, 1, 128, 8, 8, p, 4, 4, p, p, p, 1, p, 1, p, None, None) == -1           # lens_out is lens
  assert L.af_kv_compact(p, 1, 1, 128, 8, 8, p, 4, 4, p, p, p, 0, p, 1, p + 64, None, None) == -1
  assert L.af_attn_tree_scratch_bytes(1, 0, 1, 1, 64) == 0 and L.af_attn_tree_scratch_bytes(1, 1, 3, 2, 64) == 0
  assert L.af_kv_reserve_scratch_bytes(-1, 4) == 0


def test_plan_ops_are_checked(tmp_path):
  """The plan ops `sample` and `attn_tree`: a whole plan is taken, one with a buffer missing or too small is not."""
  from aneforge_b200 import _runtime as R
  from aneforge_b200.plan import PlanBuilder
  lib = R.load_library()

  def plan(**change):
    pb = PlanBuilder()
    size = dict(qkv=4 * 8 * 192, K=2 * 4 * 16 * 64, V=2 * 4 * 16 * 64, table=4 * 2 * 4, lens=8, mask=32, att=2 * 8 * 64,
                scr=lib.af_attn_tree_scratch_bytes(2, 4, 1, 1, 64), logits=4 * 2 * 100, u=8, temp=8, topk=8, topp=8, minp=8, tok=8)
    size.update({k: v for k, v in change.items() if k in size})
    for k, v in size.items():
      pb.buf(k, v, "ext" if k in ("K", "V", "table", "lens") else "state")
    kv = dict(qkv="qkv", kc="K", vc="V", table="table", lens="lens", mask="mask", out="att", scr="scr", b=2, t=4, h=1, kv=1, dh=64,
              p=4, page=16, w=4, scale=0.125)
    kv.update({k: v for k, v in change.items() if k in kv and k not in size})
    pb.op("attn_tree", **kv)
    pb.op("sample", logits="logits", nb=2, v=100, u="u", temp="temp", topk="topk", topp="topp", minp="minp", tok="tok")
    d = tmp_path / f"p{len(list(tmp_path.iterdir()))}"
    d.mkdir()
    (d / "plan.txt").write_text(pb.text())
    return lib.af_compile_check(str(d).encode(), b"", 1, None)

  assert plan() == 0
  for bad in (dict(K=2), dict(table=4), dict(scr=64), dict(mask=16), dict(logits=400), dict(tok=4), dict(b=0), dict(t=257),
              dict(kv=2), dict(vc="none"), dict(u=4)):
    assert plan(**bad) == -1, bad


def test_no_stream_for_a_host_tensor():
  """Wrappers without checks of their own (rmsnorm, attn_decode, gemv_tc, ...) launch nothing on host memory."""
  with pytest.raises(ValueError, match="CUDA tensor"):
    K._stream(torch.zeros(2))


class On(torch.Tensor):
  """A host tensor that says it lies on GPU `dev`."""
  dev = 0
  is_cuda = property(lambda self: self.dev >= 0)

  def get_device(self):
    return self.dev


def on(dev, t):
  t = t.as_subclass(On)
  t.dev = dev
  return t


class Calls:
  """A library that takes every call down, with the device it was made on."""

  def __init__(self):
    self.made = []

  def __getattr__(self, name):
    if name.endswith("_bytes"):
      return lambda *a: 64
    return lambda *a: self.made.append((name, torch._C._cuda_getDevice(), a[-1])) or 0


@pytest.fixture
def calls(monkeypatch):
  c, now = Calls(), [0]

  class Device:
    def __init__(self, d):
      self.d = d

    def __enter__(self):
      self.was, now[0] = now[0], self.d

    def __exit__(self, *a):
      now[0] = self.was

  monkeypatch.setattr(K.R, "lib", lambda: c)
  monkeypatch.setattr(K.R, "load_library", lambda: c)
  monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: now[0], raising=False)
  monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda d: 100 + d, raising=False)
  monkeypatch.setattr(torch.cuda, "device", Device)
  return c


def operands(dev):
  """For each entry point: the call, and its tensors by name."""
  i = lambda *s: on(dev, torch.zeros(s, dtype=torch.int32))
  f = lambda *s: on(dev, torch.zeros(s))
  h = lambda *s: on(dev, torch.zeros(s).half())
  books = dict(table=i(3, 2), lens=i(3), refs=i(4), err=i(1))
  return {
    "af_sample": (lambda **k: K.sample(**k), dict(
      logits=f(2, 8), u=f(2), temperature=f(2), top_k=i(2), top_p=f(2), min_p=f(2), out=(i(2), f(2)))),
    "af_attn_tree": (lambda **k: K.attn_tree(H=1, KV=1, dh=64, scale=1.0, **k), dict(
      qkv=f(2, 192), kc=h(4, 1, 8, 64), vc=h(4, 1, 8, 64), table=i(2, 1), lens=i(2), cos_t=h(8, 64), sin_t=h(8, 64), mask=i(2, 1, 1),
      depth=i(2, 1), nodes=i(2), qn=h(64), kn=h(64), scratch=on(dev, torch.zeros(64, dtype=torch.uint8)), err=i(1), out=h(2, 64))),
    "af_kv_fork": (lambda **k: K.kv_fork(page=8, **k), dict(books, src=i(1), dst=i(1))),
    "af_kv_reserve": (lambda **k: K.kv_reserve(**k), dict(books, pool=h(1, 2, 4, 1, 8, 8), slots=i(1), rows=i(1), scratch=i(64))),
    "af_kv_free": (lambda **k: K.kv_free(page=8, **k), dict(books, slots=i(1), keep=i(1))),
    "af_kv_compact": (lambda **k: K.kv_compact(**k), dict(
      pool=h(1, 2, 4, 1, 8, 8), table=i(3, 2), lens=i(3), slots=i(1), path=i(1, 2), n_path=i(1), lens_out=i(3), err=i(1))),
  }


@pytest.mark.parametrize("entry", ["af_sample", "af_attn_tree", "af_kv_fork", "af_kv_reserve", "af_kv_free", "af_kv_compact"])
def test_every_operand_lies_on_the_calls_device(entry, calls):
  """A tensor of the host or of another GPU, the workspace and the error word among them, is refused before a launch."""
  call, good = operands(0)[entry]
  call(**good)
  assert [c[0] for c in calls.made] == [entry]
  for name, t in good.items():
    for dev in (-1, 1):
      bad = tuple(on(dev, x.clone()) for x in t) if isinstance(t, tuple) else on(dev, t.clone())
      with pytest.raises(ValueError):
        call(**dict(good, **{name: bad}))
  if "err" in good:
    with pytest.raises(ValueError):
      call(**dict(good, err=on(0, torch.zeros(1))))
  assert len(calls.made) == 1


@pytest.mark.parametrize("entry", ["af_sample", "af_attn_tree", "af_kv_fork", "af_kv_reserve", "af_kv_free", "af_kv_compact"])
def test_a_call_runs_on_its_operands_gpu(entry, calls):
  """With GPU 0 current and the operands on GPU 1, the launch is made on GPU 1, on its stream."""
  call, good = operands(1)[entry]
  call(**good)
  call, good = operands(0)[entry]
  call(**good)
  assert calls.made == [(entry, 1, 101), (entry, 0, 100)] and torch._C._cuda_getDevice() == 0


def test_compact_refuses_more_slots_than_the_other_page_calls():
  from aneforge_b200 import build, _runtime as R
  L = ctypes.CDLL(str(build.build()))
  for name, res, args in R.SIGNATURES:
    getattr(L, name).restype, getattr(L, name).argtypes = res, args
  p = 1 << 20                                              # never read
  for n in (-1, 1025):
    assert L.af_kv_compact(p, 1, 1, 128, 8, 8, p, 4, 4, p, p, p, 1, p, n, p + 64, None, None) == -1
    assert b"invalid argument" in L.af_last_error()


def test_a_vocabulary_whose_weights_pass_64_bits_is_refused(calls):
  """2^24 equal logits weigh 2^40 each: their sum would be 0."""
  from aneforge_b200 import build, _runtime as R
  u = on(0, torch.zeros(1))
  K.sample(on(0, torch.empty(1, (1 << 24) - 1)), u)
  with pytest.raises(ValueError):
    K.sample(on(0, torch.empty(1, 1 << 24)), u)
  assert len(calls.made) == 1
  L = ctypes.CDLL(str(build.build()))
  for name, res, args in R.SIGNATURES:
    getattr(L, name).restype, getattr(L, name).argtypes = res, args
  p = 1 << 20                                              # never read
  for dtype in (0, 1, 2):
    assert L.af_sample(p, dtype, 1 << 24, 1, 1 << 24, p, None, None, None, None, 1.0, 0, 1.0, 0.0, p, None, None) == -1
    assert b"invalid argument" in L.af_last_error()
