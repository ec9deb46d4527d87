"""Attention of drafted trees over a paged cache (`kernels.attn_tree`) against the formula in 64 bits.

Bound of an output element: q, k and v are rounded to fp16 in both (q and k after a rotation in fp32, so that a
rounding can fall the other way: 2^-11 of an element of either, which moves a score by less than
2^-11 * 2 * sum |q k| scale); the weights are rounded to fp16 before the product with v (2^-11), the output to fp16
(2^-11), and score, sum and exponential carry fp32 errors (2^-18 for these sizes). With A the weighted sum of |v|:
|error| <= (2^-10 + 2^-12) A + 2^-24, and 2^-10 * (largest score sum) A more where RoPE is on."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def need_gpu():
  if not torch.cuda.is_available():
    pytest.skip("no CUDA device")


def setup(B, T, H, KV, dh, lens, page, seed=0, rope=False, extra_pages=3, tree="random", width=None, fill=float("nan"), qscale=1.5):
  """Inputs on the GPU; every cache row that holds nothing is NaN."""
  g = torch.Generator().manual_seed(seed)
  W = width or -(-(max(lens) + T) // page)
  P = B * W + extra_pages
  perm = torch.randperm(P, generator=g)[:B * W].view(B, W).to(torch.int32)
  kc = torch.full((P, KV, page, dh), fill, dtype=torch.float16)
  vc = kc.clone()
  for b in range(B):
    for j in range(lens[b]):
      kc[perm[b, j // page], :, j % page] = torch.randn(KV, dh, generator=g).half()
      vc[perm[b, j // page], :, j % page] = torch.randn(KV, dh, generator=g).half()
  qkv = torch.randn(B * T, (H + 2 * KV) * dh, generator=g)
  qkv[:, :H * dh] *= qscale
  from aneforge_b200.kernels import tree_layout
  rng = np.random.default_rng(seed)
  lay = [tree_layout([-1] + [int(rng.integers(max(0, t - 5), t)) for t in range(1, T)]) for _ in range(B)]
  if tree == "chain":
    lay = [tree_layout(list(range(-1, T - 1)))] * B
  depth = torch.tensor(np.stack([l[0] for l in lay]))
  mask = torch.tensor(np.stack([l[1] for l in lay]))
  d = dict(qkv=qkv, kc=kc, vc=vc, table=perm.contiguous(), lens=torch.tensor(lens, dtype=torch.int32), depth=depth, mask=mask)
  if rope:
    from aneforge_b200.llm import rope_tables
    c, s = rope_tables(W * page, dh, 10000.0)
    d.update(cos=torch.tensor(c), sin=torch.tensor(s))
  return {k: v.cuda() for k, v in d.items()}


def call(d, H, KV, dh, scale, **kw):
  from aneforge_b200 import kernels as K
  args = dict(mask=d["mask"], depth=d["depth"])
  args.update(kw)
  return K.attn_tree(d["qkv"], d["kc"], d["vc"], d["table"], d["lens"], d.get("cos"), d.get("sin"), H, KV, dh, scale, **args)


def reference(d, H, KV, dh, scale, nodes=None):
  """(out, bound) in 64 bits; d as it is before the call."""
  B, W = d["table"].shape
  T, page, G = d["qkv"].shape[0] // B, d["kc"].shape[2], H // KV
  table, lens = d["table"].cpu().tolist(), d["lens"].cpu().tolist()
  words = d["mask"].cpu().numpy().view(np.uint32)
  kc, vc, qkv = d["kc"].cpu().double().numpy(), d["vc"].cpu().double().numpy(), d["qkv"].cpu().numpy()
  out = np.zeros((B, T, H, dh))
  bound = np.full((B, T, H, dh), 2.0 ** -24)
  for b in range(B):
    n = lens[b]
    live = T if nodes is None else min(T, max(0, nodes[b]))
    x = qkv[b * T:b * T + live].reshape(live, H + 2 * KV, dh).astype(np.float32)
    qk = x[:, :H + KV]
    if "cos" in d:
      at = n + d["depth"][b, :live].cpu().numpy()
      c, s = d["cos"].cpu().float().numpy()[at][:, None], d["sin"].cpu().float().numpy()[at][:, None]
      rot = np.concatenate([-qk[..., dh // 2:], qk[..., :dh // 2]], -1)
      qk = qk * c + rot * s
    h16 = lambda a: a.astype(np.float16).astype(np.float64)
    q, k, v = h16(qk[:, :H]), h16(qk[:, H:]), h16(x[:, H + KV:])
    for h in range(KV):
      kk = np.stack([kc[table[b][j // page], h, j % page] for j in range(n)] + [k[t, h] for t in range(live)] or [np.zeros(dh)])
      vv = np.stack([vc[table[b][j // page], h, j % page] for j in range(n)] + [v[t, h] for t in range(live)] or [np.zeros(dh)])
      for t in range(live):
        see = list(range(n)) + [n + u for u in range(live) if words[b, t, u // 32] >> (u % 32) & 1]
        if not see:
          continue
        for g in range(G):
          sc = kk[see] @ q[t, h * G + g] * scale
          e = np.exp(sc - sc.max())
          w = e / e.sum()
          a = w @ np.abs(vv[see])
          out[b, t, h * G + g] = w @ vv[see]
          more = 2.0 ** -10 * (np.abs(kk[see]) @ np.abs(q[t, h * G + g])).max() * scale if "cos" in d else 0.0
          bound[b, t, h * G + g] += (2.0 ** -10 + 2.0 ** -12 + more) * a
  return out.reshape(B * T, H * dh), bound.reshape(B * T, H * dh)


def check(d, H, KV, dh, nodes=None, **kw):
  scale = dh ** -0.5
  ref, bound = reference(d, H, KV, dh, scale, nodes)
  before = d["kc"].clone(), d["vc"].clone()
  if nodes is not None:
    kw["nodes"] = torch.tensor(nodes, dtype=torch.int32).cuda()
  err = torch.zeros(1, dtype=torch.int32).cuda()
  out = call(d, H, KV, dh, scale, err=err, **kw).cpu().double().numpy()
  assert int(err) == 0
  assert np.isfinite(out).all()
  off = np.abs(out - ref) - bound
  assert (off <= 0).all(), f"{off.max()} over the bound at {np.unravel_index(off.argmax(), off.shape)}"
  # the nodes' rows are in the cache, every other row is as it was
  B, T, page = d["table"].shape[0], d["depth"].shape[1], d["kc"].shape[2]
  mine = torch.zeros(d["kc"].shape[0], page, dtype=torch.bool)
  for b in range(B):
    for t in range(T if nodes is None else min(T, max(0, nodes[b]))):
      j = int(d["lens"][b]) + t
      p = int(d["table"][b, j // page])
      mine[p, j % page] = True
      want = d["qkv"][b * T + t].view(H + 2 * KV, dh)[H + KV:].half()
      assert torch.equal(d["vc"][p, :, j % page], want)
      if "cos" not in d:
        assert torch.equal(d["kc"][p, :, j % page], d["qkv"][b * T + t].view(H + 2 * KV, dh)[H:H + KV].half())
  same = lambda a, b: torch.equal(torch.nan_to_num(a, nan=77.0), torch.nan_to_num(b, nan=77.0))
  keep = ~mine.cuda()
  for now, old in zip((d["kc"], d["vc"]), before):
    assert same(now.transpose(1, 2)[keep], old.transpose(1, 2)[keep])


@pytest.mark.parametrize("dh", [16, 32, 64, 128])
@pytest.mark.parametrize("H,KV", [(1, 1), (4, 1), (6, 2), (8, 8), (16, 2)])
def test_heads(dh, H, KV):
  check(setup(2, 5, H, KV, dh, [70, 3], 16, seed=dh + H), H, KV, dh)


@pytest.mark.parametrize("dh", [32, 64, 128])
@pytest.mark.parametrize("T", [1, 2, 8, 31, 32, 33, 64, 100])
def test_node_counts(dh, T):
  check(setup(2, T, 4, 1, dh, [150, 0], 32, seed=T), 4, 1, dh)


def test_most_nodes():
  check(setup(1, 256, 2, 1, 128, [40], 64, seed=9), 2, 1, 128)
  check(setup(1, 256, 2, 1, 64, [300], 64, seed=9), 2, 1, 64)


@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("n", [0, 1, 15, 16, 63, 64, 127, 128, 129, 255, 256, 600, 1500])
def test_prefix_lengths(dh, n):
  check(setup(1, 3, 8, 2, dh, [n], 64, seed=n), 8, 2, dh)


@pytest.mark.parametrize("dh", [32, 64, 128])
@pytest.mark.parametrize("page", [1, 5, 8, 16, 24, 37, 64, 100, 128, 256, 1000])
def test_page_sizes(dh, page):
  check(setup(2, 9, 4, 2, dh, [333, 130], page, seed=page), 4, 2, dh)


@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("rows", [340, 341, 512])
def test_one_page_for_each_sequence(dh, rows):
  """A cache of one block a sequence is a table of one page each."""
  check(setup(3, 7, 4, 1, dh, [333, 1, 200], rows, seed=rows), 4, 1, dh)


def test_ragged_batches():
  lens = [0, 5, 900, 128, 64, 1, 333, 2000]
  check(setup(8, 6, 8, 2, 128, lens, 16, seed=4), 8, 2, 128)
  check(setup(8, 6, 8, 2, 64, lens, 64, seed=5), 8, 2, 64)


@pytest.mark.parametrize("dh", [16, 64, 128])
def test_rope_and_chain(dh):
  d = setup(2, 6, 4, 2, dh, [90, 17], 16, seed=dh, rope=True, tree="chain")
  check(d, 4, 2, dh)
  again = call(d, 4, 2, dh, dh ** -0.5)
  alone = call(d, 4, 2, dh, dh ** -0.5, mask=None, depth=None)       # the defaults are a chain
  assert torch.equal(again, alone)
  check(setup(2, 6, 4, 2, dh, [90, 17], 16, seed=dh + 1, rope=True), 4, 2, dh)


@pytest.mark.parametrize("dh", [32, 64, 128])
def test_qk_norm(dh):
  """Per-head RMSNorm of q and k before RoPE, as the decode kernel forms it: f32 x / max(|x|, floor) * g."""
  d = setup(1, 4, 4, 2, dh, [50], 16, seed=2)
  g = torch.Generator().manual_seed(3)
  qn, kn = (torch.rand(dh, generator=g) + 0.5).half(), (torch.rand(dh, generator=g) + 0.5).half()
  x = d["qkv"].view(4, 8, dh)
  unit = lambda y, w: y / y.double().square().sum(-1, keepdim=True).sqrt().clamp(min=0.5).float() * w.float().cuda()
  e = dict(d, qkv=torch.cat([unit(x[:, :4], qn), unit(x[:, 4:6], kn), x[:, 6:]], 1).reshape(4, -1),
           kc=d["kc"].clone(), vc=d["vc"].clone())
  got = call(d, 4, 2, dh, 1.0, qn=qn.cuda(), kn=kn.cuda(), qn_floor=0.5, kn_floor=0.5)
  ref, bound = reference(e, 4, 2, dh, 1.0)
  # q and k can round the other way, as with RoPE: |q|, |k| <= 1.5, so a score moves by 2^-10 * 2.25 at most
  assert (np.abs(got.cpu().double().numpy() - ref) <= bound * 4).all()


def test_rows_that_see_nothing():
  for dh in (32, 64, 128):
    d = setup(3, 40, 4, 2, dh, [0, 130, 0], 16, seed=6)
    d["mask"][0, 7] = 0                                    # empty prefix, no node
    d["mask"][0, 0] = 0
    d["mask"][1] = 0                                       # the prefix only
    d["mask"][2] = 0
    check(d, 4, 2, dh)
    assert (call(d, 4, 2, dh, 1.0)[80:] == 0).all()


def test_live_nodes():
  for dh in (32, 64, 128):
    check(setup(4, 9, 4, 2, dh, [20, 130, 0, 64], 16, seed=8), 4, 2, dh, nodes=[9, 0, 3, 1])


@pytest.mark.parametrize("dh", [32, 64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_not_finite_nodes_stay_with_who_sees_them(dh, bad):
  d = setup(1, 12, 4, 2, dh, [140], 16, seed=10)
  d["mask"][:] = 1                                         # every node sees node 0 only
  d["mask"][0, 5] = 0b100001                               # and node 5 itself
  clean = call(dict(d, kc=d["kc"].clone(), vc=d["vc"].clone()), 4, 2, dh, 0.1)
  d["qkv"].view(12, 8, dh)[5, 4:] = bad                    # node 5's k and v
  out = call(d, 4, 2, dh, 0.1)
  keep = torch.arange(12) != 5
  assert torch.equal(out[keep], clean[keep]) or torch.allclose(out[keep].float(), clean[keep].float(), atol=2.0 ** -9)
  assert torch.isfinite(out[keep]).all() and not torch.isfinite(out[5]).any()


def test_large_scores():
  """One key outweighs all others by e^100s: the maximum is taken out before the exponential."""
  d = setup(1, 4, 4, 1, 128, [300], 64, seed=12, qscale=100.0)
  check(d, 4, 1, 128)
  d = setup(1, 4, 4, 1, 64, [300], 64, seed=12, qscale=100.0)
  check(d, 4, 1, 64)


def test_pages_of_a_pool_and_scratch_reuse():
  """K and V as views of a pool [layers, 2, P, ...], pages apart by a stride; one scratch for calls of other sizes."""
  from aneforge_b200 import kernels as K
  for dh in (64, 128):
    d = setup(2, 5, 4, 2, dh, [100, 31], 16, seed=13)
    P = d["kc"].shape[0]
    wide = torch.full((P, 2, 2, 2, 16, dh), float("nan"), dtype=torch.float16).cuda()
    wide[:, 1, 0], wide[:, 1, 1] = d["kc"], d["vc"]
    want = call(d, 4, 2, dh, 0.125)
    scr = K.attn_tree_scratch(8, 64, 4, 2, dh)
    for _ in range(3):
      got = call(dict(d, kc=wide[:, 1, 0], vc=wide[:, 1, 1]), 4, 2, dh, 0.125, scratch=scr)
      assert torch.equal(got, want)
    e = setup(8, 64, 4, 2, dh, [700] * 8, 16, seed=14)
    a = call(e, 4, 2, dh, 0.125, scratch=scr)
    b = call(e, 4, 2, dh, 0.125)
    assert torch.equal(a, b)
    assert torch.equal(call(d, 4, 2, dh, 0.125, scratch=scr), want)


def test_other_stream_and_repeat():
  d = setup(4, 16, 8, 2, 128, [1000, 50, 513, 2000], 64, seed=15)
  want = call(d, 8, 2, 128, 0.09)
  for _ in range(5):
    assert torch.equal(call(d, 8, 2, 128, 0.09), want)     # the same bits every time
  s = torch.cuda.Stream()
  s.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(s):
    x = dict(d, qkv=torch.zeros_like(d["qkv"]))
    x["qkv"].copy_(d["qkv"])
    got = call(x, 8, 2, 128, 0.09)
  s.synchronize()
  assert torch.equal(got, want)


def test_rows_without_a_page_are_reported():
  """A table that ends before the nodes: recorded, nothing outside the pool is touched, the rest is right."""
  for dh in (32, 64, 128):
    d = setup(2, 4, 4, 2, dh, [30, 20], 16, seed=16, width=3)
    d["table"][0, 2] = -1                                  # rows 32.. of sequence 0: nodes 2 and 3
    err = torch.zeros(1, dtype=torch.int32).cuda()
    out = call(d, 4, 2, dh, 0.1, err=err)
    assert int(err) == 2 and torch.isfinite(out[4:]).all()
    e = setup(2, 4, 4, 2, dh, [30, 20], 16, seed=16, width=3)
    assert torch.equal(out[4:], call(e, 4, 2, dh, 0.1)[4:])
    f = setup(2, 4, 4, 2, dh, [30, 20], 16, seed=16, width=2)   # the last two nodes of sequence 0 have no entry
    err.zero_()
    out = call(f, 4, 2, dh, 0.1, err=err)
    assert int(err) == 2 and torch.isfinite(out).all()


def test_matches_the_decode_step():
  """One node over pages gives what the decode attention gives over its own cache."""
  from aneforge_b200 import kernels as K
  from aneforge_b200.llm import rope_tables
  for dh, H, KV in ((128, 32, 8), (64, 4, 2)):
    M, n = 256, 200
    g = torch.Generator().manual_seed(dh)
    kc = torch.randn(1, KV, M, dh, generator=g).half().cuda()
    vc = torch.randn(1, KV, M, dh, generator=g).half().cuda()
    qkv = torch.randn(1, (H + 2 * KV) * dh, generator=g).cuda()
    c, s = (torch.tensor(t).cuda() for t in rope_tables(M, dh, 500000.0))
    pos = torch.tensor([n], dtype=torch.int32).cuda()
    k2, v2 = kc.clone(), vc.clone()
    want = K.attn_decode(qkv, k2, v2, pos, c, s, H, KV, dh, dh ** -0.5, n_split=4)
    got = K.attn_tree(qkv, kc, vc, torch.zeros(1, 1, dtype=torch.int32).cuda(), pos, c, s, H, KV, dh, dh ** -0.5)
    assert torch.equal(kc, k2) and torch.equal(vc, v2)
    # both within 2^-10 of the weighted |v| (at most 3 here) of the formula
    assert (got.float() - want.float()).abs().max() < 2 * 2.0 ** -10 * 3


@pytest.mark.parametrize("B,T,H,KV,dh,lens,page", [(2, 1, 8, 2, 128, [700, 0], 64), (3, 33, 8, 2, 64, [129, 1000, 5], 16),
                                                   (1, 70, 4, 1, 128, [3000], 64), (2, 5, 4, 2, 32, [40, 100], 8)])
def test_workspace_may_hold_anything(B, T, H, KV, dh, lens, page):
  """A workspace full of NaN, and one that another size has used before."""
  from aneforge_b200 import kernels as K
  outs = []
  for fill in (0, 255, None):
    scratch = K.attn_tree_scratch(B, T, H, KV, dh)
    if fill is not None:
      scratch.fill_(fill)
    else:
      scratch = K.attn_tree_scratch(4, 64, H, KV, dh) if T < 64 else K.attn_tree_scratch(B, 2 * T, H, KV, dh)
      big = setup(4, 17, H, KV, dh, [900, 64, 0, 333], page, seed=9)
      call(big, H, KV, dh, 0.1, scratch=scratch)
    d = setup(B, T, H, KV, dh, lens, page, seed=3)
    outs.append(call(d, H, KV, dh, 0.1, scratch=scratch))
  assert torch.isfinite(outs[0]).all()
  assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("dh,page", [(16, 16), (32, 5), (64, 5), (64, 16), (128, 7), (128, 64)])
def test_nan_stays_where_nothing_finite_is_seen(dh, page):
  """A softmax over NaN scores alone, or over a first tile of them, is NaN in every form, not zeros."""
  d = setup(2, 3, 4, 2, dh, [0, 50], page, seed=17)
  x = d["qkv"].view(2, 3, 8, dh)
  x[0, 0, 4:6] = float("nan")                              # sequence 0: node 0's k, the only key that it sees
  d["mask"][0, :, 0] = torch.tensor([1, 2, 4], dtype=torch.int32)
  x[1, 1, 0] = float("nan")                                # sequence 1: one query head of node 1
  out = call(d, 4, 2, dh, 0.1).view(2, 3, 4, dh)
  assert torch.isnan(out[0, 0]).all() and torch.isfinite(out[0, 1:]).all()
  assert torch.isnan(out[1, 1, 0]).all() and torch.isfinite(out[1, 1, 1:]).all() and torch.isfinite(out[1, ::2]).all()
  e = setup(1, 1, 4, 2, dh, [70], page, seed=18)
  p = int(e["table"][0, 0])
  for r in range(32):                                      # the first 32 keys are NaN, the others are not
    e["kc"][int(e["table"][0, r // page]), :, r % page] = float("nan")
  assert torch.isnan(call(e, 4, 2, dh, 0.1)).all()


@pytest.mark.parametrize("dh,page", [(32, 16), (64, 16), (128, 16), (128, 64), (64, 5)])
@pytest.mark.parametrize("T,H,KV", [(1, 4, 2), (9, 8, 2), (70, 4, 1), (40, 8, 1)])
def test_pages_missing_from_a_prefix(dh, page, T, H, KV):
  """Rows (and nodes) of pages that the table does not name, or names outside the pool, are left out and recorded."""
  d = setup(2, T, H, KV, dh, [700, 300], page, seed=19 + T)
  P, lost = d["kc"].shape[0], [2, 640 // page, 333 // page]
  full = d["table"].clone()
  d["table"][0, lost[0]], d["table"][0, lost[1]], d["table"][1, lost[2] - 40 // page] = -1, P, -5
  gone = [[j for j in range(700 + T) if j // page in lost[:2]], [j for j in range(300 + T) if j // page == lost[2] - 40 // page]]
  err = torch.zeros(1, dtype=torch.int32).cuda()
  scale = dh ** -0.5
  out = call(d, H, KV, dh, scale, err=err).double().cpu().view(2, T, H, dh)
  assert int(err) == 2
  kc, vc = d["kc"].double().cpu(), d["vc"].double().cpu()
  qkv, words = d["qkv"].cpu().view(2, T, H + 2 * KV, dh), d["mask"].cpu().numpy().view(np.uint32)
  for b, n in enumerate((700, 300)):
    rows = [j for j in range(n) if j not in set(gone[b])]
    at = [(int(full[b, j // page]), j % page) for j in rows]
    x = qkv[b].half().double()
    for h in range(KV):
      k = torch.cat([torch.stack([kc[p, h, r] for p, r in at]), x[:, H + h]])
      v = torch.cat([torch.stack([vc[p, h, r] for p, r in at]), x[:, H + KV + h]])
      sees = torch.ones(T, len(rows) + T, dtype=torch.bool)
      sees[:, len(rows):] = torch.tensor([[n + u not in gone[b] and bool(words[b, t, u // 32] >> (u % 32) & 1) for u in range(T)]
                                          for t in range(T)])
      for g in range(H // KV):
        w = torch.softmax((x[:, h * (H // KV) + g] @ k.T * scale).masked_fill(~sees, float("-inf")), 1)
        bound = (2.0 ** -10 + 2.0 ** -12) * (w @ v.abs()) + 2.0 ** -24
        assert ((out[b, :, h * (H // KV) + g] - w @ v).abs() <= bound).all()
