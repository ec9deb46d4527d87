"""Token sampling on the device (`kernels.sample`) against the definition in 64 bits on the host.

The uniform number of a row is put in the middle of the interval that the 64-bit distribution gives a chosen token, so
the token has to be equal whenever that interval is wider than the rounding of the weights: fp32 quotient, difference
and exponential (a relative 2^-20 of a weight for |z| <= 64) and u itself (2^-24), floor to 2^-40 of the largest weight
for each of V tokens. The tests choose tokens whose interval is over 2^-17."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

NEG = float("-inf")


@pytest.fixture(scope="module", autouse=True)
def need_gpu():
  if not torch.cuda.is_available():
    pytest.skip("no CUDA device")


def distribution(l, temp, k=0, p=1.0, mp=0.0):
  """64-bit probabilities of the kept tokens of one row (fp32 values l)."""
  l = np.where(np.isnan(l), -np.inf, l.astype(np.float64))
  n = l.size
  with np.errstate(invalid="ignore", over="ignore"):
    z = l / temp
    e = np.where(l == l.max(), 1.0, np.exp(z - z.max()))
  alive = np.ones(n, bool)
  if 0 < k < n:
    alive &= l >= np.sort(l)[n - k]
  if 0 < p < 1:
    order = np.lexsort((np.arange(n), -np.where(alive, l, -np.inf)))
    m = np.where(alive, e, 0.0)[order]
    cum = np.cumsum(m)
    inside = np.zeros(n, bool)
    inside[order] = cum - m < p * cum[-1]
    alive &= inside
  alive &= e >= min(mp, 1.0)
  e = np.where(alive, e, 0.0)
  return e / e.sum()


def pick(prob, rng):
  """A likely token, and the uniform number in the middle of its interval."""
  wide = np.flatnonzero(prob > 2.0 ** -17)
  t = int(rng.choice(wide))
  cum = np.cumsum(prob)
  return t, np.float32(cum[t] - prob[t] / 2)


def run(l, u, **kw):
  from aneforge_b200 import kernels as K
  tok, logp = K.sample(l, torch.tensor(np.asarray(u, np.float32)).cuda(), **kw)
  return tok.cpu().numpy(), logp.cpu().numpy()


def check(l, sets, seed=0, dtype=torch.float32):
  """Rows l [R, V] (numpy, representable in dtype), a setting (temperature, top_k, top_p, min_p) for each."""
  rng = np.random.default_rng(seed)
  x = torch.tensor(l).to(dtype).cuda()
  lf = x.float().cpu().numpy()
  probs = [distribution(lf[r], *sets[r]) for r in range(len(sets))]
  want = [pick(p, rng) for p in probs]
  col = lambda i, dt: torch.tensor([s[i] for s in sets], dtype=dt).cuda()
  tok, logp = run(x, [w[1] for w in want], temperature=col(0, torch.float32), top_k=col(1, torch.int32),
                  top_p=col(2, torch.float32), min_p=col(3, torch.float32))
  assert tok.tolist() == [w[0] for w in want]
  ref = np.array([np.log(probs[r][want[r][0]]) for r in range(len(sets))])
  np.testing.assert_allclose(logp, ref, rtol=2.0 ** -18, atol=2.0 ** -18)


def rows(R, V, seed, spread=2.5):
  rng = np.random.default_rng(seed)
  l = rng.standard_normal((R, V)).astype(np.float32) * spread
  for r in range(R):
    l[r, rng.integers(0, V, min(V, 12))] += rng.random(min(V, 12)).astype(np.float32) * 9
  return l


# p and min_p are chosen as fp32 values, as the kernel gets them
SETS = [(1.0, 0, 1.0, 0.0), (0.7, 50, 1.0, 0.0), (1.0, 0, 0.875, 0.0), (1.3, 0, 1.0, 0.0625), (0.9, 40, 0.9375, 0.03125),
        (1.0, 1, 1.0, 0.0), (0.5, 1000, 0.5, 0.0), (2.0, 3, 0.25, 0.5)]


@pytest.mark.parametrize("V", [1, 2, 31, 257, 997, 4096, 32000, 50257, 128256, 300001])
def test_every_setting_over_the_sizes(V):
  check(rows(len(SETS), V, V), SETS, V)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("V", [5, 1000, 50257])
def test_sixteen_bit_rows_with_many_ties(dtype, V):
  check(rows(len(SETS), V, V), SETS, V, dtype)


@pytest.mark.parametrize("R", [1, 3, 40, 200])
def test_row_counts(R):
  check(rows(R, 3001, R), [SETS[r % len(SETS)] for r in range(R)], R)


@pytest.mark.parametrize("R", [1, 2, 9, 17, 37, 74, 75, 148, 149, 300])
def test_row_counts_of_a_whole_vocabulary(R):
  base = rows(8, 128256, 5)
  l = np.stack([np.roll(base[r % 8], 17 * r) for r in range(R)])
  check(l, [SETS[r % len(SETS)] for r in range(R)], R)


@pytest.mark.parametrize("V", [7, 1025, 20000, 128256])
def test_equal_logits(V):
  """All tokens tie: top-k keeps them all, the nucleus the first ceil(p V) of them."""
  l = np.full((3, V), -2.0, np.float32)
  n = int(np.ceil(0.5 * V))
  tok, logp = run(torch.tensor(l).cuda(), [1 - 2.0 ** -24, 1 - 2.0 ** -24, 0.0], top_k=torch.tensor([1, 0, 0], dtype=torch.int32).cuda(),
                  top_p=torch.tensor([1.0, 0.5, 0.5]).cuda())
  assert tok.tolist() == [V - 1, n - 1, 0]
  np.testing.assert_allclose(logp, -np.log([V, n, n]), rtol=2.0 ** -18, atol=2.0 ** -18)


@pytest.mark.parametrize("levels", [2, 5])
@pytest.mark.parametrize("V", [600, 30000])
def test_few_levels(V, levels):
  """Whole classes of ties: the nucleus ends inside one, cut by index."""
  rng = np.random.default_rng(V + levels)
  l = rng.integers(0, levels, (len(SETS), V)).astype(np.float32) * 0.5
  check(l, SETS, 1)


def test_greedy_takes_the_first_largest():
  l = rows(4, 5000, 3)
  l[0, 4321] = l[0, 77] = 50.0
  l[2] = -1.0
  l[3, 10] = 0.0
  l[3, :] = np.minimum(l[3], 0.0)
  l[3, 5] = -0.0                                           # -0 and +0 are equal: the first of them
  l[3, 6:] = -1.0
  l[3, :5] = -1.0
  tok, logp = run(torch.tensor(l).cuda(), [0.9] * 4, temperature=0.0)
  assert tok.tolist() == [int(np.argmax(r)) for r in l] and tok[3] == 5
  assert (logp == 0).all()


def test_masked_places():
  """Masks as -inf, as the type's lowest value, NaN and +inf."""
  low = float(np.finfo(np.float32).min)
  l = np.full((6, 3000), NEG, np.float32)
  l[0, 2999] = -7.0                                        # one token left
  l[1] = low
  l[1, [5, 6]] = 1.0                                       # the lowest value instead of -inf
  l[2] = np.nan
  l[2, 1234] = 0.5
  l[3, [3, 9, 2000]] = np.inf                              # +inf: only those, alike
  l[3, 4] = 3.0
  # row 4: nothing at all; row 5: only NaN
  l[5] = np.nan
  tok, logp = run(torch.tensor(l).cuda(), [0.5, 0.75, 0.3, 0.5, 0.5, 0.5], top_k=40, top_p=0.9375, min_p=0.125)
  assert tok.tolist() == [2999, 6, 1234, 9, -1, -1]
  np.testing.assert_allclose(logp[:4], [0, -np.log(2), 0, -np.log(3)], atol=2.0 ** -18)
  assert (logp[4:] == NEG).all()
  for kw in (dict(), dict(top_p=0.5), dict(top_k=7), dict(temperature=0.0)):
    tok, logp = run(torch.tensor(l[4:]).cuda(), [0.5, 0.5], **kw)
    assert tok.tolist() == [-1, -1] and (logp == NEG).all()


def test_ends_of_u_and_settings():
  l = rows(1, 4000, 11)
  x = torch.tensor(l).cuda()
  p = distribution(l[0], 1.0)
  one = 1 - 2.0 ** -24
  assert run(x, [0.0])[0][0] == 0                          # every token has some weight here
  assert run(x, [one])[0][0] == np.flatnonzero(np.cumsum(p) < 1 - 2.0 ** -23).max() + 1 or p[3990:].max() < 2.0 ** -20
  best = int(l[0].argmax())
  for kw in (dict(top_k=1), dict(top_p=1e-9), dict(min_p=1.0), dict(min_p=3.0), dict(temperature=1e-6)):
    for u in (0.0, 0.5, one, 1.0, -1.0, float("nan")):     # u outside [0, 1) takes the first or the last kept
      assert run(x, [u], **kw)[0][0] == best, (kw, u)
  same = run(x, [0.3])[0][0]
  for kw in (dict(top_k=4000), dict(top_k=-1), dict(top_k=1 << 30), dict(top_p=0.0), dict(top_p=1.5), dict(min_p=-1.0)):
    assert run(x, [0.3], **kw)[0][0] == same, kw


def test_strides_streams_and_outputs():
  from aneforge_b200 import kernels as K
  l = rows(5, 2000, 21)
  pad = torch.full((5, 2003), 99.0).cuda()
  pad[:, 1:2001] = torch.tensor(l).cuda()
  u = torch.tensor([0.1, 0.3, 0.5, 0.7, 0.9]).cuda()
  want, wl = K.sample(torch.tensor(l).cuda(), u, top_p=0.9, top_k=100)
  out = torch.empty(5, dtype=torch.int32).cuda(), torch.empty(5).cuda()
  got, gl = K.sample(pad[:, 1:2001], u, top_p=0.9, top_k=100, out=out)
  assert got is out[0] and torch.equal(got, want) and torch.equal(gl, wl)
  half = pad.half()
  a, _ = K.sample(half[:, 1:2001], u, top_p=0.9)
  b, _ = K.sample(half[:, 1:2001].contiguous(), u, top_p=0.9)
  assert torch.equal(a, b)
  s = torch.cuda.Stream()
  s.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(s):
    x = torch.zeros(5, 2000, device="cuda")
    x.copy_(pad[:, 1:2001])
    got, _ = K.sample(x, u, top_p=0.9, top_k=100)
  s.synchronize()
  assert torch.equal(got, want)
  assert K.sample(torch.empty(0, 10).cuda(), torch.empty(0).cuda())[0].shape == (0,)


def test_same_result_alone_and_in_a_batch():
  """A row's token and log-probability do not depend on the rows beside it."""
  from aneforge_b200 import kernels as K
  x = torch.tensor(rows(150, 40000, 31)).cuda()
  u = torch.rand(150, generator=torch.Generator().manual_seed(1)).cuda()
  for kw in (dict(), dict(top_p=0.9), dict(top_k=64, top_p=0.9, min_p=0.01)):
    tok, logp = K.sample(x, u, **kw)
    for r in (0, 77, 149):
      t, lp = K.sample(x[r:r + 1], u[r:r + 1], **kw)
      assert t[0] == tok[r] and lp[0] == logp[r]


def test_agrees_with_the_host_sampler():
  """`llm.sample_token` draws one number from numpy's generator and takes it through the same distribution."""
  from aneforge_b200.llm import sample_token
  l = rows(30, 3000, 41)
  for r in range(30):
    kw = [dict(temperature=0.8), dict(temperature=1.0, top_k=20), dict(temperature=1.2, top_p=0.875)][r % 3]
    np.random.seed(r)
    u = np.float32(np.random.random_sample())
    p = distribution(l[r], kw["temperature"], kw.get("top_k", 0), kw.get("top_p", 1.0))
    cum = np.cumsum(p)
    if np.abs(cum - float(u)).min() < 2.0 ** -19:           # on the edge between two tokens: either is right
      continue
    np.random.seed(r)
    host = sample_token(l[r], **kw)
    assert run(torch.tensor(l[r:r + 1]).cuda(), [u], **kw)[0][0] == host


@pytest.mark.parametrize("V,dtype", [(393217, torch.float32), (500001, torch.bfloat16)])
def test_rows_longer_than_a_clusters_registers(V, dtype):
  l = np.stack([rows(1, V, 40 + i, 3.0)[0] for i in range(4)])
  check(l, [(1.0, 0, 1.0, 0.0), (0.7, 50, 1.0, 0.0), (1.0, 0, 0.6, 0.0), (0.9, 1000, 0.8, 0.02)], seed=4, dtype=dtype)


@pytest.mark.parametrize("V,dtype", [(3, torch.float32), (700, torch.bfloat16), (5001, torch.float32), (50257, torch.float16),
                                     (128256, torch.float32)])
def test_many_rows_agree_with_few(V, dtype):
  """Rows and settings of every kind alone and many times over: another split of the work, the same tokens."""
  inf, nan = float("inf"), float("nan")
  rng = np.random.default_rng(V)
  l = np.stack([rows(1, V, 60 + i, 2.0 + i % 3)[0] for i in range(24)])
  l[1] = -inf
  l[2] = nan
  l[3, V // 2:] = -inf
  l[4, ::2] = nan
  l[5, V // 3] = inf
  l[6] = 0.25
  l[7] = np.round(l[7])
  l[8] = np.where(rng.random(V) < 0.5, -3.0, 1.0)
  l[9] = -3.0e38
  l[10, :] = -60.0
  l[10, V - 1] = 10.0
  l[11, [0, V - 1]] = inf
  sets = [(1.0, 0, 1.0, 0.0), (0.7, 40, 0.9, 0.0), (1.0, 0, 0.95, 0.0), (0.0, 0, 1.0, 0.0), (1.3, 0, 1.0, 0.02),
          (0.9, 1000, 0.99, 0.01), (1.0, 0, 0.3, 0.1), (1e-3, 0, 0.5, 0.0), (5.0, 400, 1.0, 0.0), (2.0, 0, 0.999999, 0.0),
          (1.0, 3000, 0.5, 0.0), (1.0, 20, 1.0, 1.0)]
  x = torch.tensor(l).to(dtype).cuda()
  for shift in range(3):
    pick = [sets[(r + 5 * shift) % len(sets)] for r in range(24)]
    u = rng.random(24).astype(np.float32)

    def go(reps):
      col = lambda i, dt: torch.tensor([s[i] for s in pick], dtype=dt).cuda().repeat(reps)
      return run(x.repeat(reps, 1), np.tile(u, reps), temperature=col(0, torch.float32), top_k=col(1, torch.int32),
                 top_p=col(2, torch.float32), min_p=col(3, torch.float32))

    tok, logp = go(1)
    toks, logps = go(8)
    assert toks.reshape(8, 24).tolist() == [tok.tolist()] * 8
    np.testing.assert_allclose(logps.reshape(8, 24), np.tile(logp, (8, 1)), rtol=2.0 ** -20, atol=2.0 ** -20)


@pytest.mark.parametrize("reps", [1, 24])                  # clusters; one block a row
@pytest.mark.parametrize("V,dtype", [(31, torch.float32), (3001, torch.bfloat16), (50257, torch.float32)])
def test_an_infinite_temperature_draws_evenly(V, dtype, reps):
  """Every token that is not masked weighs the same; a token past the row, or a masked one, is never drawn."""
  rng = np.random.default_rng(V)
  l = rows(5, V, 81)
  l[1, ::3] = NEG
  l[2, V // 2:] = NEG
  l[3, 1::2] = np.nan
  l[4, :] = NEG
  l[4, V - 1] = 3.0
  x = torch.tensor(l).to(dtype)
  lf = x.float().numpy()
  for k, p, mp in ((0, 1.0, 0.0), (7, 1.0, 0.0), (600, 1.0, 0.0), (0, 0.75, 0.0), (0, 1.0, 0.5), (20, 0.5, 0.25)):
    for scalar in (False, True):
      want = [pick(distribution(lf[r], 1e300, k, p, mp), rng) for r in range(5)]
      temp = 1e39 if scalar else torch.full((5 * reps,), float("inf")).cuda()        # 1e39 is infinite in 32 bits
      tok, logp = run(x.repeat(reps, 1).cuda(), [w[1] for w in want] * reps, temperature=temp, top_k=k, top_p=p, min_p=mp)
      assert tok.tolist() == [w[0] for w in want] * reps, (k, p, mp)
      ref = [np.log(distribution(lf[r], 1e300, k, p, mp)[want[r][0]]) for r in range(5)]
      np.testing.assert_allclose(logp, ref * reps, atol=2.0 ** -18)


@pytest.mark.parametrize("reps", [1, 24])                  # clusters; one block a row
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_temperatures_near_zero(dtype, reps):
  """Logits whose quotient or difference overflows: the largest takes all the weight, however it is chosen."""
  l = rows(5, 3001, 71)
  l[0] -= l[0].max() + 1.0                                 # the largest will be 0: 0 times an infinite scale is no distance
  l[1] -= l[1].max() + 1.0                                 # all quotients -inf
  l[2] += 8.0 - l[2].max()                                 # many quotients +inf
  l[3, 100:] = NEG
  l[4, ::2] = np.nan
  x = torch.tensor(l).to(dtype)
  x[0, 17], x[1, 3000], x[2, 0], x[3, 50], x[4, 7] = 0.0, -0.5, 20.0, 30.0, 25.0
  want = [17, 3000, 0, 50, 7]
  if dtype == torch.float32:
    x[0, 0], want[0] = 0.0, 0
    x[0, 17] = -1e-30
  x = x.repeat(reps, 1).cuda()
  n = 5 * reps
  for temp in (1e-45, 1e-39, 2e-38, 1e-36):
    for kw in (dict(), dict(top_k=40), dict(top_k=600), dict(min_p=0.25), dict(top_p=0.5), dict(top_k=40, top_p=0.5, min_p=0.1)):
      out = torch.full((n,), -7, dtype=torch.int32).cuda(), torch.full((n,), 5.0).cuda()
      tok, logp = run(x, np.tile(np.float32([0.0, 0.5, 0.9, 0.99, 0.2]), reps), temperature=torch.full((n,), temp).cuda(), out=out, **kw)
      assert tok.tolist() == want * reps, (temp, kw)
      assert (logp == 0).all(), (temp, kw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_longest_rows(dtype):
  """2^24 - 1 tokens that tie: sums just under 2^64."""
  V, one = (1 << 24) - 1, 1 - 2.0 ** -24
  x = torch.full((1, V + 3), 7.0, dtype=dtype, device="cuda")
  for l in (x[:, :V], x[:, 3:]):                           # on a 16-byte boundary, and off one
    for kw, n in ((dict(), V), (dict(top_p=0.5), 1 << 23), (dict(top_k=5), V), (dict(min_p=0.5), V)):
      for u, at in ((0.0, 0), (one, n - 1)):
        tok, logp = run(l, [u], **kw)
        assert tok.tolist() == [at], (kw, u)
        np.testing.assert_allclose(logp, -np.log(n), rtol=2.0 ** -18)


@pytest.mark.parametrize("reps", [1, 120])
def test_min_p_of_large_logits(reps):
  """z = l / temperature rounds to steps of 0.5 here, so tokens of other logits have the same z as the largest: they
  are as probable, and min-p keeps them however the row is split."""
  lmax, temp = np.float32(3000000.25), np.float32(0.7)
  near = lmax - np.float32(0.25) * np.arange(12, dtype=np.float32)
  z = near / temp
  as_good = int((z == z[0]).sum())
  assert as_good > 1 and z.dtype == np.float32
  l = np.full((1, 2000), 2.9e6, np.float32)
  l[0, 500:512] = near[::-1]
  first = 512 - as_good
  x = torch.tensor(l).cuda().repeat(reps, 1)
  tok, logp = run(x, [0.0] * reps, temperature=float(temp), min_p=1.0)
  assert tok.tolist() == [first] * reps
  np.testing.assert_allclose(logp, -np.log(as_good), atol=2.0 ** -18)


@pytest.mark.parametrize("reps", [1, 120])
@pytest.mark.parametrize("k", [40, 600])
def test_top_k_of_large_quotients(k, reps):
  """z in steps of 128: two logits whose quotients lie 68 apart round to one z, and are as probable."""
  temp = np.float32(1.752e-9)
  l = np.full((1, 2000), -5.0, np.float32)
  l[0, 901] = np.float32(1.9) + np.float32(2.0 ** -22)
  l[0, 900] = l[0, 901] - np.float32(2.0 ** -23)
  z = l[0, 900:902] / temp
  assert z[0] == z[1] and l[0, 900] < l[0, 901]
  x = torch.tensor(l).cuda().repeat(reps, 1)
  for u, at in ((0.0, 900), (0.75, 901)):
    tok, logp = run(x, [u] * reps, temperature=float(temp), top_k=k)
    assert tok.tolist() == [at] * reps
    np.testing.assert_allclose(logp, -np.log(2.0), rtol=2.0 ** -18)


@pytest.mark.parametrize("V", [4099, 50257])
def test_runs_of_heavy_tokens_among_light_ones(V):
  """Many rows: a warp queues the tokens that can be kept, 0 to 32 of each 32 places in every order of counts."""
  rng = np.random.default_rng(V)
  l = np.full((100, V), -30.0, np.float32)
  for r in range(100):
    i = 0
    while i < V:
      n = int(rng.integers(0, 33))
      at = i + rng.permutation(32)[:n]
      l[r, at[at < V]] = rng.random((at < V).sum()).astype(np.float32)
      i += 32
  check(l, [[(1.0, 0, 1.0, 0.25), (1.0, 0, 0.75, 0.0), (0.75, 0, 0.5, 0.5)][r % 3] for r in range(100)], V)
