"""Forking, reserving, freeing and compacting sequences of a paged cache (`kernels.kv_*`) against a model in Python:
whole numbers and moved rows, so everything has to be equal."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def need_gpu():
  if not torch.cuda.is_available():
    pytest.skip("no CUDA device")


class Model:
  """The same bookkeeping, one step after another."""

  def __init__(self, L, P, KV, page, dh, S, W, seed=0):
    rng = np.random.default_rng(seed)
    self.pool = rng.standard_normal((L, 2, P, KV, page, dh)).astype(np.float16)
    self.table, self.lens, self.refs = np.full((S, W), -1, np.int32), np.zeros(S, np.int32), np.zeros(P, np.int32)
    self.page, self.W = page, W

  def free(self, slots, keep=None):
    for i, s in enumerate(slots):
      k = 0 if keep is None else min(max(keep[i], 0), self.lens[s])
      for w in range(-(-k // self.page), self.W):
        if self.table[s, w] >= 0:
          self.refs[self.table[s, w]] -= 1
          self.table[s, w] = -1
      self.lens[s] = k

  def fork(self, src, dst):
    self.free(dst)
    for a, b in zip(src, dst):
      for w in range(-(-int(self.lens[a]) // self.page)):
        self.table[b, w] = self.table[a, w]
        if self.table[a, w] >= 0:
          self.refs[self.table[a, w]] += 1
      self.lens[b] = self.lens[a]

  def reserve(self, slots, rows):
    free = iter(np.flatnonzero(self.refs == 0).tolist())
    for s, r in zip(slots, rows):
      n = int(self.lens[s])
      for w in range(n // self.page, -(-(n + r) // self.page) if r else 0):
        p = self.table[s, w]
        if p < 0:
          self.table[s, w] = q = next(free)
          self.refs[q] = 1
        elif self.refs[p] > 1:
          self.table[s, w] = q = next(free)
          self.refs[q] = 1
          self.refs[p] -= 1
          self.pool[:, :, q, :, :n % self.page] = self.pool[:, :, p, :, :n % self.page]

  def compact(self, slots, path, n):
    for i, s in enumerate(slots):
      for j in range(n[i]):
        a, b = int(self.lens[s]) + path[i][j], int(self.lens[s]) + j
        self.pool[:, :, self.table[s, b // self.page], :, b % self.page] = \
          self.pool[:, :, self.table[s, a // self.page], :, a % self.page]
      self.lens[s] += n[i]


class Device:
  def __init__(self, m):
    t = lambda a: torch.tensor(a).cuda()
    self.pool, self.table, self.lens, self.refs = t(m.pool), t(m.table), t(m.lens), t(m.refs)
    self.err, self.page = torch.zeros(1, dtype=torch.int32).cuda(), m.page

  def i(self, v):
    return torch.tensor(np.asarray(v, np.int32).reshape(np.shape(v))).cuda()

  def free(self, slots, keep=None):
    from aneforge_b200 import kernels as K
    K.kv_free(self.table, self.lens, self.refs, self.i(slots), self.page, None if keep is None else self.i(keep), err=self.err)

  def fork(self, src, dst):
    from aneforge_b200 import kernels as K
    K.kv_fork(self.table, self.lens, self.refs, self.i(src), self.i(dst), self.page, err=self.err)

  def reserve(self, slots, rows):
    from aneforge_b200 import kernels as K
    K.kv_reserve(self.pool, self.table, self.lens, self.refs, self.i(slots), self.i(rows), err=self.err)

  def compact(self, slots, path, n):
    from aneforge_b200 import kernels as K
    self.lens = K.kv_compact(self.pool, self.table, self.lens, self.i(slots), self.i(path), self.i(n), err=self.err)

  def same(self, m):
    assert np.array_equal(self.table.cpu().numpy(), m.table)
    assert np.array_equal(self.lens.cpu().numpy(), m.lens)
    assert np.array_equal(self.refs.cpu().numpy(), m.refs)
    assert np.array_equal(self.pool.cpu().numpy().view(np.uint16), m.pool.view(np.uint16))
    assert int(self.err) == 0


@pytest.mark.parametrize("page", [1, 3, 16, 64])
@pytest.mark.parametrize("KV,dh", [(1, 8), (2, 64), (3, 128)])
def test_a_life_of_sequences(page, KV, dh):
  """Random steps as a server takes them."""
  rng = np.random.default_rng(page * 100 + dh)
  S, W = 12, 6 + 40 // page
  m = Model(2, S * W + 5, KV, page, dh, S, W, page)
  d = Device(m)
  for step in range(60):
    k = int(rng.integers(1, 7))
    slots = rng.permutation(S)[:k].tolist()
    room = [int(W * page - m.lens[s]) for s in slots]
    what = step % 4 if step < 8 else int(rng.integers(0, 5))
    if what == 0:                                          # grow, and fill what was reserved
      rows = [int(rng.integers(0, min(r, 25) + 1)) for r in room]
      for x in (m, d):
        x.reserve(slots, rows)
      m.lens[slots] += np.array(rows, np.int32)
      d.lens = torch.tensor(m.lens).cuda()
    elif what == 1:
      T = 12
      ok = [i for i, r in enumerate(room) if r >= T]
      slots = [slots[i] for i in ok]
      if not slots:
        continue
      for x in (m, d):
        x.reserve(slots, [T] * len(slots))
      path = [sorted(rng.permutation(T)[:5].tolist()) for _ in slots]
      n = [int(rng.integers(0, 6)) for _ in slots]
      for x in (m, d):
        x.compact(slots, path, n)
    elif what == 2:
      half = len(slots) // 2
      if not half:
        continue
      src, dst = [slots[int(rng.integers(0, half))] for _ in slots[half:]], slots[half:]
      for x in (m, d):
        x.fork(src, dst)
    elif what == 3:
      keep = [int(rng.integers(0, m.lens[s] + 3)) for s in slots]
      for x in (m, d):
        x.free(slots, keep)
    else:
      for x in (m, d):
        x.free(slots[:2])
    d.same(m)
  held = np.zeros_like(m.refs)
  np.add.at(held, m.table[m.table >= 0], 1)
  assert np.array_equal(held, m.refs)


def test_many_slots_and_pages():
  S, W, page = 1024, 9, 16
  m = Model(1, 12000, 1, page, 8, S, W)
  d = Device(m)
  rng = np.random.default_rng(0)
  rows = rng.integers(0, W * page, S).tolist()
  for x in (m, d):
    x.reserve(list(range(S)), rows)
  m.lens[:] = rows
  d.lens = torch.tensor(m.lens).cuda()
  src, dst = list(range(500)), list(range(500, 1000))
  for x in (m, d):
    x.fork(src, dst)
    x.reserve(list(range(0, 1000, 3)), [1] * len(range(0, 1000, 3)))
  d.same(m)


def test_one_prompt_many_samples():
  """All sharers of a tail page but the last listed copy its rows."""
  m = Model(3, 200, 2, 16, 64, 40, 8)
  d = Device(m)
  for x in (m, d):
    x.reserve([0], [37])
  m.lens[0] = 37
  d.lens = torch.tensor(m.lens).cuda()
  for x in (m, d):
    x.fork([0] * 39, list(range(1, 40)))
  assert int(d.refs.max()) == 40
  for x in (m, d):
    x.reserve(list(range(40))[::-1], [5] * 40)
  d.same(m)
  assert d.table[:, 2].unique().numel() == 40 and d.table[:, 0].unique().numel() == 1


def test_too_few_pages_change_nothing():
  m = Model(1, 4, 1, 16, 8, 3, 4)
  d = Device(m)
  for x in (m, d):
    x.reserve([0, 1], [32, 16])
  d.same(m)
  d.reserve([2, 0], [16, 64])                              # three pages wanted, one is free
  assert int(d.err) == 4
  d.err.zero_()
  d.same(m)
  for x in (m, d):
    x.reserve([2], [16])
  d.same(m)


def test_refused_slots_and_paths():
  m = Model(1, 40, 1, 8, 8, 4, 4)
  d = Device(m)
  for x in (m, d):
    x.reserve([0, 1], [20, 20])
  m.lens[:2] = 10
  d.lens = torch.tensor(m.lens).cuda()

  def refused(code):
    assert int(d.err) == code
    d.err.zero_()
    d.same(m)

  d.reserve([4], [1]); refused(5)                          # no such slot
  d.reserve([-1], [1]); refused(5)
  d.reserve([3], [33]); refused(2)                         # more rows than the table has
  d.free([7]); refused(5)
  d.fork([0], [0]); refused(5)                             # onto itself
  d.fork([9], [1]); refused(5)
  d.fork([0, 2], [2, 3]); m.free([]); assert int(d.err) == 5  # slot 2 is both: the pair that reads it is left out
  d.err.zero_(); m.fork([0], [2]); d.same(m)
  d.reserve([1, 1], [10, 30]); assert int(d.err) == 5      # the second mention is left out
  d.err.zero_(); m.reserve([1], [10]); d.same(m)
  for path, n in (([3, 2], 2), ([0, 0], 2), ([-1, 1], 2), ([1, 40], 2), ([0, 1], 3), ([0, 1], -1)):
    d.compact([0], [path], [n]); refused(5)
  d.compact([5], [[0, 1]], [1]); refused(5)
  d.compact([0], [[1, 9]], [2]); m.compact([0], [[1, 9]], [2]); d.same(m)


def test_nothing_to_do():
  m = Model(1, 4, 1, 16, 8, 3, 4)
  d = Device(m)
  for x in (m, d):
    x.reserve([], [])
    x.free([])
    x.fork([], [])
    x.reserve([1], [0])
  d.same(m)


def test_rows_past_32_bits():
  """A pool whose last pages lie more than 2^31 elements in."""
  if torch.cuda.get_device_properties(0).total_memory < 40 << 30:
    pytest.skip("needs 20 GB")
  P = 1100
  pool = torch.zeros((2, 2, P, 8, 64, 1024), dtype=torch.float16, device="cuda")     # 2.3e9 elements
  assert pool.numel() > 1 << 31
  from aneforge_b200 import kernels as K
  i = lambda *v: torch.tensor(v, dtype=torch.int32).cuda()
  table, lens, refs = i(P - 1, -1, P - 1, -1).view(2, 2), i(40, 40), torch.ones(P, dtype=torch.int32).cuda()
  refs[P - 1], refs[P - 2] = 2, 0
  pool[:, :, P - 1, :, :40] = torch.randn((2, 2, 8, 40, 1024), device="cuda").half()
  K.kv_reserve(pool, table, lens, refs, i(0, 1), i(9, 9))
  assert table.tolist() == [[P - 2, -1], [P - 1, -1]]
  assert torch.equal(pool[:, :, P - 2, :, :40], pool[:, :, P - 1, :, :40]) and bool((pool[:, :, P - 2, :, 40:] == 0).all())
  pool[:, :, P - 1, :, 47] = 3.0
  out = K.kv_compact(pool, table, lens, i(1), i(7).view(1, 1), i(1))
  assert out.tolist() == [40, 41] and bool((pool[:, :, P - 1, :, 40] == 3.0).all())


@pytest.mark.parametrize("KV,dh", [(1, 8), (8, 128)])
def test_compact_of_a_slot_listed_twice(KV, dh):
  """Only the first mention moves rows and counts, as for the other calls; the second one is recorded."""
  S, T = 300, 12
  m = Model(2, S * 2, KV, 16, dh, S, 2)
  d = Device(m)
  for x in (m, d):
    x.reserve(list(range(S)), [30] * S)
  m.lens[:] = 15
  d.lens = torch.tensor(m.lens).cuda()
  slots = list(range(S))
  path = [[1, 4, 7, 11]] * S
  for where in (1, 40, S - 1):                             # the same warp's, another's, another pass of the block's
    slots[where] = slots[0]
  n = [1 + i % 4 for i in range(S)]
  d.compact(slots, path, n)
  assert int(d.err) == 5
  d.err.zero_()
  ok = [i for i in range(S) if slots.index(slots[i]) == i]
  assert len(ok) == S - 3
  m.compact([slots[i] for i in ok], [path[i] for i in ok], [n[i] for i in ok])
  d.same(m)
  d.compact([2, 2], [[0, 3], [1, 2]], [2, 2])
  assert int(d.err) == 5
  d.err.zero_()
  m.compact([2], [[0, 3]], [2])
  d.same(m)


@pytest.mark.parametrize("page", [1, 8])
def test_lengths_and_reservations_outside_the_table(page):
  """A length under 0, and rows whose count passes 32 bits: refused like any that the table cannot hold."""
  most = (1 << 31) - 1
  m = Model(1, 64, 1, page, 8, 4, 64 // page)
  d = Device(m)
  for x in (m, d):
    x.reserve([0, 1], [20, 20])

  def at(*lens):
    m.lens[:] = lens
    d.lens = torch.tensor(m.lens).cuda()

  def refused(code):
    assert int(d.err) == code
    d.err.zero_()
    d.same(m)

  for n in (-1, -20, -most - 1):
    at(n, 10, 0, 0)
    d.reserve([0], [5]); refused(2)
    d.reserve([0], [most]); refused(2)
    d.reserve([0], [0]); d.same(m)
    d.compact([0], [[1, 2]], [2]); refused(5)
    d.reserve([0, 1], [5, 2])                              # the others get theirs
    m.reserve([1], [2]); refused(2)
  at(10, 10, most, 0)
  d.reserve([1], [most]); refused(2)
  d.reserve([2], [1]); refused(2)
  d.reserve([2], [most]); refused(2)
  at(-3, 10, 0, 0)
  d.free([0])
  m.lens[0] = 0; m.free([0]); d.same(m)
