"""Generation over a paged cache: many samples of one prompt (`paged.sample_generate`) and speculative decoding with
a drafted tree (`speculative.tree_generate`). At temperature 0 every token is the oracle's greedy token, or within
the runner's own tie margin of it; with a temperature the tokens are distributed as the model's own."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from oracle.model import Config, OracleModel, random_llama_weights         # noqa: E402
from tests.test_llm_gpu import teacher_forced_check, to_b200_cfg            # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def need_gpu():
  if not torch.cuda.is_available():
    pytest.skip("no CUDA device")


SHAPES = {
  "dh64": dict(dim=256, n_layers=2, n_heads=4, n_kv_heads=2, ffn_dim=512, vocab=512, head_dim=64),
  "dh128": dict(dim=512, n_layers=2, n_heads=8, n_kv_heads=2, ffn_dim=1024, vocab=1024, head_dim=128),
  "dh32_qknorm": dict(dim=128, n_layers=2, n_heads=4, n_kv_heads=4, ffn_dim=256, vocab=512, head_dim=32, qk_norm=True),
}


def _model(shape="dh64", seed=0, compress="int8"):
  from aneforge_b200.llm import LlamaPrefill
  cfg = Config(rope_base=10000.0, **SHAPES[shape])
  w = random_llama_weights(cfg, seed=seed, std=0.05)
  if cfg.qk_norm:
    rng = np.random.default_rng(seed + 100)
    for layer in w["layers"]:
      for k in ("q_norm", "k_norm"):
        layer[k] = rng.uniform(0.5, 1.5, cfg.dh).astype(np.float32)
  return cfg, w, LlamaPrefill(to_b200_cfg(cfg), w, compress=compress)


def _prompt(cfg, n, seed):
  return [int(t) for t in np.random.default_rng(seed).integers(0, cfg.vocab, n)]


@pytest.mark.parametrize("shape,compress,page,P", [("dh64", "int8", 64, 17), ("dh64", None, 16, 33), ("dh128", "int4", 8, 40),
                                                   ("dh128", "int8", 64, 64), ("dh32_qknorm", "int8", 5, 23)])
def test_greedy_samples_are_the_models_own(shape, compress, page, P):
  from aneforge_b200.paged import sample_generate
  cfg, w, m = _model(shape, compress=compress)
  prompt = _prompt(cfg, P, 3)
  st = {}
  outs = sample_generate(m, prompt, 3, 20, temperature=0.0, page=page, stats=st)
  assert all(o == outs[0] for o in outs)
  assert teacher_forced_check(OracleModel(cfg, w, compress, precision="device"), prompt, outs[0], P + 20) <= 2
  # the last token drawn has no row: P + 19 rows a sequence, the prompt's whole pages shared
  assert st["pages"] == P // page + 3 * (-(-(P + 19) // page) - P // page)
  stop = outs[0][7]
  first = outs[0].index(stop)
  assert sample_generate(m, prompt, 2, 20, temperature=0.0, page=page, eos_id=stop) == [outs[0][:first + 1]] * 2
  assert sample_generate(m, prompt, 1, 1, temperature=0.0) == [outs[0][:1]]
  assert sample_generate(m, prompt, 2, 0) == [[], []]
  m.release()


@pytest.mark.parametrize("kind", ["gpt2", "qwen3_moe", "gemma"])
def test_other_families(kind, tmp_path):
  from aneforge_b200 import llm
  from aneforge_b200.paged import sample_generate
  from aneforge_b200.speculative import tree_generate
  from tests.test_adapters_gpu import _oracle_cfg
  from tests.test_loaders_cpu import _tiny
  d, _ = _tiny(kind, tmp_path, hidden_size=256, intermediate_size=512, num_attention_heads=4, num_key_value_heads=2,
               head_dim=64, vocab_size=512, initializer_range=0.08)
  m = llm.from_pretrained(str(d), compress="int8")
  prompt = [int(t) for t in np.random.default_rng(3).integers(0, 512, 19)]
  om = OracleModel(_oracle_cfg(m.cfg), m.w, "int8", precision="device")
  for toks in (sample_generate(m, prompt, 2, 16, temperature=0.0)[1], tree_generate(m, m, prompt, 16, branches=(2, 2))):
    assert len(toks) == 16
    assert teacher_forced_check(om, prompt, toks, 48, n_check=16) <= 2
  m.release()


@pytest.mark.parametrize("shape,branches,draft_seed,page", [("dh64", (3, 2, 1), 1, 64), ("dh64", (1,), 1, 16),
                                                            ("dh128", (4, 3, 2), 2, 8), ("dh128", (1, 1, 1, 1), 0, 64),
                                                            ("dh64", (2, 2, 2, 2), 0, 16), ("dh32_qknorm", (2, 3), 0, 7)])
def test_tree_generate_is_greedy(shape, branches, draft_seed, page):
  from aneforge_b200.speculative import tree_generate
  cfg, w, target = _model(shape)
  _, _, draft = _model(shape, seed=draft_seed)
  prompt = _prompt(cfg, 21, 5)
  st, seen = {}, []
  toks = tree_generate(target, draft, prompt, 30, branches=branches, page=page, stats=st, on_token=seen.append)
  assert len(toks) == 30 and seen == toks
  assert teacher_forced_check(OracleModel(cfg, w, "int8", precision="device"), prompt, toks, 21 + 30) <= 2
  assert st["accepted"] + st["verify_steps"] + 1 >= 30
  if draft_seed == 0:                          # the draft is the target: whole paths are accepted
    assert st["verify_steps"] <= -(-29 // (len(branches) + 1)) + 2
  stop = toks[11]
  assert tree_generate(target, draft, prompt, 30, branches=branches, page=page, eos_id=stop) == toks[:toks.index(stop) + 1]
  target.release(); draft.release()


def test_tree_sampling_follows_the_target():
  """100 runs of three tokens, two candidates a step: eight sequences, counted against the product of the target's
  own probabilities, within five standard deviations."""
  from aneforge_b200.speculative import tree_generate
  cfg, _, target = _model()
  _, _, draft = _model(seed=4)
  prompt = _prompt(cfg, 9, 6)

  def two(ids):
    lg = target.prefill(ids)[0].astype(np.float64) / 0.9
    k = np.argsort(-lg)[:2]
    p = np.exp(lg[k] - lg[k[0]])
    return list(zip(k.tolist(), (p / p.sum()).tolist()))

  want = {(a, b, c): pa * pb * pc for a, pa in two(prompt) for b, pb in two(prompt + [a]) for c, pc in two(prompt + [a, b])}
  N, got = 100, {}
  for s in range(N):
    key = tuple(tree_generate(target, draft if s % 2 else target, prompt, 3, branches=(2, 1), temperature=0.9, top_k=2, seed=s))
    got[key] = got.get(key, 0) + 1
  assert set(got) <= set(want)
  for key, p in want.items():
    assert abs(got.get(key, 0) - N * p) <= 5 * np.sqrt(N * p * (1 - p)) + 1, (key, got.get(key, 0), N * p)
  a = tree_generate(target, draft, prompt, 12, temperature=0.9, seed=7)
  assert a == tree_generate(target, draft, prompt, 12, temperature=0.9, seed=7)
  target.release(); draft.release()


def test_samples_follow_the_logits_of_the_step():
  """Each drawn token is the one that its random number picks from the step's own logits (temperature 0.8)."""
  from aneforge_b200.paged import PagedKV, TreeStep
  cfg, _, m = _model()
  prompt, B = _prompt(cfg, 70, 8), 64
  kv = PagedKV(m.cfg, B, 80, device=m.device)
  step = TreeStep(m, kv, B, temperature=0.8)
  pre, real, _ = m._prefill_hidden(prompt)
  u = np.random.default_rng(1).random(B, np.float32)
  with torch.cuda.stream(step.stream):
    kv.seed(0, pre, real)
    kv.fork([0] * (B - 1), range(1, B))
    kv.reserve(range(B), [1] * B)
    step.tok.fill_(5)
    step.u.copy_(torch.from_numpy(u)[:, None])
    step.run()
    step.check()
    lg, tok, logp = (t.view(B, -1).cpu().numpy().astype(np.float64) for t in (step.logits, step.out, step.logp))
  # the same token after the same rows; 2^-9: fp16 rounding in two layers, and another cut of the sums
  assert np.abs(lg - lg[0]).max() <= 2.0 ** -9 * np.abs(lg).max()
  p = np.exp((lg - lg.max(1, keepdims=True)) / 0.8)
  p /= p.sum(1, keepdims=True)
  cum = np.cumsum(p, 1)
  for i in range(B):
    t = int(tok[i, 0])
    lo = cum[i, t - 1] if t else 0.0
    assert lo - 1e-5 <= u[i] <= cum[i, t] + 1e-5
    assert abs(logp[i, 0] - np.log(p[i, t])) < 1e-4
  step.release()
  m.release()


def test_refusals():
  from aneforge_b200.paged import PagedKV, TreeStep, sample_generate
  from aneforge_b200.speculative import tree_generate
  cfg, _, m = _model()
  _, _, other = _model("dh128")
  kv = PagedKV(m.cfg, 2, 64, pages=1, page=16, device=m.device)
  with pytest.raises(ValueError):
    PagedKV(m.cfg, 0, 64)
  with pytest.raises(ValueError):
    TreeStep(m, kv, 3)
  with pytest.raises(ValueError):
    TreeStep(m, kv, 1, [-1, 0], feed=True)
  with pytest.raises(ValueError):
    TreeStep(other, kv, 1)
  with pytest.raises(ValueError):
    TreeStep(m, kv, 1, [0])                    # a node cannot be its own parent
  with pytest.raises(ValueError):
    sample_generate(m, [], 2)
  with pytest.raises(ValueError):
    sample_generate(m, [cfg.vocab], 2)
  with pytest.raises(ValueError):
    tree_generate(m, other, [1, 2, 3])         # another vocabulary
  with pytest.raises(ValueError):
    tree_generate(m, m, [1, 2, 3], branches=(300,))
  with pytest.raises(ValueError):
    tree_generate(m, m, [1, 2, 3], branches=(0,))
  kv.reserve([0], [17])                        # two pages of a pool of one
  with pytest.raises(RuntimeError, match="exhausted"):
    kv.check()
  kv.check()
  kv.reserve([5], [1])
  with pytest.raises(RuntimeError, match="slot"):
    kv.check()
  m.release(); other.release()
