"""Engine on CPU: drafted tokens and shared prefixes change how many steps a generation takes, not what it says."""
import pytest
import torch

from nmoe_b200.serve import BlockPool, Engine, Sequence, ServeConfig, Transformer
from nmoe_b200.serve.engine import LookupDraft


@pytest.fixture(scope="module")
def model():
  torch.manual_seed(0)
  cfg = ServeConfig(num_hidden_layers=3, num_experts=4, experts_per_token=2, vocab_size=64, hidden_size=64, intermediate_size=64,
                    head_dim=16, num_attention_heads=4, num_key_value_heads=2, sliding_window=8, initial_context_length=64,
                    rope_scaling_factor=1.0, probe_layer=2, judge_layer=3)
  m = Transformer(cfg, dtype=torch.float32)
  m.init_weights(std=0.2)
  return m


PROMPTS = [[3, 1, 4, 1, 5, 9, 2, 6, 5, 3, 5, 8] * 2 + t for t in ([7, 7], [10, 11, 12, 13, 14], [3, 1, 4, 1])] + [[20, 21, 22]]


def test_lookup_proposes_what_followed():
  d = LookupDraft()
  t = [1, 2, 3, 4, 9, 1, 2, 3]
  assert d.propose(t, 4) == [4, 9, 1, 2] and d.propose(t, 1) == [4]
  assert d.propose(t + [8], 4) == []                           # nothing like (2, 3, 8) or (3, 8) before
  assert d.propose(t + [8, 2, 3], 5) == [8, 2, 3]              # the pair (2, 3), its latest place: index 7, then 8
  assert LookupDraft().propose([5], 3) == [] and LookupDraft().propose([5, 5, 5], 3) == [5]


def test_reserve_takes_only_free_blocks():
  pool = BlockPool(num_blocks=4, block_size=4)
  a, b = Sequence([1, 2, 3, 4, 5]), Sequence([6])
  pool.allocate(a)
  pool.allocate(b)
  assert pool.reserve(a, 2) == 2 and len(a.block_table) == 2   # fits its own block
  assert pool.reserve(a, 20) == 7 and len(a.block_table) == 3 and pool.n_free == 0
  assert pool.reserve(b, 9) == 3
  pool.release(a)
  pool.release(b)
  assert pool.n_free == 4


@pytest.mark.parametrize("k", [1, 3, 7])
@pytest.mark.parametrize("num_blocks", [None, 22])
def test_drafts_leave_greedy_output_as_it_is(model, k, num_blocks):
  plain = Engine(model, max_seq_len=80, max_batch=3, block_size=4).generate(PROMPTS, max_new_tokens=30, stop_tokens=[60])
  eng = Engine(model, max_seq_len=80, max_batch=3, block_size=4, num_blocks=num_blocks)
  seen = []
  out = eng.generate(PROMPTS, max_new_tokens=30, stop_tokens=[60], draft_tokens=k, on_token=lambda sid, t: seen.append(t))
  assert out == plain
  assert eng.steps["drafted"] > 0 and 0 < eng.steps["accepted"] <= eng.steps["drafted"]
  assert eng.pool.n_free == eng.num_blocks and not eng.drafts
  # a stop token ends a sequence where it stands: what was drafted behind it is not handed out
  assert len(seen) == sum(len(o) for o in out) + sum(1 for o in out if len(o) < 30)


def test_drafts_save_steps(model, monkeypatch):
  """With the right continuation proposed every time, 61 tokens take one prefill and ceil(60 / 5) steps."""
  plain = Engine(model, max_seq_len=200, max_batch=4, block_size=4).generate(PROMPTS, max_new_tokens=61)
  full = [p + o for p, o in zip(PROMPTS, plain)]
  monkeypatch.setattr(LookupDraft, "propose", lambda self, t, k: next(f for f in full if f[:len(t)] == t)[len(t):len(t) + k])
  eng = Engine(model, max_seq_len=200, max_batch=4, block_size=4)
  assert eng.generate(PROMPTS, max_new_tokens=61, draft_tokens=4) == plain
  assert eng.steps["decode"] == 12 and eng.steps["accepted"] == eng.steps["drafted"] == 4 * 48


def test_drafts_with_sampling(model):
  """top_k = 1 leaves one token: sampling has to say what greedy says.  With more, the same seed repeats itself."""
  greedy = Engine(model, max_seq_len=80, max_batch=4, block_size=4).generate(PROMPTS, max_new_tokens=20)
  run = lambda top_k, seed: Engine(model, max_seq_len=80, max_batch=4, block_size=4).generate(
    PROMPTS, max_new_tokens=20, temperature=0.7, top_k=top_k, generator=torch.Generator().manual_seed(seed), draft_tokens=3)
  assert run(1, 0) == greedy
  assert run(8, 1) == run(8, 1) and run(8, 1) != run(8, 2)
  assert all(len(o) == 20 for o in run(8, 3))


def test_a_shared_prefix_is_found_and_changes_nothing(model, monkeypatch):
  from nmoe_b200.serve import engine as E
  from nmoe_b200.serve import ops as S
  calls = []
  inner = S.shared_prefix_decode
  monkeypatch.setattr(S, "shared_prefix_decode", lambda q, k, v, t, c, n, *a: calls.append((len(q), n)) or inner(q, k, v, t, c, n, *a))
  run = lambda: Engine(model, max_seq_len=80, max_batch=3, block_size=4).generate(PROMPTS[:3], max_new_tokens=10)
  # the three are admitted together: none finds the other's blocks, so nothing is shared ...
  monkeypatch.setattr(E, "MIN_SHARED_TOKENS", 4)
  plain = run()
  assert not calls
  # ... until one has gone before
  eng = Engine(model, max_seq_len=80, max_batch=3, block_size=4)
  eng.generate(PROMPTS[:1], max_new_tokens=1)
  assert eng.generate(PROMPTS[:3], max_new_tokens=10) == plain
  assert calls and set(calls) == {(3, 24)}
  calls.clear()
  monkeypatch.setattr(E, "MIN_SHARED_TOKENS", 25)
  eng.generate(PROMPTS[:3], max_new_tokens=10)
  assert not calls


def test_draft_arguments():
  with pytest.raises(ValueError):
    Engine.generate(None, [], draft_tokens=-1)


def test_a_cache_view_can_be_used_again(model):
  """A prompt in chunks through one view whose slots, tables and lengths the caller moves on, then decode with it: every pass
  sees what the view holds when it is called."""
  from nmoe_b200.serve.model import CacheView
  cfg, bs, n = model.cfg, 4, 23
  shape = (cfg.num_hidden_layers, 8, bs, cfg.num_key_value_heads, cfg.head_dim)
  ids = torch.tensor([(7 * i + 3) % 64 for i in range(n + 1)])
  want = model(ids.view(1, -1), torch.arange(n + 1).view(1, -1))[0]
  view = CacheView(torch.zeros(shape), torch.zeros(shape), None, block_tables=torch.arange(8, dtype=torch.int32).view(1, 8), block_size=bs)
  at = 0
  for m in (8, 4, 11):
    view.slots, view.prefix_lens = torch.arange(at, at + m, dtype=torch.int32).view(1, m), [at]
    got = model(ids[at:at + m].view(1, m), torch.arange(at, at + m).view(1, m), cache=view)[0]
    assert torch.allclose(got, want[at:at + m], atol=1e-4)       # fp32 throughout, logits of order one
    at += m
  view.slots, view.context_lens = torch.tensor([n], dtype=torch.int32), torch.tensor([n + 1], dtype=torch.int32)
  got = model(ids[n:], torch.tensor([n]), cache=view, is_prefill=False)
  assert got.shape == (1, 64) and torch.allclose(got[0], want[n], atol=1e-4)


def test_a_cast_model_keeps_its_rotary_frequencies(model):
  """A model that is cast as a whole says what one of that type with the same weights says, at far positions too."""
  import copy
  ids, pos = torch.arange(20).view(1, 20), torch.arange(500, 520).view(1, 20)
  for dtype in (torch.bfloat16, torch.float64):
    want = Transformer(model.cfg, dtype=dtype)
    want.load_state_dict({k: v.to(dtype) for k, v in model.state_dict().items()})
    cast = copy.deepcopy(model).to(dtype)
    assert cast.embed.dtype == dtype and torch.equal(cast.inv_freq, model.inv_freq) and cast.inv_freq.dtype == torch.float32
    assert torch.equal(cast(ids, pos), want(ids, pos))
  assert torch.equal(copy.deepcopy(model).bfloat16().float().inv_freq, model.inv_freq)


@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_a_step_in_which_nobody_drafts_is_a_plain_one(model, monkeypatch, temperature):
  """With nothing proposed, draft_tokens changes neither the steps (a shared prefix is attended to once) nor what they say."""
  from nmoe_b200.serve import engine as E
  from nmoe_b200.serve import ops as S
  calls = {"shared_prefix_decode": 0, "paged_extend": 0}
  for name in calls:
    def count(*a, _inner=getattr(S, name), _name=name, **kw):
      calls[_name] += 1
      return _inner(*a, **kw)
    monkeypatch.setattr(S, name, count)
  monkeypatch.setattr(E, "MIN_SHARED_TOKENS", 4)

  def run(k, propose):
    monkeypatch.setattr(LookupDraft, "propose", propose)
    eng = Engine(model, max_seq_len=80, max_batch=3, block_size=4)
    eng.generate(PROMPTS[:1], max_new_tokens=1)
    calls.update(shared_prefix_decode=0, paged_extend=0)
    out = eng.generate(PROMPTS[:3], max_new_tokens=10, draft_tokens=k, temperature=temperature, generator=torch.Generator().manual_seed(1))
    return out, dict(calls), eng.steps

  none = lambda self, t, k: []
  plain, plain_calls, plain_steps = run(0, none)
  out, got, steps = run(4, none)
  assert got == plain_calls and got["shared_prefix_decode"] == 9 and steps == plain_steps      # one layer of three has no window
  assert temperature > 0 or out == plain
  # one drafting sequence is enough to make it a packed step
  out, got, _ = run(4, lambda self, t, k: [t[-1]][:k] if len(t) == 30 else [])
  assert got["paged_extend"] > plain_calls["paged_extend"] and 0 < got["shared_prefix_decode"] < 9
  assert temperature > 0 or out == plain


@pytest.mark.parametrize("hq,hkv,D,least", [(64, 8, 64, 128), (32, 4, 128, 128), (14, 2, 64, 128), (8, 2, 64, 256), (16, 16, 128, 256)])
def test_a_prefix_is_shared_where_that_is_faster(hq, hkv, D, least):
  from types import SimpleNamespace
  import numpy as np
  cfg = ServeConfig(num_attention_heads=hq, num_key_value_heads=hkv, head_dim=D)
  eng = SimpleNamespace(block_size=16, model=SimpleNamespace(cfg=cfg))
  for blocks in range(1, 40):
    tables = np.concatenate((np.tile(np.arange(blocks), (4, 1)), 100 + np.arange(8).reshape(4, 2)), 1).astype(np.int32)
    assert Engine._shared_len(eng, tables, blocks * 16 + 20) == (blocks * 16 if blocks * 16 >= least else 0)
  assert Engine._shared_len(eng, tables[:1], 40 * 16) == 0


def test_grade_prompts_asks_for_drafts_only_where_they_are_wanted():
  from nmoe_b200.data.score import ByteTokenizer, grade_prompts
  answer = '{"helpfulness": 3, "correctness": 4, "coherence": 2, "complexity": 1, "density": 0}'

  class Plain:                                      # an engine of one's own, with the arguments that generate has always had
    def generate(self, prompts, *, max_new_tokens, stop_tokens):
      return [list(answer.encode()) for _ in prompts]

  class Drafting:
    def generate(self, prompts, *, max_new_tokens, stop_tokens, draft_tokens):
      assert draft_tokens == 3
      return [list(answer.encode()) for _ in prompts]
  tok = ByteTokenizer()
  assert grade_prompts(Plain(), tok, ["a", "b"])[1]["scores"]["correctness"] == 4
  assert grade_prompts(Drafting(), tok, ["a"], draft_tokens=3)[0]["scores"]["helpfulness"] == 3


def test_a_refused_draft_count_leaves_earlier_labels(tmp_path):
  from nmoe_b200.data.cli import main
  out, docs = tmp_path / "labels.jsonl", tmp_path / "docs.jsonl"
  out.write_text("earlier labels\n")
  docs.write_text('{"id": "a", "text": "x"}\n')
  with pytest.raises(SystemExit, match="draft-tokens"):
    main(["hydra-oracle-label", "--checkpoint", str(tmp_path / "none"), "--input", str(docs), "--output", str(out), "--draft-tokens", "-1"])
  assert out.read_text() == "earlier labels\n"
