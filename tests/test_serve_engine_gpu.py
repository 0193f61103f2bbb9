"""The serving engine on the GPU with its operators together: append, shared prefix, drafted tokens, verification."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def models():
  from nmoe_b200.serve import ServeConfig, Transformer
  cfg = ServeConfig(num_hidden_layers=3, num_experts=8, experts_per_token=2, vocab_size=512, hidden_size=256, intermediate_size=160,
                    head_dim=64, num_attention_heads=8, num_key_value_heads=2, sliding_window=16, initial_context_length=128,
                    rope_scaling_factor=1.0, probe_layer=2, judge_layer=3)
  mg = Transformer(cfg, dtype=torch.bfloat16, device=torch.device("cuda"), max_tokens=1024)
  mg.init_weights(std=0.05)
  mc = Transformer(cfg, dtype=torch.float32)
  mc.load_state_dict({k: v.float().cpu() for k, v in mg.state_dict().items()})
  yield mg, mc
  mg.rdep.close()


def _cos(a, b):
  return torch.nn.functional.cosine_similarity(a.float().cpu().flatten(), b.float().cpu().flatten(), dim=0).item()


def test_decode_behind_a_shared_prefix_tracks_the_fp32_model(models):
  from nmoe_b200.ops import tc_gemm as G
  from nmoe_b200.serve import Engine
  mg, mc = models
  g = torch.Generator().manual_seed(0)
  rubric = torch.randint(0, 512, (150,), generator=g).tolist()
  docs = [rubric + torch.randint(0, 512, (n,), generator=g).tolist() for n in (3, 40, 17, 90, 1)]
  eg, ec = Engine(mg, max_seq_len=320, max_batch=8), Engine(mc, max_seq_len=320, max_batch=8)
  for e in (eg, ec):                     # the rubric goes before, so that all five find its blocks
    e.generate([rubric], max_new_tokens=1)
    for d in docs:
      e.add(d, 6)
  lg, ids_g = eg.step()
  lc, ids_c = ec.step()
  assert eg.steps["cached_tokens"] == ec.steps["cached_tokens"] == 5 * 144
  assert _cos(lg, lc) > 0.97
  for _ in range(4):
    for sg, sc, t in zip(ids_g, ids_c, lc.argmax(-1).tolist()):
      eg.update(sg, t)
      ec.update(sc, t)
    lg, ids_g = eg.step()
    lc, ids_c = ec.step()
    assert _cos(lg, lc) > 0.95           # bf16 + MXFP8 experts vs fp32, a few near-tied routing decisions flip
  G.check_status()


def test_drafted_step_scores_like_single_steps(models):
  """Logits of a packed step over drafted tokens against the fp32 model's one-token steps over the same tokens."""
  from nmoe_b200.ops import tc_gemm as G
  from nmoe_b200.serve import Engine
  mg, mc = models
  g = torch.Generator().manual_seed(1)
  prompts = [torch.randint(0, 512, (n,), generator=g).tolist() * 2 for n in (9, 20, 33)]
  eg, ec = Engine(mg, max_seq_len=160, max_batch=4), Engine(mc, max_seq_len=160, max_batch=4)
  for e in (eg, ec):
    for p in prompts:
      e.add(p, 40)
    e.step()
    for s, p in zip(list(e.running), prompts):
      e.update(s.seq_id, p[0])           # the text starts over: the lookup finds what follows
  logits, tokens, cache, lens = eg._decode_drafts(list(eg.running), 3)
  assert lens == [4, 4, 4] and tokens.tolist() == sum((p[:4] for p in prompts), [])
  for j in range(4):
    lc, ids = ec.step()
    assert _cos(logits[j::4], lc) > 0.95
    for sid, p in zip(ids, prompts):
      ec.update(sid, p[j + 1])
  G.check_status()


@pytest.mark.parametrize("temperature,top_k", [(0.0, 0), (0.8, 0), (0.8, 5)])
def test_generate_with_drafts_and_a_shared_rubric(models, temperature, top_k, monkeypatch):
  """Whatever is proposed (here mostly nonsense, in numbers that change from step to step), generation goes through."""
  from nmoe_b200.ops import tc_gemm as G
  from nmoe_b200.serve import Engine
  from nmoe_b200.serve.engine import LookupDraft
  monkeypatch.setattr(LookupDraft, "propose", lambda self, t, k: [(7 * t[-1] + i) % 512 for i in range(min(k, len(t) % 5))])
  mg, _ = models
  g = torch.Generator().manual_seed(2)
  rubric = torch.randint(0, 512, (100,), generator=g).tolist()
  prompts = [rubric + rubric[b:b + 20] for b in range(6)]
  eng = Engine(mg, max_seq_len=256, max_batch=4, num_blocks=48)          # two admission waves, blocks run short
  gen = torch.Generator(device="cuda").manual_seed(3)
  out = eng.generate(prompts, max_new_tokens=30, temperature=temperature, top_k=top_k, generator=gen, draft_tokens=4)
  assert all(len(o) == 30 and all(0 <= t < 512 for t in o) for o in out)
  assert eng.steps["drafted"] > 0 and eng.pool.n_free == eng.num_blocks
  G.check_status()


def test_a_model_cast_as_a_whole_still_runs(models):
  """Module.to casts the rotary frequencies with the weights; the step takes them as they are."""
  mg, _ = models
  ids = torch.arange(24, device="cuda").view(1, 24)
  pos = torch.arange(24, device="cuda").view(1, 24)
  kept = mg.inv_freq
  try:
    mg.inv_freq = kept.bfloat16().float()
    want = mg(ids, pos)
    mg.inv_freq = kept.bfloat16()
    got = mg(ids, pos)
  finally:
    mg.inv_freq = kept
  assert torch.equal(got, want)


@pytest.mark.parametrize("draft_tokens", [0, 4])
def test_attention_forms_of_a_step_agree(models, draft_tokens, monkeypatch):
  """Every attention call that generation makes behind a shared rubric, with and without drafts, against paged_decode row by row on
  the same cache: equal up to one rounding of each, on layers with and without a window."""
  from nmoe_b200.ops import tc_gemm as G
  from nmoe_b200.serve import Engine
  from nmoe_b200.serve import ops as S
  from nmoe_b200.serve.engine import LookupDraft
  monkeypatch.setattr(LookupDraft, "propose", lambda self, t, k: t[-2:][:k] if len(t) % 3 else [])
  seen = {"shared_prefix_decode": 0, "paged_extend": 0}

  def check(o, q, kc, vc, tables, ctx, sinks, scale, window):
    ref = S.paged_decode(q, kc, vc, tables, ctx, sinks, scale, window).double()
    # two roundings to bf16, 2^-8 of the value each, and what the fp32 sums may leave of values of order one
    assert ((o.double() - ref).abs() <= 2.0 ** -7 * 1.01 * ref.abs() + 2.0 ** -14).all()

  inner_s, inner_e = S.shared_prefix_decode, S.paged_extend
  def shared(q, kc, vc, tables, ctx, n, sinks, scale, window=0):
    o = inner_s(q, kc, vc, tables, ctx, n, sinks, scale, window)
    check(o, q, kc, vc, tables, ctx, sinks, scale, window)
    seen["shared_prefix_decode"] += 1
    return o
  def extend(q, kc, vc, tables, ctx, starts, lens, sinks, scale, window=0, **kw):
    o = inner_e(q, kc, vc, tables, ctx, starts, lens, sinks, scale, window, **kw)
    if kw["max_q_len"] <= 5:                       # a step, not a prompt: each token as a sequence of its own
      rows = torch.repeat_interleave(torch.arange(len(lens), device=lens.device), lens.long())
      at = torch.arange(len(rows), device=lens.device) - starts[rows]
      check(o, q, kc, vc, tables[rows].contiguous(), (ctx[rows] - lens[rows] + 1 + at).int(), sinks, scale, window)
      seen["paged_extend"] += 1
    return o
  monkeypatch.setattr(S, "shared_prefix_decode", shared)
  monkeypatch.setattr(S, "paged_extend", extend)
  mg, _ = models
  g = torch.Generator().manual_seed(4)
  rubric = torch.randint(0, 512, (300,), generator=g).tolist()
  eng = Engine(mg, max_seq_len=400, max_batch=8)
  eng.generate([rubric], max_new_tokens=1)
  out = eng.generate([rubric + torch.randint(0, 512, (n,), generator=g).tolist() for n in (3, 40, 17, 39)], max_new_tokens=12, draft_tokens=draft_tokens)
  assert all(len(o) == 12 for o in out) and seen["shared_prefix_decode"] > 0 and (seen["paged_extend"] > 0) == (draft_tokens > 0)
  G.check_status()
