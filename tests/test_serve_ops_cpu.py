"""Operators of a serving step on CPU tensors: the plain statements against 64-bit definitions, and what is refused."""
import pytest
import torch

from nmoe_b200.serve import ops as S
from serve_oracle import attend, paged, rope, verify


def i32(x):
  return torch.tensor(x, dtype=torch.int32)


def _attention_case(window=0, dtype=torch.float32):
  g = torch.Generator().manual_seed(window)
  lens, ctx, starts = [1, 3, 0, 9], [5, 3, 40, 30], [9, 10, 13, 0]
  k, v, tables = paged(ctx, 8, 2, 16, g, dtype=dtype)
  q = torch.randn(15, 6, 16, generator=g).to(dtype)
  return q, k, v, tables, ctx, starts, lens, torch.randn(6, generator=g)


@pytest.mark.parametrize("window", [0, 4])
def test_paged_extend_plain(window):
  q, k, v, tables, ctx, starts, lens, sinks = _attention_case(window)
  want, _, owned = attend(q, k, v, tables, ctx, starts, lens, sinks, 0.25, window)
  out = S.paged_extend(q, k, v, tables, i32(ctx), i32(starts), i32(lens), sinks, 0.25, window)
  # fp32 throughout: a few hundred roundings of 2^-24 on values of order one
  assert (out.double() - want).abs().max() < 1e-5 and (out[~owned] == 0).all()
  keep = torch.full_like(q, 2.0)
  S.paged_extend(q, k, v, tables, i32(ctx), i32(starts), i32(lens), sinks, 0.25, window, out=keep)
  assert torch.equal(keep[owned], out[owned]) and (keep[~owned] == 2.0).all()


def test_a_nan_in_q_stays_in_its_row():
  q, k, v, tables, ctx, starts, lens, sinks = _attention_case()
  args = (k, v, tables, i32(ctx), i32(starts), i32(lens), sinks, 0.25)
  clean = S.paged_extend(q, *args)
  q[4, 1, 0] = float("nan")
  out = S.paged_extend(q, *args)
  assert out[4, 1].isnan().all()
  out[4, 1] = clean[4, 1]
  assert torch.equal(out, clean)


def test_shared_prefix_decode_plain_equals_paged_decode():
  g = torch.Generator().manual_seed(0)
  ctx = [21, 40, 0, 33, 12]
  k, v, tables = paged([max(c, 20) for c in ctx], 8, 2, 16, g, shared=20, dtype=torch.float32)
  q, sinks = torch.randn(5, 6, 16, generator=g), torch.randn(6, generator=g)
  out = S.shared_prefix_decode(q, k, v, tables, i32(ctx), 20, sinks, 0.25)
  ref = S.paged_decode(q, k, v, tables, i32(ctx), sinks, 0.25)
  assert torch.allclose(out, ref, atol=1e-5) and (out[2] == 0).all()


def test_rope_append_plain():
  g = torch.Generator().manual_seed(0)
  qkv, pos = torch.randn(7, 8 * 16, generator=g), torch.randint(0, 10_000_000, (7,), generator=g)
  inv = 10000.0 ** (-torch.arange(0, 16, 2).float() / 16)
  y, _, vv = rope(qkv, pos, inv, 1.2, 4, 2)
  kc, vc = torch.zeros(3, 4, 2, 16), torch.zeros(3, 4, 2, 16)
  q, k, v = S.rope_append(qkv, pos, inv, 1.2, 4, 2, kc, vc, i32([3, -1, 0, 11, -1, 5, 6]), need_kv=True)
  assert (torch.cat((q, k), 1).double() - y).abs().max() < 1e-5 and torch.equal(v.double(), vv)
  assert torch.equal(kc.view(-1, 2, 16)[[3, 0, 11, 5, 6]], k[[0, 2, 3, 5, 6]]) and int((vc.view(-1, 32) != 0).any(-1).sum()) == 5
  assert S.rope_append(qkv, pos, inv, 1.2, 4, 2)[1:] == (None, None)


@pytest.mark.parametrize("dist", [False, True])
def test_verify_draft_plain(dist):
  g = torch.Generator().manual_seed(4)
  lens = [1, 4, 0, 2, 6, 3] * 20
  N, V = sum(lens), 30
  starts = [sum(lens[:b]) for b in range(len(lens))]
  target, draft = torch.softmax(torch.randn(N, V, generator=g), -1), torch.softmax(torch.randn(N, V, generator=g), -1)
  tokens, u = torch.multinomial(draft, 1, generator=g).squeeze(1), torch.rand(N, generator=g)
  want, count = verify(target.tolist(), tokens.tolist(), u.double().tolist(), starts, lens, draft.tolist() if dist else None)
  out, n = S.verify_draft(target, tokens, u, i32(starts), i32(lens), draft if dist else None)
  assert out.tolist() == want and n.tolist() == count and 1 < max(count)


def test_refusals():
  q, k, v, tables, ctx, starts, lens, sinks = _attention_case()
  ok = dict(q=q, k_cache=k, v_cache=v, block_tables=tables, context_lens=i32(ctx), q_starts=i32(starts), q_lens=i32(lens), sinks=sinks,
            scale=0.25)
  S.paged_extend(**ok)
  for bad in (dict(q=q[0]), dict(q=q[:, :5]), dict(k_cache=k[:, :, :1]), dict(k_cache=k.transpose(1, 2)), dict(v_cache=v.half()),
              dict(block_tables=tables.long()), dict(block_tables=tables[:2]), dict(context_lens=torch.tensor(ctx)), dict(sinks=sinks[:3]),
              dict(q_starts=torch.tensor(starts)), dict(q_lens=i32(lens[:2])), dict(window=-1), dict(max_q_len=-1), dict(scale=0.0),
              dict(out=torch.zeros(3, 6, 16)), dict(out=q.transpose(0, 1).contiguous().transpose(0, 1))):
    with pytest.raises(ValueError):
      S.paged_extend(**{**ok, **bad})
  qd = q[:4]
  ok = dict(q=qd, k_cache=k, v_cache=v, block_tables=tables, context_lens=i32(ctx), prefix_len=0, sinks=None, scale=0.25)
  S.shared_prefix_decode(**ok)
  for bad in (dict(q=q), dict(prefix_len=-1), dict(prefix_len=10_000), dict(window=-3), dict(context_lens=i32(ctx[:3]))):
    with pytest.raises(ValueError):
      S.shared_prefix_decode(**{**ok, **bad})
  qkv, pos, inv = torch.randn(3, 8 * 16), torch.arange(3), torch.ones(8)
  kc = torch.zeros(2, 4, 2, 16)
  ok = dict(qkv=qkv, positions=pos, inv_freq=inv, conc=1.0, n_heads=4, n_kv_heads=2, k_cache=kc, v_cache=kc.clone(), slots=i32([0, 1, -1]))
  S.rope_append(**ok)
  for bad in (dict(qkv=qkv[0]), dict(n_heads=5), dict(n_heads=0), dict(positions=pos.float()), dict(positions=pos[:2]), dict(inv_freq=inv[:4]),
              dict(inv_freq=inv.double()), dict(slots=None), dict(v_cache=None), dict(slots=torch.tensor([0, 1, 2])), dict(slots=i32([0])),
              dict(k_cache=kc.bfloat16(), v_cache=kc.bfloat16())):
    with pytest.raises(ValueError):
      S.rope_append(**{**ok, **bad})
  t = torch.rand(4, 9)
  ok = dict(target_probs=t, tokens=torch.zeros(4, dtype=torch.long), uniforms=torch.rand(4), q_starts=i32([0]), q_lens=i32([4]))
  S.verify_draft(**ok)
  for bad in (dict(target_probs=t[0]), dict(target_probs=t.double()), dict(target_probs=t[:, :0]), dict(tokens=torch.zeros(4)),
              dict(tokens=torch.zeros(3, dtype=torch.long)), dict(uniforms=torch.rand(4).double()), dict(uniforms=torch.rand(5)),
              dict(q_starts=torch.tensor([0])), dict(q_lens=i32([4, 1])), dict(draft_probs=t[:2]), dict(draft_probs=t.half()),
              dict(out=torch.zeros(4)), dict(out=i32([0, 0]))):
    with pytest.raises(ValueError):
      S.verify_draft(**{**ok, **bad})


def test_verify_draft_refuses_to_write_over_its_tokens():
  t, u, one = torch.rand(4, 9), torch.rand(4), i32([0])
  room = torch.zeros(9, dtype=torch.int32)
  for at in (0, 3, 4, 5):                           # tokens are room[4:8] (the last one has its own place)
    if at in (0,):
      S.verify_draft(t, room[4:8], u, one, i32([4]), out=room[0:4])
    else:
      with pytest.raises(ValueError, match="overlap"):
        S.verify_draft(t, room[4:8], u, one, i32([4]), out=room[at:at + 4])
  with pytest.raises(ValueError, match="overlap"):
    S.verify_draft(t, room[1:9:2], u, one, i32([4]), out=room[4:8])


def test_sizes_past_32_bits_are_refused():
  q, k, v, tables, ctx, starts, lens, sinks = _attention_case()
  S.paged_extend(q, k, v, tables, i32(ctx), i32(starts), i32(lens), sinks, 0.25, 2 ** 31 - 1)
  with pytest.raises(ValueError, match="32 bits"):
    S.paged_extend(q, k, v, tables, i32(ctx), i32(starts), i32(lens), sinks, 0.25, 2 ** 32 + 5)
  t = torch.rand(1, 1).expand(2, 2 ** 30 + 1)
  with pytest.raises(ValueError, match="2\\^30"):
    S.verify_draft(t, i32([0, 0]), torch.rand(2), i32([0]), i32([2]))


def test_status_record_made_in_inference_mode_can_be_reset():
  from nmoe_b200.ops import tc_gemm as G
  from nmoe_b200.ops._lib import NativeLibraryError
  dev = torch.device("cpu")
  G._STATUS.pop(dev, None)
  try:
    with torch.inference_mode():
      G.status_buffer(dev)
    G.status_buffer(dev)[0] = 2
    with pytest.raises(NativeLibraryError, match="code=2"):
      G.check_status(dev)
    G.check_status(dev)
  finally:
    G._STATUS.pop(dev, None)


def test_c_entries_refuse_sizes_that_are_none():
  """Empty and senseless sizes come back as numbers from the C entries (no GPU is asked for anything)."""
  import ctypes
  from nmoe_b200.ops import _lib as L
  if not L.available():
    pytest.skip("library not built")
  lib = L.lib()
  ws = lib.nmoe_paged_extend_workspace
  ws.restype = ctypes.c_longlong
  for n_rows, B, Hq, Hkv, D, bs, width, mq in ((0, 0, 8, 2, 64, 16, 3, 0), (3, 0, 8, 2, 64, 16, 3, 1), (3, 2, 8, 0, 64, 16, 3, 3), (3, 2, 8, 2, 64, 0, 3, 3),
                                               (3, 2, 1, 2, 64, 16, 3, 3), (3, 2, 8, 2, 64, 16, 0, 3)):
    assert ws(n_rows, B, Hq, Hkv, D, bs, width, mq, 0, 0) == 0
    assert lib.nmoe_paged_extend_launches(B, Hq, Hkv, D, bs, width, mq, 0, 0) in (0, 1)
  call = S._fn("nmoe_paged_extend", "plppplppppipiiiiiiiiiifiplpp")
  args = lambda **kw: [{**dict(q=0, qs=512, k=0, v=0, bt=0, bts=3, ctx=0, st=0, ln=0, sk=0, sf=0, out=0, n=3, B=2, Hq=8, Hkv=2, D=64, bs=16, nb=4, w=3, mq=3,
                               win=0, scale=1.0, pre=0, ws=0, wf=0, status=0, stream=0), **kw}[k] for k in
                       "q qs k v bt bts ctx st ln sk sf out n B Hq Hkv D bs nb w mq win scale pre ws wf status stream".split()]
  assert call(*args(B=0)) == 0 and call(*args(n=0)) == 0 and call(*args(mq=0)) == 0
  for bad, rc in ((dict(Hkv=0), -1), (dict(Hq=9), -1), (dict(Hq=1), -1), (dict(bs=0), -1), (dict(scale=0.0), -1), (dict(scale=float("nan")), -1), (dict(n=-1), -1),
                  (dict(D=96), -2), (dict(q=8), -3), (dict(out=2), -3), (dict(qs=100), -3), (dict(nb=1 << 30), -4), (dict(pre=5, st=16), -5),
                  (dict(w=100000, B=1), -6), (dict(pre=48), -6)):
    assert call(*args(**bad)) == rc, bad
  rope = S._fn("nmoe_rope_append", "plpipfppplpppiiiipp")
  r = lambda **kw: [{**dict(x=0, xs=768, pos=0, p64=1, inv=0, conc=1.0, slots=0, k=0, v=0, ns=0, q=0, ko=0, vo=0, n=1, hq=8, hkv=2, d=64, status=0, stream=0),
                     **kw}[k] for k in "x xs pos p64 inv conc slots k v ns q ko vo n hq hkv d status stream".split()]
  assert rope(*r(n=0)) == 0
  for bad, rc in ((dict(n=-1), -1), (dict(hq=0), -1), (dict(d=8), -1), (dict(d=520), -1), (dict(xs=100), -1), (dict(slots=16), -2), (dict(x=8), -3), (dict(k=4), -3)):
    assert rope(*r(**bad)) == rc, bad
  ver = S._fn("nmoe_verify_draft", "plplpippppp" + "iiipp")
  assert ver(0, 5, 0, 0, 0, 1, 0, 0, 0, 0, 0, 3, 0, 5, 0, 0) == 0
  assert ver(0, 5, 0, 0, 0, 1, 0, 0, 0, 0, 0, 3, 2, 0, 0, 0) == -1 and ver(0, 5, 0, 0, 0, 1, 0, 0, 0, 0, 0, -3, 2, 5, 0, 0) == -1


def test_contexts_below_zero_are_empty():
  q, k, v, tables, ctx, starts, lens, sinks = _attention_case()
  args = (k, v, tables, i32([ctx[0], 0, ctx[2], ctx[3]]), i32(starts), i32(lens), sinks, 0.25)
  want = S.paged_extend(q, *args)
  low = S.paged_extend(q, *args[:3], i32([ctx[0], -2 ** 31, ctx[2], ctx[3]]), *args[4:])
  assert torch.equal(low, want) and (low[10:13] == 0).all()
  out = S.shared_prefix_decode(q[:4], k, v, tables, i32([5, -2 ** 31, -1, 30]), 0, sinks, 0.25)
  assert torch.equal(out, S.shared_prefix_decode(q[:4], k, v, tables, i32([5, 0, 0, 30]), 0, sinks, 0.25)) and (out[1:3] == 0).all()


OUTSIDE = [-1, -8, 8, 2 ** 31 - 1, -2 ** 31, 2 ** 32 + 3, -2 ** 63]


@pytest.mark.parametrize("x", OUTSIDE)
@pytest.mark.parametrize("dist", [False, True])
def test_a_drafted_token_outside_the_vocabulary_fails(x, dist):
  """Whatever the row holds at either end: the token is not emitted, and the redraw takes the whole row."""
  target = torch.tensor([[0.25, 0, 0, 0, 0, 0, 0, 1.0]]).repeat(4, 1)
  draft = torch.zeros(4, 8) if dist else None
  for u, new in ((0.0, 0), (0.19, 0), (0.21, 7), (0.99, 7)):       # the first entry holds a fifth of the row
    for at in (1, 3):
      toks = torch.tensor([0, 7, 7, 7])
      toks[at] = x
      uni = torch.zeros(4)
      uni[0] = u
      out, n = S.verify_draft(target, toks, uni, i32([0]), i32([4]), draft)
      assert out.tolist() == [7] * (at - 1) + [new] + [-1] * (4 - at) and n.tolist() == [at]
      _reported(1011)


def _reported(where):
  from nmoe_b200.ops import tc_gemm as G
  from nmoe_b200.ops._lib import NativeLibraryError
  with pytest.raises(NativeLibraryError, match=f"code=2 where={where}"):
    G.check_status(torch.device("cpu"))


def test_paged_extend_plain_skips_and_reports_bad_pages_and_lengths():
  q, k, v, tables, ctx, starts, lens, sinks = _attention_case()
  call = lambda t=tables, c=ctx, s=starts, n=lens, k=k, v=v, **kw: S.paged_extend(q, k, v, t, i32(c), i32(s), i32(n), sinks, 0.25, **kw)
  good = call()
  # a page outside the cache counts as zeros: what a page of zeros gives
  bad, zk, zv = tables.clone(), torch.cat((k, torch.zeros_like(k[:1]))), torch.cat((v, torch.zeros_like(v[:1])))
  bad[3, 1] = len(k)
  zeros = call(t=bad, k=zk, v=zv)
  for page in (-1, len(k), -2 ** 31, 2 ** 31 - 1):
    bad[3, 1] = page
    assert torch.equal(call(t=bad), zeros)
    _reported(1022)
  # a context past its table is cut there
  assert torch.equal(call(t=tables[:, :4].contiguous(), c=[5, 3, 32, 90]), call(t=tables[:, :4].contiguous(), c=[5, 3, 32, 32]))
  _reported(1021)
  # rows outside q, and more of them than announced: the sequence is skipped, the others are not
  for s, n, kw in (([9, 10, 13, -1], lens, {}), ([9, 10, 13, 7], lens, {}), (starts, [1, 3, 0, -9], {}), (starts, lens, dict(max_q_len=8))):
    out = call(s=s, n=n, **kw)
    _reported(1020)
    assert torch.equal(out[9:], good[9:]) and (out[:9] == 0).all()


def test_paged_extend_plain_ignores_what_lies_before_the_window():
  q, k, v, tables, ctx, starts, lens, sinks = _attention_case(4)
  args = (i32(ctx), i32(starts), i32(lens), sinks, 0.25, 4)
  want = S.paged_extend(q, k, v, tables, *args)
  for t in range(ctx[3] - lens[3] - 4 + 1):
    k[tables[3, t // 8].long(), t % 8] = float("nan")
    v[tables[3, t // 8].long(), t % 8] = float("inf")
  assert torch.equal(S.paged_extend(q, k, v, tables, *args), want)
  tables[3, :2] = -1                                # pages that nobody looks at
  assert torch.equal(S.paged_extend(q, k, v, tables, *args), want)


def test_rope_append_plain_skips_and_reports_a_slot_past_the_cache():
  g = torch.Generator().manual_seed(0)
  qkv, pos, inv = torch.randn(4, 4 * 16, generator=g), torch.arange(4), torch.ones(8)
  kc, vc = torch.zeros(2, 4, 1, 16), torch.zeros(2, 4, 1, 16)
  q, k, v = S.rope_append(qkv, pos, inv, 1.0, 2, 1, kc, vc, i32([7, 8, 2 ** 31 - 1, 2]), need_kv=True)
  _reported(1000)
  assert int((vc != 0).any(-1).sum()) == 2 and torch.equal(kc.view(8, 16)[[7, 2]], k[[0, 3], 0]) and q.shape == (4, 2, 16)


def test_verify_draft_plain_skips_and_reports():
  target, u = torch.full((3, 8), 0.125), torch.zeros(3)
  for s0, n in ((1, 3), (-1, 2), (0, -1), (2, 2 ** 31 - 1), (4, 0)):
    out, count = S.verify_draft(target, torch.tensor([0, 1, 1]), u, i32([s0, 0]), i32([n, 1]))
    _reported(1010)
    assert count.tolist() == [0, 1] and out.tolist() == [0, -1, -1]
  out, count = S.verify_draft(target, torch.tensor([0, 8, 1]), u, i32([0]), i32([3]))
  _reported(1011)
  assert count.tolist() == [1] and out.tolist() == [0, -1, -1]


def test_paged_extend_writes_over_q_or_beside_it():
  q, k, v, tables, ctx, starts, lens, sinks = _attention_case()
  room = torch.zeros(40, 6, 16)
  call = lambda at, out: S.paged_extend(room[at:at + 15], k, v, tables, i32(ctx), i32(starts), i32(lens), sinks, 0.25, out=out)
  want = S.paged_extend(q, k, v, tables, i32(ctx), i32(starts), i32(lens), sinks, 0.25, out=q.clone())
  for at, to in ((10, 10), (0, 15), (20, 5)):
    room[at:at + 15] = q
    room[to:to + 15] = q                            # rows of no sequence stay
    assert torch.equal(call(at, room[to:to + 15]), want)
  for at, to in ((10, 11), (10, 9), (10, 24), (0, 14), (14, 0)):
    with pytest.raises(ValueError, match="overlap"):
      call(at, room[to:to + 15])
  wide = torch.zeros(15, 8, 16)                     # q inside a wider projection, out in the same memory
  with pytest.raises(ValueError, match="overlap"):
    S.paged_extend(wide[:, :6], k, v, tables, i32(ctx), i32(starts), i32(lens), sinks, 0.25, out=wide.view(-1)[:15 * 96].view(15, 6, 16))
