"""Operators of a serving step on the GPU against their definitions in 64 bits."""
import pytest
import torch

from serve_oracle import attend, paged, rope, verify

pytestmark = pytest.mark.gpu

DEV = "cuda"


def i32(x):
  return torch.tensor(x, dtype=torch.int32, device=DEV)


def within(got, want, bound, what=""):
  off = (got.double().cpu() - want).abs()
  bad = off > bound
  assert torch.isfinite(got).all(), what
  assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / bound).max()):.2f} bounds"


# ------------------------------------------------------------------------------------------------ rotate and append
@pytest.mark.parametrize("N,hq,hkv,D,bs,far,pos_dtype", [
  (1, 64, 8, 64, 16, 100, torch.int64), (5, 8, 2, 64, 8, 4096, torch.int32), (37, 14, 2, 64, 12, 200_000, torch.int64),
  (130, 32, 4, 128, 16, 2_000_000_000, torch.int64), (3, 1, 1, 16, 1, 50, torch.int32), (9, 3, 1, 80, 5, 1000, torch.int64),
  (600, 16, 16, 128, 64, 9000, torch.int64), (2500, 8, 2, 64, 16, 40000, torch.int64), (7, 2, 1, 512, 4, 70, torch.int32)])
def test_rope_append(N, hq, hkv, D, bs, far, pos_dtype):
  from nmoe_b200.serve import ops as S
  g = torch.Generator().manual_seed(N)
  qkv = torch.randn(N, (hq + 2 * hkv) * D, generator=g).bfloat16()
  pos = torch.randint(0, far, (N,), generator=g).to(pos_dtype)
  inv = (150000.0 ** (-torch.arange(0, D, 2).float() / D)).contiguous()
  blocks = (N + bs - 1) // bs + 2
  kc, vc = torch.randn(blocks, bs, hkv, D, generator=g).bfloat16(), torch.randn(blocks, bs, hkv, D, generator=g).bfloat16()
  slots = torch.randperm(blocks * bs, generator=g)[:N].int()
  slots[::3] = -1
  y, bound, v = rope(qkv, pos, inv, 1.3, hq, hkv)
  kd, vd = kc.to(DEV), vc.to(DEV)
  q, k, vo = S.rope_append(qkv.to(DEV), pos.to(DEV), inv.to(DEV), 1.3, hq, hkv, kd, vd, slots.to(DEV), need_kv=True)
  within(q, y[:, :hq], bound[:, :hq], "q")
  within(k, y[:, hq:], bound[:, hq:], "k")
  assert torch.equal(vo.cpu().double(), v)
  # the cache: live slots hold exactly the dense rows, every other slot what it held
  ek, ev = kc.view(-1, hkv, D).clone(), vc.view(-1, hkv, D).clone()
  live = slots >= 0
  ek[slots[live].long()], ev[slots[live].long()] = k.cpu()[live], vo.cpu()[live]
  assert torch.equal(kd.cpu().view(-1, hkv, D), ek) and torch.equal(vd.cpu().view(-1, hkv, D), ev)
  # no dense K/V wanted: the same q and the same cache
  kd2, vd2 = kc.to(DEV), vc.to(DEV)
  q2, k2, v2 = S.rope_append(qkv.to(DEV), pos.to(DEV), inv.to(DEV), 1.3, hq, hkv, kd2, vd2, slots.to(DEV))
  assert k2 is None and v2 is None and torch.equal(q2, q) and torch.equal(kd2, kd) and torch.equal(vd2, vd)
  # no cache at all, strided and misaligned rows
  wide = torch.zeros(N, qkv.size(1) + 24, dtype=torch.bfloat16, device=DEV)
  for off in (8, 3):
    wide[:, off:off + qkv.size(1)] = qkv.to(DEV)
    q3, k3, _ = S.rope_append(wide[:, off:off + qkv.size(1)], pos.to(DEV), inv.to(DEV), 1.3, hq, hkv, need_kv=True)
    assert torch.equal(q3, q) and torch.equal(k3, k)


def test_rope_append_skips_and_reports_a_slot_past_the_cache():
  from nmoe_b200.ops import tc_gemm as G
  from nmoe_b200.ops._lib import NativeLibraryError
  from nmoe_b200.serve import ops as S
  G.check_status()
  qkv = torch.randn(3, 4 * 64, device=DEV).bfloat16()
  kc = torch.zeros(2, 4, 1, 64, device=DEV, dtype=torch.bfloat16)
  vc = torch.zeros_like(kc)
  S.rope_append(qkv, torch.arange(3, device=DEV), torch.ones(32, device=DEV), 1.0, 2, 1, kc, vc, i32([7, 8, 2]))
  with pytest.raises(NativeLibraryError, match="code=2 where=1000"):
    G.check_status()
  assert int((vc != 0).any(-1).sum()) == 2


# ------------------------------------------------------------------------------------------------ attention
SHAPES = [(64, 8, 64, 16), (8, 2, 64, 8), (14, 2, 64, 12), (16, 16, 128, 16), (32, 4, 128, 64), (16, 1, 128, 5), (1, 1, 64, 1),
          (129, 1, 64, 16)]


@pytest.mark.parametrize("hq,hkv,D,bs", SHAPES)
@pytest.mark.parametrize("window,use_sinks", [(0, False), (0, True), (37, True), (1, False)])
def test_paged_extend(hq, hkv, D, bs, window, use_sinks):
  from nmoe_b200.serve import ops as S
  g = torch.Generator().manual_seed(hq * 1000 + window)
  lens = [1, 3, 0, 70, 2, 17, 1, 5]
  ctx = [1, 3, 40, 70, 1, 300, 129, 64]            # one new token alone, a whole prompt, none, more new tokens than context, ...
  if hq == 129:
    lens, ctx = lens[:3], ctx[:3]
  k, v, tables = paged(ctx, bs, hkv, D, g)
  # rows in an order of their own, with gaps
  starts, at = [0] * len(lens), 3
  for b in reversed(range(len(lens))):
    starts[b] = at
    at += lens[b] + b % 2
  N = at + 4
  q = torch.randn(N, hq, D, generator=g).bfloat16()
  sinks = torch.randn(hq, generator=g).bfloat16() if use_sinks else None
  want, bound, owned = attend(q, k, v, tables, ctx, starts, lens, sinks, D ** -0.5, window)
  args = (q.to(DEV), k.to(DEV), v.to(DEV), tables.to(DEV), i32(ctx), i32(starts), i32(lens), None if sinks is None else sinks.to(DEV),
          D ** -0.5, window)
  out = S.paged_extend(*args, max_q_len=max(lens))
  within(out.cpu()[owned], want[owned], bound[owned])
  assert (out.cpu()[~owned] == 0).all()
  keep = torch.full((N, hq, D), 3.0, dtype=torch.bfloat16, device=DEV)
  S.paged_extend(*args, out=keep)                   # no bound of the lengths: the same bits; rows of no sequence stay
  assert torch.equal(keep.cpu()[owned], out.cpu()[owned]) and (keep.cpu()[~owned] == 3.0).all()


@pytest.mark.parametrize("D,hq,hkv", [(64, 8, 1), (128, 4, 2)])
def test_paged_extend_long_context_and_prefill(D, hq, hkv):
  from nmoe_b200.serve import ops as S
  g = torch.Generator().manual_seed(D)
  lens, ctx = [1, 5, 333], [5003, 2500, 700]
  k, v, tables = paged(ctx, 16, hkv, D, g)
  starts = [0, 1, 6]
  q = (2 * torch.randn(339, hq, D, generator=g)).bfloat16()
  want, bound, _ = attend(q, k, v, tables, ctx, starts, lens, None, D ** -0.5, 0)
  out = S.paged_extend(q.to(DEV), k.to(DEV), v.to(DEV), tables.to(DEV), i32(ctx), i32(starts), i32(lens), None, D ** -0.5)
  within(out, want, bound)


@pytest.mark.parametrize("what", ["beyond", "before"])
def test_paged_extend_ignores_what_lies_outside(what):
  """NaN in the slots that no token may see: behind the context in its last page, before every window."""
  from nmoe_b200.serve import ops as S
  g = torch.Generator().manual_seed(5)
  lens, ctx, window = [3, 1], [90, 201], 20 if what == "before" else 0
  k, v, tables = paged(ctx, 16, 2, 64, g)
  clean = k.clone(), v.clone()
  for b in range(2):
    for t in (range(ctx[b], (ctx[b] + 15) // 16 * 16) if what == "beyond" else range(0, ctx[b] - lens[b] - window + 1)):
      k[tables[b, t // 16].long(), t % 16] = float("nan")
      v[tables[b, t // 16].long(), t % 16] = float("inf")
  q = torch.randn(4, 8, 64, generator=g).bfloat16()
  want, bound, _ = attend(q, *clean, tables, ctx, [0, 3], lens, None, 0.125, window)
  out = S.paged_extend(q.to(DEV), k.to(DEV), v.to(DEV), tables.to(DEV), i32(ctx), i32([0, 3]), i32(lens), None, 0.125, window)
  within(out, want, bound)


@pytest.mark.parametrize("bs", [8, 16, 32, 48, 64, 128, 192, 7])
@pytest.mark.parametrize("D,hq,hkv,window", [(64, 8, 2, 0), (128, 8, 2, 0), (64, 16, 2, 150)])
def test_paged_extend_page_sizes(bs, D, hq, hkv, window):
  """Pages that hold whole boxes of a block, or more than a block, or neither; many rows, few rows."""
  from nmoe_b200.serve import ops as S
  g = torch.Generator().manual_seed(bs)
  lens, ctx = [100, 3, 37], [500, 777, 65]
  k, v, tables = paged(ctx, bs, hkv, D, g)
  for b in range(3):                                # behind the context: nothing that may be read into a product
    for t in range(ctx[b], (ctx[b] + bs - 1) // bs * bs):
      k[tables[b, t // bs].long(), t % bs] = float("nan")
      v[tables[b, t // bs].long(), t % bs] = float("nan")
  starts = [0, 100, 103]
  q = torch.randn(140, hq, D, generator=g).bfloat16()
  want, bound, _ = attend(q, k, v, tables, ctx, starts, lens, None, D ** -0.5, window)
  out = S.paged_extend(q.to(DEV), k.to(DEV), v.to(DEV), tables.to(DEV), i32(ctx), i32(starts), i32(lens), None, D ** -0.5, window)
  within(out, want, bound)


@pytest.mark.parametrize("bs", [2, 4, 6, 12, 20, 24, 36, 80])
@pytest.mark.parametrize("D,window", [(64, 0), (128, 0), (64, 150)])
def test_paged_extend_pages_of_small_boxes(bs, D, window):
  """Pages of an even number of keys that is no power of two, or a small one: many rows, contexts that end inside a page."""
  from nmoe_b200.serve import ops as S
  g = torch.Generator().manual_seed(bs)
  lens, ctx = [100, 1, 37], [501, 777, 65]
  k, v, tables = paged(ctx, bs, 2, D, g)
  for b in range(3):
    for t in range(ctx[b], (ctx[b] + bs - 1) // bs * bs):
      k[tables[b, t // bs].long(), t % bs] = float("nan")
      v[tables[b, t // bs].long(), t % bs] = float("nan")
  q = torch.randn(138, 8, D, generator=g).bfloat16()
  want, bound, _ = attend(q, k, v, tables, ctx, [0, 100, 101], lens, None, D ** -0.5, window)
  out = S.paged_extend(q.to(DEV), k.to(DEV), v.to(DEV), tables.to(DEV), i32(ctx), i32([0, 100, 101]), i32(lens), None, D ** -0.5, window)
  within(out, want, bound)


def test_paged_extend_strided_operands():
  from nmoe_b200.serve import ops as S
  g = torch.Generator().manual_seed(8)
  lens, ctx = [2, 50], [300, 50]
  k, v, tables = paged(ctx, 16, 2, 64, g)
  q = torch.randn(52, 8, 64, generator=g).bfloat16()
  want, bound, _ = attend(q, k, v, tables, ctx, [0, 2], lens, None, 0.125, 0)
  kd, vd = k.to(DEV), v.to(DEV)
  rest = (i32(ctx), i32([0, 2]), i32(lens), None, 0.125)
  base = S.paged_extend(q.to(DEV), kd, vd, tables.to(DEV), *rest)
  within(base, want, bound)
  fused = torch.zeros(52, 12 * 64 + 8, dtype=torch.bfloat16, device=DEV)
  for off in (0, 8, 1):                             # q heads inside a fused projection; misaligned rows are copied once
    view = fused[:, off:off + 512].view(52, 8, 64) if off == 0 else fused[:, off:off + 512].unflatten(1, (8, 64))
    view.copy_(q)
    assert torch.equal(S.paged_extend(view, kd, vd, tables.to(DEV), *rest), base)
  heads_first = q.to(DEV).transpose(0, 1).contiguous().transpose(0, 1)
  assert torch.equal(S.paged_extend(heads_first, kd, vd, tables.to(DEV), *rest), base)
  wide = torch.zeros(2, tables.size(1) + 5, dtype=torch.int32, device=DEV)
  wide[:, :tables.size(1)] = tables.to(DEV)
  assert torch.equal(S.paged_extend(q.to(DEV), kd, vd, wide[:, :tables.size(1)], *rest), base)
  pairs = torch.stack((i32(ctx), i32(lens)), 1)     # every second number
  assert torch.equal(S.paged_extend(q.to(DEV), kd, vd, tables.to(DEV), pairs[:, 0], i32([0, 2]), pairs[:, 1], None, 0.125), base)


def test_empty_calls():
  from nmoe_b200.serve import ops as S
  kc = torch.zeros(2, 16, 2, 64, device=DEV, dtype=torch.bfloat16)
  none, t0 = i32([]), torch.zeros(0, 3, dtype=torch.int32, device=DEV)
  q = torch.zeros(0, 8, 64, device=DEV, dtype=torch.bfloat16)
  assert S.paged_extend(q, kc, kc, t0, none, none, none, None, 0.125).shape == (0, 8, 64)
  assert S.shared_prefix_decode(q, kc, kc, t0, none, 0, None, 0.125).shape == (0, 8, 64)
  q3 = torch.ones(3, 8, 64, device=DEV, dtype=torch.bfloat16)
  t = torch.zeros(2, 1, dtype=torch.int32, device=DEV)
  assert (S.paged_extend(q3, kc, kc, t, i32([0, 4]), i32([0, 3]), i32([0, 0]), None, 0.125) == 0).all()
  qq, k, v = S.rope_append(torch.zeros(0, 12 * 64, device=DEV, dtype=torch.bfloat16), torch.zeros(0, device=DEV, dtype=torch.long),
                           torch.ones(32, device=DEV), 1.0, 8, 2, kc, kc.clone(), none, need_kv=True)
  assert qq.shape == (0, 8, 64) and k.shape == v.shape == (0, 2, 64)
  out, n = S.verify_draft(torch.zeros(0, 5, device=DEV), torch.zeros(0, device=DEV, dtype=torch.long), torch.zeros(0, device=DEV), i32([0]), i32([0]))
  assert out.numel() == 0 and n.tolist() == [0]


def test_paged_extend_large_scores_and_extreme_sinks():
  from nmoe_b200.serve import ops as S
  g = torch.Generator().manual_seed(6)
  lens, ctx = [4, 40], [400, 40]
  k, v, tables = paged(ctx, 16, 1, 64, g)
  k = (k.float() * 30).bfloat16()                   # scores of some hundreds that grow and fall along the context
  q = (torch.randn(44, 4, 64, generator=g) * 4).bfloat16()
  sinks = torch.tensor([float("-inf"), -1e30, 60.0, 3000.0])
  want, bound, _ = attend(q, k, v, tables, ctx, [0, 4], lens, sinks, 0.125, 0)
  out = S.paged_extend(q.to(DEV), k.to(DEV), v.to(DEV), tables.to(DEV), i32(ctx), i32([0, 4]), i32(lens), sinks.to(DEV), 0.125)
  within(out, want, bound)


@pytest.mark.parametrize("lens,ctx,D", [([5], [700], 64), ([1], [30_000], 64), ([1] * 9, [90] * 9, 128), ([140], [900], 64),
                                        ([90], [140], 128), ([60], [9000], 128), ([3, 0, 2], [3, 0, 50], 64)])
@pytest.mark.parametrize("window", [0, 50])
def test_paged_extend_a_nan_in_q_stays_in_its_row(lens, ctx, D, window):
  from nmoe_b200.serve import ops as S
  g = torch.Generator().manual_seed(D)
  k, v, tables = paged(ctx, 16, 2, D, g)
  starts = [sum(lens[:b]) for b in range(len(lens))]
  q = torch.randn(sum(lens), 8, D, generator=g).bfloat16()
  want, bound, _ = attend(q, k, v, tables, ctx, starts, lens, None, D ** -0.5, window)
  r = sum(lens) // 2
  q[r, 2, 7], q[r, 5] = float("nan"), float("inf")
  out = S.paged_extend(q.to(DEV), k.to(DEV), v.to(DEV), tables.to(DEV), i32(ctx), i32(starts), i32(lens), None, D ** -0.5, window).cpu()
  assert out[r, [2, 5]].isnan().all()
  out[r, [2, 5]] = want[r, [2, 5]].bfloat16()
  within(out, want, bound)


def test_shared_prefix_decode_a_nan_in_q_stays_in_its_row():
  from nmoe_b200.serve import ops as S
  g = torch.Generator().manual_seed(1)
  for B, hq in ((3, 8), (40, 8)):
    ctx = [200 + 3 * b for b in range(B)]
    k, v, tables = paged(ctx, 16, 2, 64, g, shared=160)
    q = torch.randn(B, hq, 64, generator=g).bfloat16()
    want, bound, _ = attend(q, k, v, tables, ctx, list(range(B)), [1] * B, None, 0.125, 0)
    q[1, 3, 0] = float("nan")
    out = S.shared_prefix_decode(q.to(DEV), k.to(DEV), v.to(DEV), tables.to(DEV), i32(ctx), 160, None, 0.125).cpu()
    assert out[1, 3].isnan().all()
    out[1, 3] = want[1, 3].bfloat16()
    within(out, want, bound)


def test_a_cache_past_32_bits():
  """Pages behind the first 2^32 bytes and 2^31 elements of a cache give what the same pages give in a small one."""
  from nmoe_b200.serve import ops as S
  bs, hkv, D, far = 64, 8, 64, 2 ** 31 // (64 * 8 * 64) + 3
  g = torch.Generator().manual_seed(2)
  ctx, lens, starts = [640, 130], [60, 3], [0, 60]
  k, v, tables = paged(ctx, bs, hkv, D, g, shared=64)
  n = k.size(0)
  big = [torch.empty(far + n, bs, hkv, D, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
  for c, small in zip(big, (k, v)):
    c[far:] = small.to(DEV)
  small = (k.to(DEV), v.to(DEV))
  t_small = tables.to(DEV)
  t_big = torch.where(t_small >= 0, t_small + far, t_small)
  q = torch.randn(63, 64, D, generator=g).bfloat16().to(DEV)
  call = lambda c, t: (S.paged_extend(q, *c, t, i32(ctx), i32(starts), i32(lens), None, 0.125),
                       S.paged_extend(q[60:], *c, t[1:], i32(ctx[1:]), i32([0]), i32([3]), None, 0.125),
                       S.shared_prefix_decode(q[:2], *c, t, i32(ctx), 64, None, 0.125))
  for a, b in zip(call(small, t_small), call(big, t_big)):
    assert torch.equal(a, b)
  qkv = torch.randn(5, 80 * D, generator=g).bfloat16().to(DEV)
  slots = i32([0, 7, n * bs - 1, -1, bs])
  pos, inv = torch.arange(5, device=DEV), torch.ones(32, device=DEV)
  S.rope_append(qkv, pos, inv, 1.0, 64, 8, *small, slots)
  S.rope_append(qkv, pos, inv, 1.0, 64, 8, *big, torch.where(slots >= 0, slots + far * bs, slots))
  assert all(torch.equal(c[far:], s) for c, s in zip(big, small))


def test_calls_on_two_streams_at_once():
  """Calls with workspaces and clusters beside each other, as two engines in one process make them."""
  from nmoe_b200.serve import ops as S
  g = torch.Generator().manual_seed(3)
  cases = []
  for ctx, lens in (([30_000], [1]), ([900, 4000, 80], [70, 5, 80])):
    k, v, tables = paged(ctx, 16, 2, 64, g)
    starts = [sum(lens[:b]) for b in range(len(lens))]
    q = torch.randn(sum(lens), 8, 64, generator=g).bfloat16().to(DEV)
    cases.append((q, k.to(DEV), v.to(DEV), tables.to(DEV), i32(ctx), i32(starts), i32(lens), None, 0.125))
  ctx = [2000 + b for b in range(30)]
  k, v, tables = paged(ctx, 16, 2, 64, g, shared=1600)
  shared = (torch.randn(30, 8, 64, generator=g).bfloat16().to(DEV), k.to(DEV), v.to(DEV), tables.to(DEV), i32(ctx), 1600, None, 0.125)
  step = lambda: [S.paged_extend(*c) for c in cases] + [S.shared_prefix_decode(*shared)]
  want = step()
  streams = [torch.cuda.Stream() for _ in range(2)]
  got = [[], []]
  torch.cuda.synchronize()
  for _ in range(5):
    for i, s in enumerate(streams):
      with torch.cuda.stream(s):
        got[i].append(step())
  torch.cuda.synchronize()
  for runs in got:
    for run in runs:
      assert all(torch.equal(a, b) for a, b in zip(run, want))


def test_paged_extend_reports_bad_pages_and_lengths():
  from nmoe_b200.ops import tc_gemm as G
  from nmoe_b200.ops._lib import NativeLibraryError
  from nmoe_b200.serve import ops as S
  G.check_status()
  g = torch.Generator().manual_seed(7)
  ctx = [40, 40, 40]
  k, v, tables = paged(ctx, 16, 2, 64, g)
  q = torch.randn(6, 8, 64, generator=g).bfloat16()
  args = lambda t, c, s, n: S.paged_extend(q.to(DEV), k.to(DEV), v.to(DEV), t.to(DEV), i32(c), i32(s), i32(n), None, 0.125, max_q_len=2)
  good = args(tables, ctx, [0, 2, 4], [2, 2, 2])
  G.check_status()
  bad = tables.clone()
  bad[1, 1] = 1 << 20
  for t, c, s, n, where in ((bad, ctx, [0, 2, 4], [2, 2, 2], 1022), (tables, [40, 1000, 40], [0, 2, 4], [2, 2, 2], 1021),
                            (tables, ctx, [0, 5, 4], [2, 2, 2], 1020), (tables, ctx, [0, -1, 4], [2, 2, 2], 1020),
                            (tables, ctx, [0, 2, 4], [2, 3, 2], 1020)):
    out = args(t, c, s, n)
    with pytest.raises(NativeLibraryError, match="code=2 where="):
      G.check_status()
    assert torch.equal(out[:2], good[:2]) and torch.equal(out[5:], good[5:])      # the other sequences are not touched


@pytest.mark.parametrize("hq,hkv,D,bs", SHAPES)
@pytest.mark.parametrize("prefix,window,use_sinks", [(0, 0, True), (100, 0, False), (128, 0, True), (129, 60, True), (257, 200, False)])
def test_shared_prefix_decode(hq, hkv, D, bs, prefix, window, use_sinks):
  from nmoe_b200.serve import ops as S
  g = torch.Generator().manual_seed(hq + prefix)
  ctx = [prefix + n for n in (1, 2, 70, 16, 33)]
  k, v, tables = paged(ctx, bs, hkv, D, g, shared=prefix)
  q = torch.randn(len(ctx), hq, D, generator=g).bfloat16()
  sinks = torch.randn(hq, generator=g) if use_sinks else None
  want, bound, _ = attend(q, k, v, tables, ctx, list(range(len(ctx))), [1] * len(ctx), sinks, D ** -0.5, window)
  out = S.shared_prefix_decode(q.to(DEV), k.to(DEV), v.to(DEV), tables.to(DEV), i32(ctx), prefix,
                               None if sinks is None else sinks.to(DEV), D ** -0.5, window)
  within(out, want, bound)


def test_shared_prefix_decode_many_rows_and_odd_contexts():
  """More rows than one tile, padding rows (context 0), sequences shorter than the prefix."""
  from nmoe_b200.serve import ops as S
  g = torch.Generator().manual_seed(9)
  prefix, hq, hkv, D = 700, 16, 2, 64
  ctx = [prefix + 1 + (7 * b) % 90 for b in range(70)]
  ctx[0], ctx[3], ctx[20], ctx[69], ctx[40] = 0, 0, 5, 700, 650
  k, v, tables = paged([max(c, prefix) for c in ctx], 16, hkv, D, g, shared=prefix)
  tables[0] = -1                                    # a padding row has no pages, in the first place neither
  q = torch.randn(70, hq, D, generator=g).bfloat16()
  sinks = torch.randn(hq, generator=g).bfloat16()
  want, bound, _ = attend(q, k, v, tables, ctx, list(range(70)), [1 if c else 0 for c in ctx], sinks, 0.125, 0)
  for lo, hi in ((0, 70), (0, 3), (18, 22)):        # as a whole, a few rows, a few among them shorter than the prefix
    out = S.shared_prefix_decode(q[lo:hi].to(DEV), k.to(DEV), v.to(DEV), tables[lo:hi].to(DEV), i32(ctx[lo:hi]), prefix, sinks.to(DEV), 0.125)
    within(out, want[lo:hi], bound[lo:hi] + 1e-30)


@pytest.mark.parametrize("B,prefix,suffix", [(2, 6000, 40), (3, 100, 5000), (300, 130, 20)])
def test_shared_prefix_decode_long_and_wide(B, prefix, suffix):
  """A long prefix of few sequences (split over many CTAs), long ends behind a short one, more sequences than are ranked."""
  from nmoe_b200.serve import ops as S
  g = torch.Generator().manual_seed(B)
  ctx = [prefix + suffix + b % 7 for b in range(B)]
  k, v, tables = paged(ctx, 16, 1, 64, g, shared=prefix)
  q = torch.randn(B, 4, 64, generator=g).bfloat16()
  want, bound, _ = attend(q, k, v, tables, ctx, list(range(B)), [1] * B, None, 0.125, 0)
  out = S.shared_prefix_decode(q.to(DEV), k.to(DEV), v.to(DEV), tables.to(DEV), i32(ctx), prefix, None, 0.125)
  within(out, want, bound)


# ------------------------------------------------------------------------------------------------ drafted tokens
def _verify_case(B, V, lens, dist, seed, dyadic=False):
  g = torch.Generator().manual_seed(seed)
  N = sum(lens)
  starts = [sum(lens[:b]) for b in range(B)]
  if dyadic:      # multiples of 1/16: sums are exact in every order, and uniforms fall on borders
    target = torch.randint(0, 4, (N, V), generator=g).float() / 16
    draft = torch.randint(0, 4, (N, V), generator=g).float() / 16
    u = torch.randint(0, 16, (N,), generator=g).float() / 16
  else:
    target = torch.softmax(2 * torch.randn(N, V, generator=g), -1)
    draft = torch.softmax(2 * target.roll(1, 0).log().mul(0.4) + torch.randn(N, V, generator=g) * 0.3, -1)
    u = torch.rand(N, generator=g)
  tokens = torch.multinomial(draft + 1e-9, 1, generator=g).squeeze(1)
  return target, tokens, u, starts, draft if dist else None


@pytest.mark.parametrize("V", [1, 2, 7, 100, 4096, 50_001])
@pytest.mark.parametrize("dist", [False, True])
@pytest.mark.parametrize("dyadic", [False, True])
def test_verify_draft(V, dist, dyadic):
  from nmoe_b200.serve import ops as S
  lens = [1, 5, 2, 0, 3, 9, 1, 4, 6] * (1 if V > 5000 else 5)
  target, tokens, u, starts, draft = _verify_case(len(lens), V, lens, dist, V, dyadic)
  want, count = verify(target.tolist(), tokens.tolist(), u.double().tolist(), starts, lens, None if draft is None else draft.tolist())
  for tok in (tokens, tokens.int()):
    out, n = S.verify_draft(target.to(DEV), tok.to(DEV), u.to(DEV), i32(starts), i32(lens), None if draft is None else draft.to(DEV))
    assert n.tolist() == count and out.tolist() == want


def test_verify_draft_strided_rows_gaps_and_degenerate_rows():
  from nmoe_b200.serve import ops as S
  V, lens = 1003, [3, 3, 3, 2, 1, 2]
  target, tokens, u, _, draft = _verify_case(6, V, lens, True, 3)
  starts = [9, 0, 3, 6, 13, 15]                     # any order, gaps at 8, 12 and 14
  N = 18
  pad = lambda t: torch.cat((t, t[:N - t.size(0)]), 0)
  target, tokens, u, draft = pad(target), pad(tokens), pad(u), pad(draft)
  draft[1] = target[0]                              # the two agree: nothing to redraw from if it failed
  tokens[1], target[0, tokens[1]] = int(target[0].argmin()), 0.0
  draft[1, tokens[1]] = 0.0                         # 0 < 0 fails, the difference is empty: drawn from the target
  target[14], target[15] = 0.0, 0.0
  target[13] = 0.0                                  # a row without a positive entry
  u[6] = 0.99999994                                 # the largest number below 1
  u[3] = 0.0
  want, count = verify(target.tolist(), tokens.tolist(), u.double().tolist(), starts, lens, draft.tolist())
  wide = torch.zeros(N, V + 5, device=DEV)
  wide[:, 2:V + 2] = target.to(DEV)
  keep = torch.full((N,), 77, dtype=torch.int32, device=DEV)
  out, n = S.verify_draft(wide[:, 2:V + 2], tokens.to(DEV), u.to(DEV), i32(starts), i32(lens), draft.to(DEV), out=keep)
  assert n.tolist() == count and out.tolist() == [77 if x is None else x for x in want]
  out2, _ = S.verify_draft(wide[:, 2:V + 2], tokens.to(DEV), u.to(DEV), i32(starts), i32(lens), draft.to(DEV))
  assert out2.tolist() == [-1 if x is None else x for x in want]


def test_verify_draft_emits_the_target_distribution():
  """Tokens drawn from the draft and verified are distributed as the target: every frequency within 5.5 standard deviations
  (24 of them, chance of a false alarm below 1e-6)."""
  from nmoe_b200.serve import ops as S
  g = torch.Generator().manual_seed(1)
  V, B = 24, 200_000
  p, q = torch.softmax(torch.randn(V, generator=g), -1), torch.softmax(torch.randn(V, generator=g), -1)
  tokens = torch.multinomial(q, 2 * B, replacement=True, generator=g)
  u = torch.rand(2 * B, generator=g)
  starts = torch.arange(B, dtype=torch.int32) * 2
  out, n = S.verify_draft(p.expand(2 * B, V).contiguous().to(DEV), tokens.to(DEV), u.to(DEV), starts.to(DEV),
                          torch.full((B,), 2, dtype=torch.int32, device=DEV), q.expand(2 * B, V).contiguous().to(DEV))
  freq = torch.bincount(out[0::2].cpu().long(), minlength=V).double() / B
  sd = (p.double() * (1 - p.double()) / B).sqrt()
  assert ((freq - p.double()).abs() < 5.5 * sd).all()


def test_verify_draft_reports_a_token_outside_the_vocabulary():
  from nmoe_b200.ops import tc_gemm as G
  from nmoe_b200.ops._lib import NativeLibraryError
  from nmoe_b200.serve import ops as S
  G.check_status()
  target = torch.full((3, 8), 0.125, device=DEV)
  out, n = S.verify_draft(target, torch.tensor([0, 8, 1], device=DEV), torch.zeros(3, device=DEV), i32([0]), i32([3]))
  with pytest.raises(NativeLibraryError, match="code=2 where=1011"):
    G.check_status()
  assert n.tolist() == [1] and out.tolist() == [0, -1, -1]
  S.verify_draft(target, torch.tensor([0, 1, 1], device=DEV), torch.zeros(3, device=DEV), i32([1]), i32([3]))
  with pytest.raises(NativeLibraryError, match="code=2 where=1010"):
    G.check_status()


# ------------------------------------------------------------------------------------------------ streams and graphs
def test_a_captured_step_replays_with_new_inputs_on_another_stream():
  """append -> attend -> verify captured on a side stream; two graphs, replayed in turn, share nothing."""
  from nmoe_b200.serve import ops as S
  g = torch.Generator().manual_seed(2)
  hq, hkv, D, bs, V = 8, 2, 64, 16, 333
  lens, ctx = [3, 1, 4], [50, 17, 200]
  k, v, tables = paged(ctx, bs, hkv, D, g, shared=16)
  starts, N = [0, 3, 4], 8
  inv = (10000.0 ** (-torch.arange(0, D, 2).float() / D)).to(DEV)
  slots, pos = [], []
  for b in range(3):
    for t in range(ctx[b] - lens[b], ctx[b]):
      pos.append(t)
      slots.append(int(tables[b, t // bs]) * bs + t % bs)
  pos, slots = torch.tensor(pos, device=DEV), i32(slots)
  ints = i32(ctx), i32(starts), i32(lens)
  probs = torch.softmax(torch.randn(N, V, generator=g) * 2, -1).to(DEV)
  tables = tables.to(DEV)

  def step(s):
    q, _, _ = S.rope_append(s["qkv"], pos, inv, 1.0, hq, hkv, s["k"], s["v"], slots)
    o = S.paged_extend(q, s["k"], s["v"], tables, *ints, None, 0.125, max_q_len=4)
    d = S.shared_prefix_decode(q[:3], s["k"], s["v"], tables, ints[0], 16, None, 0.125)
    return (o, d) + S.verify_draft(probs, s["tok"], s["u"], *ints[1:])

  def inputs(seed):
    gg = torch.Generator().manual_seed(seed)
    return dict(qkv=torch.randn(N, (hq + 2 * hkv) * D, generator=gg).bfloat16().to(DEV), k=k.to(DEV), v=v.to(DEV),
                tok=torch.randint(0, V, (N,), generator=gg).to(DEV), u=torch.rand(N, generator=gg).to(DEV))

  side = torch.cuda.Stream()
  states, graphs, outs = [inputs(0), inputs(1)], [], []
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    for s in states:
      step(s)
      graph = torch.cuda.CUDAGraph()
      with torch.cuda.graph(graph, stream=side):
        outs.append(step(s))
      graphs.append(graph)
  torch.cuda.synchronize()
  for round_ in range(2):
    fresh = [inputs(10 + round_), inputs(20 + round_)]
    for s, f in zip(states, fresh):
      for key in s:
        s[key].copy_(f[key])
    for gr in graphs:
      gr.replay()
    torch.cuda.synchronize()
    for o, f in zip(outs, fresh):
      for a, b in zip(o, step(f)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("window", [0, 128])
@pytest.mark.parametrize("D,hq,hkv", [(64, 64, 8), (128, 32, 4)])
def test_results_do_not_change_between_runs(window, D, hq, hkv):
  """Enough CTAs to fill every SM several times over: a wait that passes too early shows as a bit that changes."""
  from nmoe_b200.ops import tc_gemm as G
  from nmoe_b200.serve import ops as S
  g = torch.Generator().manual_seed(3)
  lens = [1 + b % 5 for b in range(40)] + [300, 290]
  ctx = [200 + 37 * b for b in range(40)] + [900, 290]
  starts = [sum(lens[:b]) for b in range(len(lens))]
  k, v, tables = paged(ctx, 16, hkv, D, g)
  k, v, tables = k.to(DEV), v.to(DEV), tables.to(DEV)
  q = torch.randn(sum(lens), hq, D, generator=g).bfloat16().to(DEV)
  args = (q, k, v, tables, i32(ctx), i32(starts), i32(lens), None, D ** -0.5, window)
  one = (q[:40], k, v, tables[:1].expand(40, -1).contiguous(), i32([200] * 40), 150, None, D ** -0.5, window)
  first, shared = S.paged_extend(*args), S.shared_prefix_decode(*one)
  for _ in range(200):
    assert torch.equal(S.paged_extend(*args), first)
    assert torch.equal(S.shared_prefix_decode(*one), shared)
  G.check_status()


# ------------------------------------------------------------------------------------------------ probabilities of decode steps
def _once_rounded(q, k, v, tables, ctx, starts, lens, sinks, scale, window):
  """(out, bound, owned) where only the result is rounded to bf16: ``attend`` with its allowance for rounded probabilities
  (half a step, 2^-8 of sum p |v|) taken out again.  What is left of it: probabilities that hold 2^-15 of themselves, and a sum
  over the keys in steps of 8 whose fp32 additions each lose 2^-22 of sum p |v|."""
  from serve_oracle import BF16
  want, bound, owned = attend(q, k, v, tables, ctx, starts, lens, sinks, scale, window)
  a = attend(q, k, v.abs(), tables, ctx, starts, lens, sinks, scale, window)[0]
  return want, bound + a * (2.0 ** -15 + max(ctx) / 8 * 2.0 ** -22 - BF16), owned


@pytest.mark.parametrize("hq,hkv,D,lens,ctx,window", [
  (8, 2, 64, [1, 2, 1], [300, 77, 1000], 0), (16, 2, 64, [1, 2, 0, 1], [300, 500, 9, 64], 150), (24, 3, 64, [3, 1], [700, 20], 0),
  (16, 2, 64, [5, 4], [600, 130], 0), (64, 8, 64, [1] * 5, [400, 90, 1, 33, 700], 128), (8, 2, 128, [2, 1], [300, 500], 0),
  (16, 2, 128, [2, 1], [300, 500], 0), (32, 4, 128, [4], [5000], 0), (32, 4, 128, [4, 5], [900, 300], 100), (64, 8, 64, [9, 16], [700, 900], 0),
  (8, 1, 64, [2], [9000], 0), (70, 1, 64, [1, 1], [500, 90], 0)])
@pytest.mark.parametrize("use_sinks", [False, True])
def test_a_few_tokens_are_rounded_once(hq, hkv, D, lens, ctx, window, use_sinks):
  """Decode steps and drafted ones keep what ``paged_decode`` gives: probabilities in more than the type of the values."""
  from nmoe_b200.serve import ops as S
  g = torch.Generator().manual_seed(hq + len(ctx))
  k, v, tables = paged(ctx, 16, hkv, D, g)
  starts = [sum(lens[:b]) for b in range(len(lens))]
  q = torch.randn(sum(lens), hq, D, generator=g).bfloat16()
  sinks = torch.randn(hq, generator=g) if use_sinks else None
  want, bound, _ = _once_rounded(q, k, v, tables, ctx, starts, lens, sinks, D ** -0.5, window)
  sd = None if sinks is None else sinks.to(DEV)
  out = S.paged_extend(q.to(DEV), k.to(DEV), v.to(DEV), tables.to(DEV), i32(ctx), i32(starts), i32(lens), sd, D ** -0.5, window,
                       max_q_len=max(lens))
  within(out, want, bound)
  if max(lens) == 1 and min(lens) == 1:
    within(S.paged_decode(q.to(DEV), k.to(DEV), v.to(DEV), tables.to(DEV), i32(ctx), sd, D ** -0.5, window), want, bound, "paged_decode")


@pytest.mark.parametrize("hq,hkv,D,B,prefix,window", [(8, 2, 64, 3, 300, 0), (64, 8, 64, 20, 160, 0), (64, 8, 64, 20, 160, 100), (16, 16, 128, 2, 333, 0),
                                                      (32, 4, 128, 9, 1000, 0), (48, 1, 64, 3, 500, 0), (16, 1, 128, 40, 4000, 0)])
def test_a_shared_prefix_is_rounded_once(hq, hkv, D, B, prefix, window):
  from nmoe_b200.serve import ops as S
  g = torch.Generator().manual_seed(B)
  ctx = [prefix + 1 + 13 * b for b in range(B)]
  k, v, tables = paged(ctx, 16, hkv, D, g, shared=prefix)
  q, sinks = torch.randn(B, hq, D, generator=g).bfloat16(), torch.randn(hq, generator=g)
  want, bound, _ = _once_rounded(q, k, v, tables, ctx, list(range(B)), [1] * B, sinks, D ** -0.5, window)
  out = S.shared_prefix_decode(q.to(DEV), k.to(DEV), v.to(DEV), tables.to(DEV), i32(ctx), prefix, sinks.to(DEV), D ** -0.5, window)
  within(out, want, bound)


# ------------------------------------------------------------------------------------------------ bounds at the ends of 32 bits
@pytest.mark.parametrize("n,hq", [(6, 8), (40, 8), (200, 8), (9, 1)])
def test_the_largest_window_hides_nothing(n, hq):
  """More new tokens than context: those before position 0 see nothing, the others everything, whatever the window's size."""
  from nmoe_b200.serve import ops as S
  g = torch.Generator().manual_seed(n)
  ctx, lens = [n - 4, n + 30], [n, n]
  k, v, tables = paged(ctx, 16, 1, 64, g)
  q = torch.randn(2 * n, hq, 64, generator=g).bfloat16()
  want, bound, _ = attend(q, k, v, tables, ctx, [0, n], lens, None, 0.125, 0)
  for window in (2 ** 31 - 1, 2 ** 31 - 5, 2 ** 30, 0):
    out = S.paged_extend(q.to(DEV), k.to(DEV), v.to(DEV), tables.to(DEV), i32(ctx), i32([0, n]), i32(lens), None, 0.125, window, max_q_len=n)
    within(out, want, bound, f"window {window}")
  assert (out[:4] == 0).all()


@pytest.mark.parametrize("D,hq,hkv", [(64, 8, 2), (64, 64, 1), (128, 32, 4)])
def test_contexts_below_zero_are_empty(D, hq, hkv):
  """However far below: no position may wrap around to one that looks past the block table."""
  from nmoe_b200.ops import tc_gemm as G
  from nmoe_b200.serve import ops as S
  g = torch.Generator().manual_seed(D)
  low = -2 ** 31
  ctx, lens = [50, low, -1, low + 1, 90, low + 3], [2, 2, 3, 1, 2, 4]
  k, v, tables = paged([max(c, 0) for c in ctx], 16, hkv, D, g, shared=32)
  starts = [sum(lens[:b]) for b in range(6)]
  q = torch.randn(sum(lens), hq, D, generator=g).bfloat16()
  real = [max(c, 0) for c in ctx]
  for window in (0, 7):
    want, bound, _ = attend(q, k, v, tables, real, starts, lens, None, D ** -0.5, window)
    for most in (4, sum(lens)):
      out = S.paged_extend(q.to(DEV), k.to(DEV), v.to(DEV), tables.to(DEV), i32(ctx), i32(starts), i32(lens), None, D ** -0.5, window, max_q_len=most)
      within(out, want, bound)
    want, bound, _ = attend(q[:6], k, v, tables, real, list(range(6)), [1 if c > 0 else 0 for c in ctx], None, D ** -0.5, window)
    out = S.shared_prefix_decode(q[:6].to(DEV), k.to(DEV), v.to(DEV), tables.to(DEV), i32(ctx), 32, None, D ** -0.5, window)
    within(out, want, bound)
  G.check_status()


@pytest.mark.parametrize("dist", [False, True])
def test_verify_draft_tokens_outside_the_vocabulary_fail(dist):
  """Negative, just past the end, and numbers that 32 bits would cut to one inside."""
  from nmoe_b200.ops import tc_gemm as G
  from nmoe_b200.ops._lib import NativeLibraryError
  from nmoe_b200.serve import ops as S
  G.check_status()
  target = torch.tensor([[0.25, 0, 0, 0, 0, 0, 0, 1.0]]).repeat(4, 1)
  draft = torch.zeros(4, 8) if dist else None
  for x in (-1, -8, 8, 2 ** 31 - 1, -2 ** 31, 2 ** 32 + 3, -2 ** 63):
    for u in (0.0, 0.19, 0.21, 0.99):
      for at in (1, 3):
        toks, uni = torch.tensor([0, 7, 7, 7]), torch.zeros(4)
        toks[at], uni[0] = x, u
        want, count = S.verify_draft(target, toks, uni, i32([0]).cpu(), i32([4]).cpu(), draft)
        with pytest.raises(NativeLibraryError, match="code=2 where=1011"):
          G.check_status(torch.device("cpu"))
        out, n = S.verify_draft(target.to(DEV), toks.to(DEV), uni.to(DEV), i32([0]), i32([4]), None if draft is None else draft.to(DEV))
        with pytest.raises(NativeLibraryError, match="code=2 where=1011"):
          G.check_status()
        assert out.tolist() == want.tolist() and n.tolist() == count.tolist() == [at]


@pytest.mark.parametrize("lens,ctx,D,hq,hkv", [([1, 3], [300, 70], 64, 8, 2), ([1], [30_000], 64, 8, 1), ([200, 150], [900, 400], 64, 8, 2),
                                               ([4], [20_000], 128, 32, 4), ([60, 2, 90], [60, 700, 500], 128, 8, 2)])
def test_paged_extend_in_place(lens, ctx, D, hq, hkv):
  from nmoe_b200.serve import ops as S
  g = torch.Generator().manual_seed(len(lens))
  k, v, tables = paged(ctx, 16, hkv, D, g)
  starts = [sum(lens[:b]) for b in range(len(lens))]
  q = torch.randn(sum(lens), hq, D, generator=g).bfloat16().to(DEV)
  args = (k.to(DEV), v.to(DEV), tables.to(DEV), i32(ctx), i32(starts), i32(lens), None, D ** -0.5)
  want = S.paged_extend(q, *args, max_q_len=max(lens))
  for _ in range(5):
    x = q.clone()
    assert S.paged_extend(x, *args, max_q_len=max(lens), out=x) is x and torch.equal(x, want)


@pytest.mark.parametrize("ctx", [[50, 900, 17, 300, 9, 128], [3000, 6000, 200, 5000, 9, 4100]])
@pytest.mark.parametrize("hq,hkv,window", [(64, 8, 0), (8, 1, 0), (16, 2, 100)])
def test_lists_of_few_rows_beside_longer_ones(ctx, hq, hkv, window):
  """1 to 5 tokens in one call: lists of 8 to 40 rows, on their own, split over a cluster, and in sets that are joined."""
  from nmoe_b200.serve import ops as S
  g = torch.Generator().manual_seed(hq)
  lens = [5, 1, 3, 2, 0, 4]
  k, v, tables = paged(ctx, 16, hkv, 64, g)
  starts = [sum(lens[:b]) for b in range(6)]
  q, sinks = torch.randn(sum(lens), hq, 64, generator=g).bfloat16(), torch.randn(hq, generator=g)
  want, bound, _ = _once_rounded(q, k, v, tables, ctx, starts, lens, sinks, 0.125, window)
  kd, vd = k.to(DEV), v.to(DEV)
  out = S.paged_extend(q.to(DEV), kd, vd, tables.to(DEV), i32(ctx), i32(starts), i32(lens), sinks.to(DEV), 0.125, window, max_q_len=5)
  within(out, want, bound)
  for b in (1, 2, 5):                               # one list at a time: other splits, sets
    one = S.paged_extend(q.to(DEV), kd, vd, tables[b:b + 1].to(DEV), i32(ctx[b:b + 1]), i32(starts[b:b + 1]), i32(lens[b:b + 1]), sinks.to(DEV), 0.125,
                         window, max_q_len=5)
    rows = slice(starts[b], starts[b] + lens[b])
    within(one[rows], want[rows], bound[rows])


@pytest.mark.parametrize("D,hq,hkv,n", [(64, 8, 1, 1), (128, 32, 4, 4)])
def test_captured_calls_with_workspaces_share_nothing(D, hq, hkv, n):
  """Two graphs whose calls split their keys into sets, replayed in turn and on two streams at once, with new contents."""
  from nmoe_b200.serve import ops as S
  g = torch.Generator().manual_seed(n)
  states, graphs, outs = [], [], []
  for ctx in ([30_000], [21_000, 9000]):
    B = len(ctx)
    k, v, tables = paged(ctx, 16, hkv, D, g)
    args = (torch.randn(n * B, hq, D, generator=g).bfloat16().to(DEV), k.to(DEV), v.to(DEV), tables.to(DEV), i32(ctx), i32([n * b for b in range(B)]),
            i32([n] * B), None, D ** -0.5)
    S.paged_extend(*args, max_q_len=n)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
      outs.append(S.paged_extend(*args, max_q_len=n))
    states.append(args)
    graphs.append(graph)
  streams = [torch.cuda.Stream() for _ in graphs]
  for turn in range(3):
    for args in states:
      args[0].copy_(torch.randn(args[0].shape, generator=g).bfloat16())
    want = [S.paged_extend(*args, max_q_len=n) for args in states]
    torch.cuda.synchronize()
    for _ in range(10):
      for graph, st in zip(graphs, streams):
        with torch.cuda.stream(st):
          graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("hq,D", [(129, 64), (200, 64), (130, 128)])
def test_one_token_of_many_heads_is_rounded_once(hq, D):
  """More query heads of a KV head than a tile holds: still decode steps."""
  from nmoe_b200.serve import ops as S
  g = torch.Generator().manual_seed(hq)
  ctx = [180, 90, 161]
  k, v, tables = paged(ctx, 16, 1, D, g, shared=80)
  q, sinks = torch.randn(3, hq, D, generator=g).bfloat16(), torch.randn(hq, generator=g)
  want, bound, _ = _once_rounded(q, k, v, tables, ctx, [0, 1, 2], [1] * 3, sinks, D ** -0.5, 0)
  args = q.to(DEV), k.to(DEV), v.to(DEV), tables.to(DEV), i32(ctx)
  within(S.paged_extend(*args, i32([0, 1, 2]), i32([1] * 3), sinks.to(DEV), D ** -0.5, max_q_len=1), want, bound)
  for prefix in (0, 80):
    within(S.shared_prefix_decode(*args, prefix, sinks.to(DEV), D ** -0.5), want, bound, f"prefix {prefix}")
