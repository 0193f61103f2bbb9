"""Plain 64-bit statements of the serving operators, for the tests (CPU tensors)."""
import torch

BF16 = 2.0 ** -8          # half a step of bf16, relative to the value


def rope(qkv, pos, inv, conc, hq, hkv):
  """(rotated heads [N, Hq + Hkv, D], error bound of them, v) in fp64.

  Bound: one rounding to bf16, and before it fp32 arithmetic on cos and sin that are off by a few 2^-24."""
  N = qkv.size(0)
  x = qkv.double().view(N, hq + 2 * hkv, -1)
  D = x.size(-1)
  a = pos.double()[:, None] * inv.double()[None]
  c, s = (a.cos() * conc)[:, None], (a.sin() * conc)[:, None]
  x1, x2 = x[:, :hq + hkv, :D // 2], x[:, :hq + hkv, D // 2:]
  y = torch.cat((x1 * c - x2 * s, x2 * c + x1 * s), -1)
  mag = (x1.abs() + x2.abs()).repeat(1, 1, 2) * conc
  return y, BF16 * y.abs() + 2.0 ** -20 * mag + 1e-30, x[:, hq + hkv:]


def attend(q, k_cache, v_cache, tables, ctx, starts, lens, sinks, scale, window):
  """(out [N, Hq, D], bound, rows that belong to a sequence) in fp64.

  Bound: the probabilities are rounded to bf16 before they meet the values (half a step of each, so at most
  BF16 * sum p |v|) and the result once more (BF16 * |o|).  The scores are fp32 sums of D exact products, off by at most
  D * 2^-24 * sum |q k|, which moves p by that much in relative terms; exp2 and the normaliser add a few 2^-22."""
  N, hq, D = q.shape
  _, bs, hkv, _ = k_cache.shape
  g = hq // hkv
  out = torch.zeros(N, hq, D, dtype=torch.float64)
  bound = torch.zeros(N, hq, D, dtype=torch.float64)
  owned = torch.zeros(N, dtype=torch.bool)
  kc, vc = k_cache.double(), v_cache.double()
  for b in range(len(ctx)):
    for j in range(lens[b]):
      r = starts[b] + j
      owned[r] = True
      pos = ctx[b] - lens[b] + j
      keys = list(range(max(0, pos - window + 1) if window > 0 else 0, pos + 1))
      if not keys:
        continue
      pg = tables[b][torch.tensor(keys) // bs].long()
      k, v = kc[pg, torch.tensor(keys) % bs], vc[pg, torch.tensor(keys) % bs]            # [m, Hkv, D]
      k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
      s = (q[r].double()[None] * k).sum(-1) * scale                                     # [m, Hq]
      slip = ((q[r].double()[None] * k).abs().sum(-1) * scale).max(0).values * D * 2.0 ** -24
      m = s.max(0).values
      if sinks is not None:
        m = torch.maximum(m, sinks.double())
      e = (s - m).exp()
      den = e.sum(0) + ((sinks.double() - m).exp() if sinks is not None else 0.0)
      p = e / den
      o = torch.einsum("mh,mhd->hd", p, v)
      a = torch.einsum("mh,mhd->hd", p, v.abs())
      out[r] = o
      bound[r] = BF16 * (o.abs() + a) + a * (2.0 ** -17 + 2 * slip[:, None]) + 1e-30
  return out, bound, owned


def verify(target, tokens, u, starts, lens, draft):
  """Emitted tokens and counts, in plain Python on 64-bit numbers."""
  out, count = [None] * len(tokens), []
  for s0, n in zip(starts, lens):
    emitted = []
    for i in range(1, n):
      x = tokens[s0 + i]
      q = float(draft[s0 + i][x]) if draft is not None else 1.0
      if not u[s0 + i] * q < float(target[s0 + i - 1][x]):
        break
      emitted.append(x)
    if n > 0:
      j = len(emitted)
      p = [float(a) for a in target[s0 + j]]
      w = list(p)
      if j + 1 < n:
        if draft is not None:
          w = [max(a - float(c), 0.0) for a, c in zip(p, draft[s0 + j + 1])]
        else:
          w[tokens[s0 + j + 1]] = 0.0
        if sum(w) <= 0.0:
          w = p
      goal, c, new = u[s0] * sum(w), 0.0, None
      for i, a in enumerate(w):
        c += a
        if a > 0.0 and c > goal:
          new = i
          break
      if new is None:
        new = max((i for i, a in enumerate(w) if a > 0.0), default=len(w) - 1)
      emitted.append(new)
      for i in range(n):
        out[s0 + i] = emitted[i] if i < len(emitted) else -1
    count.append(len(emitted))
  return out, count


def paged(ctx, bs, hkv, D, gen, *, shared=0, spare=2, dtype=torch.bfloat16):
  """A cache whose pages lie in random order: (k_cache, v_cache, tables [B, width] with -1 behind each table).
  The first ``shared`` tokens of all sequences are the same (whole pages are shared, a partial one is copied)."""
  n_shared = shared // bs
  need = [(c + bs - 1) // bs for c in ctx]
  own = [max(0, m - n_shared) for m in need]
  total = n_shared + sum(own) + spare
  perm = torch.randperm(total, generator=gen).int()
  tables = torch.full((len(ctx), max(need + [n_shared]) + 1), -1, dtype=torch.int32)
  used = n_shared
  k, v = (torch.randn(total, bs, hkv, D, generator=gen).to(dtype) for _ in range(2))
  for b, m in enumerate(own):
    tables[b, :n_shared] = perm[:n_shared]
    tables[b, n_shared:n_shared + m] = perm[used:used + m]
    used += m
  rest = shared - n_shared * bs
  if rest:
    owners = [b for b in range(len(ctx)) if ctx[b] > n_shared * bs]
    for b in owners[1:]:
      for c in (k, v):
        c[tables[b, n_shared].long(), :rest] = c[tables[owners[0], n_shared].long(), :rest]
  return k, v, tables
