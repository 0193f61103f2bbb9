"""Cases for the operators of a serving step: rotate-and-append to the paged cache, attention of several new tokens
per sequence over the paged cache, attention of a batch that shares a prefix, and the verification of drafted tokens.

``run`` computes a case in plain torch operations (``own = False``) or through the framework (``own = True``).
Ragged lengths come from the case itself, so ``work`` can count them; values come from ``prepare``'s seed.
"""
import math
import random

import torch

own = False

DEV = "cuda"
NEG = float("-inf")

# (query heads, key/value heads, head size): the grading model's 64/8x64 and generic grouped, full and single-KV layouts
LAYOUTS = [(64, 8, 64), (32, 4, 128), (16, 16, 128), (8, 2, 64), (40, 8, 128), (14, 2, 64), (16, 1, 128)]


# ------------------------------------------------------------------------------------------------ cases
def listed():
  return [
    # one running sequence, one new token: pure latency
    dict(name="rope_append_1", op="rope", n=1, hq=64, hkv=8, d=64, bs=16, far=4000, pad=0.0, kv=False),
    # a decode step of a full batch (128 sequences)
    dict(name="rope_append_128", op="rope", n=128, hq=64, hkv=8, d=64, bs=16, far=4000, pad=0.0, kv=False),
    # prefill of one admission wave: 16384 prompt tokens, a fifth of them padding, rotated K and V wanted for the dense attention
    dict(name="rope_append_16384", op="rope", n=16384, hq=64, hkv=8, d=64, bs=16, far=131000, pad=0.2, kv=True),
    # a decode step with up to four drafted tokens for each of 64 sequences, contexts up to 4096
    dict(name="extend_drafts_64", op="extend", b=64, new_min=1, new_max=5, ctx_min=300, ctx_max=4096, hq=64, hkv=8, d=64, bs=16,
         window=0, sinks=True, lens=11),
    # the same with a sliding window of 128: the alternate layers of the grading model
    dict(name="extend_drafts_window", op="extend", b=33, new_min=1, new_max=5, ctx_min=40, ctx_max=4096, hq=64, hkv=8, d=64, bs=16,
         window=128, sinks=True, lens=12),
    # one sequence with a long context: the work has to be split over the keys
    dict(name="extend_long_context", op="extend", b=1, new_min=4, new_max=4, ctx_min=98765, ctx_max=98765, hq=32, hkv=4, d=128,
         bs=16, window=0, sinks=False, lens=13),
    # prompts whose first part was found in the prefix cache: ragged new parts over a cached rubric
    dict(name="extend_prefill", op="extend", b=8, new_min=200, new_max=1990, ctx_min=2400, ctx_max=4090, hq=64, hkv=8, d=64, bs=16,
         window=0, sinks=True, lens=14),
    # decode of a grading batch: 128 documents behind one rubric of 1500 tokens
    dict(name="shared_rubric_128", op="shared", b=128, prefix=1504, suf_min=20, suf_max=700, hq=64, hkv=8, d=64, bs=16, window=0,
         sinks=True, lens=15),
    # two sequences, a short odd prefix: the smallest sharing that pays at all
    dict(name="shared_pair", op="shared", b=2, prefix=333, suf_min=1, suf_max=90, hq=16, hkv=16, d=128, bs=16, window=0, sinks=False,
         lens=16),
    # a few-shot header of 16384 tokens before 64 short questions
    dict(name="shared_long_64", op="shared", b=64, prefix=16384, suf_min=5, suf_max=300, hq=32, hkv=4, d=128, bs=16, window=0,
         sinks=False, lens=17),
    # one sequence, four tokens looked up in its own text (no draft distribution), full vocabulary
    dict(name="verify_lookup_1", op="verify", b=1, draft_max=4, draft_min=4, v=201088, dist=False, lens=18),
    # 64 sequences with up to four tokens drawn from a drafter's distribution
    dict(name="verify_drafter_64", op="verify", b=64, draft_max=4, draft_min=0, v=201088, dist=True, lens=19),
  ]


def _log(rng, lo, hi):
  return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
  op = rng.choice(["rope", "extend", "shared", "verify"])
  if op == "verify":
    b, v = _log(rng, 1, 64), _log(rng, 50, 201088)
    return dict(op=op, b=b, draft_min=rng.choice([0, 1]), draft_max=rng.randint(1, 6) if b * v < 8_000_000 else 4, v=v,
                dist=rng.random() < 0.5, lens=rng.randrange(1 << 30))
  hq, hkv, d = rng.choice(LAYOUTS)
  base = dict(op=op, hq=hq, hkv=hkv, d=d, bs=rng.choice([16, 16, 16, 8, 32, 64, 12]))
  if op == "rope":
    return dict(base, n=_log(rng, 1, 12000), far=_log(rng, 100, 1_000_000), pad=rng.choice([0.0, 0.1, 0.5]), kv=rng.random() < 0.5)
  base.update(window=rng.choice([0, 0, 0, 128, rng.randint(1, 1000)]), sinks=rng.random() < 0.5, lens=rng.randrange(1 << 30))
  if op == "shared":
    b, prefix = _log(rng, 2, 128), _log(rng, 40, 16384)
    return dict(base, b=b, prefix=prefix, suf_min=1, suf_max=_log(rng, 2, max(3, min(2000, 60000 // b))))
  if rng.random() < 0.5:      # a few tokens for each sequence
    b = _log(rng, 1, 64)
    return dict(base, b=b, new_min=rng.choice([0, 1]), new_max=rng.randint(1, 8), ctx_min=1, ctx_max=_log(rng, 10, min(65536, 250000 // b)))
  b, new = _log(rng, 1, 8), _log(rng, 9, 1900)
  return dict(base, b=b, new_min=1, new_max=new, ctx_min=new, ctx_max=new + _log(rng, 1, 2000))


def _lens(case):
  """Ragged lengths of a case: (query tokens, context tokens) per sequence; the context counts the query tokens."""
  r = random.Random(case["lens"])
  if case["op"] == "verify":
    return [1 + r.randint(case["draft_min"], case["draft_max"]) for _ in range(case["b"])], None
  if case["op"] == "shared":
    return [1] * case["b"], [case["prefix"] + r.randint(case["suf_min"], case["suf_max"]) for _ in range(case["b"])]
  new = [r.randint(case["new_min"], case["new_max"]) for _ in range(case["b"])]
  return new, [max(n, r.randint(case["ctx_min"], case["ctx_max"])) for n in new]


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
  g = torch.Generator(device=DEV).manual_seed(seed)
  hg = random.Random(seed)

  def randn(*shape, dtype=torch.bfloat16, std=1.0):
    return (torch.randn(*shape, device=DEV, generator=g) * std).to(dtype)

  if case["op"] == "rope":
    n, hq, hkv, d, bs = case["n"], case["hq"], case["hkv"], case["d"], case["bs"]
    blocks = (n + bs - 1) // bs + 3
    slots = torch.randperm(blocks * bs, device=DEV, generator=g)[:n].to(torch.int32)
    slots = torch.where(torch.rand(n, device=DEV, generator=g) < case["pad"], torch.full_like(slots, -1), slots)
    pos = torch.randint(0, case["far"], (n,), device=DEV, generator=g)
    # frequencies interpolated by parts, as the grading model's long-context rotary has them
    inv = 150000.0 ** (-torch.arange(0, d, 2, dtype=torch.float32, device=DEV) / d)
    ramp = ((torch.arange(d // 2, dtype=torch.float32, device=DEV) - 0.25 * d / 2) / (0.3 * d / 2)).clamp(0, 1)
    inv = inv * (1 - ramp) + inv / 32 * ramp
    return dict(case=case, qkv=randn(n, (hq + 2 * hkv) * d, std=1.5), pos=pos, inv=inv.contiguous(), conc=0.1 * math.log(32.0) + 1.0,
                slots=slots, k_cache=randn(blocks, bs, hkv, d), v_cache=randn(blocks, bs, hkv, d))

  if case["op"] == "verify":
    q_lens, _ = _lens(case)
    n, v = sum(q_lens), case["v"]
    starts = [sum(q_lens[:i]) for i in range(len(q_lens))]
    logits = torch.randn(n, v, device=DEV, generator=g) * 2.5
    target = torch.softmax(logits, -1)
    draft = None
    if case["dist"]:      # row r: what the token at row r was drawn from, a blurred copy of the target row before it
      draft = logits.roll(1, 0).mul_(0.8).add_(torch.randn(n, v, device=DEV, generator=g))
      draft = torch.softmax(draft, -1)
      tokens = torch.multinomial(draft, 1, generator=g).squeeze(1)
    else:                 # looked-up tokens: often the likeliest one, otherwise any
      tokens = torch.where(torch.rand(n, device=DEV, generator=g) < 0.7, target.roll(1, 0).argmax(-1),
                           torch.randint(0, v, (n,), device=DEV, generator=g))
    return dict(case=case, target=target, draft=draft, tokens=tokens, u=torch.rand(n, device=DEV, generator=g),
                starts=torch.tensor(starts, dtype=torch.int32, device=DEV), lens=torch.tensor(q_lens, dtype=torch.int32, device=DEV))

  q_lens, ctx = _lens(case)
  b, hq, hkv, d, bs = case["b"], case["hq"], case["hkv"], case["d"], case["bs"]
  n_shared = case["prefix"] // bs if case["op"] == "shared" else 0       # whole pages before the sequences part
  need = [(c + bs - 1) // bs for c in ctx]
  total = n_shared + sum(m - n_shared for m in need) + 2
  perm = list(range(total))
  hg.shuffle(perm)
  width = max(need) + 1
  used, rows = n_shared, []
  for m in need:
    rows.append(perm[:n_shared] + perm[used:used + m - n_shared] + [0] * (width - m))
    used += m - n_shared
  n = sum(q_lens)
  k_cache, v_cache = randn(total, bs, hkv, d), randn(total, bs, hkv, d)
  if n_shared * bs < case.get("prefix", 0):
    # the prefix ends inside a page: each sequence has its own copy of that page's shared head
    first, r = torch.tensor([row[n_shared] for row in rows], device=DEV), case["prefix"] - n_shared * bs
    k_cache[first, :r] = k_cache[first[0], :r].clone()
    v_cache[first, :r] = v_cache[first[0], :r].clone()
  return dict(case=case, q=randn(n, hq, d, std=1.3), k_cache=k_cache, v_cache=v_cache,
              tables=torch.tensor(rows, dtype=torch.int32, device=DEV), ctx=torch.tensor(ctx, dtype=torch.int32, device=DEV),
              starts=torch.tensor([sum(q_lens[:i]) for i in range(b)], dtype=torch.int32, device=DEV),
              lens=torch.tensor(q_lens, dtype=torch.int32, device=DEV), q_lens=q_lens, ctx_lens=ctx, scale=1.0 / math.sqrt(d),
              sinks=randn(hq) if case["sinks"] else None)


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_rope(s):
  case = s["case"]
  n, hq, hkv, d = case["n"], case["hq"], case["hkv"], case["d"]
  q, k, v = s["qkv"].split([hq * d, hkv * d, hkv * d], dim=-1)
  ang = s["pos"].double().unsqueeze(-1) * s["inv"].double()              # far positions: the angle needs 64 bits
  cos, sin = (ang.cos() * s["conc"]).float().unsqueeze(1), (ang.sin() * s["conc"]).float().unsqueeze(1)

  def rot(x):
    a, b = x.float().chunk(2, dim=-1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1).to(torch.bfloat16)

  q, k, v = rot(q.reshape(n, hq, d)), rot(k.reshape(n, hkv, d)), v.reshape(n, hkv, d)
  ok = s["slots"] >= 0
  at = s["slots"][ok].long()
  s["k_cache"].view(-1, hkv, d)[at] = k[ok]
  s["v_cache"].view(-1, hkv, d)[at] = v[ok]
  return (q, k, v.contiguous(), s["k_cache"], s["v_cache"]) if case["kv"] else (q, s["k_cache"], s["v_cache"])


def _plain_attention(s):
  """Every sequence by itself: its keys and values gathered from the pages, scores, masked softmax with the sink, product."""
  case = s["case"]
  hq, hkv, d, bs, window = case["hq"], case["hkv"], case["d"], case["bs"], case["window"]
  g = hq // hkv
  kc, vc = s["k_cache"].view(-1, hkv, d), s["v_cache"].view(-1, hkv, d)
  out = torch.zeros_like(s["q"])
  r0 = 0
  for i, (n, ctx) in enumerate(zip(s["q_lens"], s["ctx_lens"])):
    if n > 0:
      first = max(0, ctx - n - window + 1) if window > 0 else 0          # the oldest key that any of these tokens sees
      pos = torch.arange(first, ctx, device=DEV)
      slot = s["tables"][i, pos // bs].long() * bs + pos % bs
      k, v = kc[slot].float().permute(1, 2, 0), vc[slot].float().transpose(0, 1)          # [Hkv, D, m], [Hkv, m, D]
      q = s["q"][r0:r0 + n].float().view(n, hkv, g, d).permute(1, 2, 0, 3).reshape(hkv, g * n, d)
      sc = torch.matmul(q, k).mul_(s["scale"]).view(hkv, g, n, -1)
      at = torch.arange(ctx - n, ctx, device=DEV).unsqueeze(1)
      hide = pos > at
      if window > 0:
        hide = hide | (pos <= at - window)
      sc.masked_fill_(hide, NEG)
      m = sc.amax(-1, keepdim=True)
      if s["sinks"] is not None:
        sk = s["sinks"].float().view(hkv, g, 1, 1)
        m = torch.maximum(m, sk)
      sc = sc.sub_(m).exp_()
      den = sc.sum(-1, keepdim=True)
      if s["sinks"] is not None:
        den = den + (sk - m).exp()
      o = torch.matmul(sc.view(hkv, g * n, -1), v).view(hkv, g, n, d) / den
      out[r0:r0 + n] = o.permute(2, 0, 1, 3).reshape(n, hq, d).to(out.dtype)
    r0 += n
  return out


def _plain_verify(s):
  """A drafted token x passes while u * q(x) < p(x); the first that fails is redrawn from max(p - q, 0), and after the last
  one the next token is drawn from p, both by the first row's number against the running sum.  64 bits: whole numbers."""
  target, draft, tokens, u = s["target"], s["draft"], s["tokens"], s["u"].double()
  out = torch.full_like(s["tokens"], -1, dtype=torch.int32)
  starts, lens, n = s["starts"].long(), s["lens"].long(), tokens.numel()
  rows = torch.arange(n, device=DEV)
  prev = (rows - 1).clamp(min=0)
  p = target[prev, tokens].double()
  q = draft[rows, tokens].double() if draft is not None else torch.ones_like(p)
  seq = torch.searchsorted(starts, rows, right=True) - 1
  is_draft = rows > starts[seq]
  fails = is_draft & ~(u * q < p)
  at = rows - starts[seq]                                                # j-th drafted token stands at row start + j
  acc = torch.scatter_reduce(lens - 1, 0, seq, torch.where(fails, at - 1, n), "amin")
  row = starts + acc                                                     # the target row of the token that is drawn
  w = target[row].double()
  cut = acc < lens - 1
  nxt = (row + 1).clamp(max=n - 1)
  if draft is not None:
    w = torch.where(cut[:, None], (w - draft[nxt].double()).clamp_(min=0), w)
  else:
    b = torch.arange(len(starts), device=DEV)
    w[b, tokens[nxt]] = torch.where(cut, torch.zeros_like(u[:1]), w[b, tokens[nxt]])
  total = w.sum(-1, keepdim=True)
  w = torch.where(total > 0, w, target[row].double())                    # nothing left of the difference: the target itself
  total = w.sum(-1, keepdim=True)
  hit = w.cumsum(-1) > u[starts][:, None] * total
  last = w.size(-1) - 1 - (w > 0).flip(-1).to(torch.int8).argmax(-1)
  new = torch.where(hit.any(-1), hit.to(torch.int8).argmax(-1), last)
  keep = is_draft & (at <= acc[seq])
  out[rows[keep] - 1] = tokens[keep].to(torch.int32)
  out[row] = new.to(torch.int32)
  return out, (acc + 1).to(torch.int32)


def run(state):
  op = state["case"]["op"]
  if not own:
    return _plain_rope(state) if op == "rope" else _plain_verify(state) if op == "verify" else _plain_attention(state)
  from nmoe_b200.serve import ops as S
  c = state["case"]
  if op == "rope":
    q, k, v = S.rope_append(state["qkv"], state["pos"], state["inv"], state["conc"], c["hq"], c["hkv"], state["k_cache"],
                            state["v_cache"], state["slots"], need_kv=c["kv"])
    return (q, k, v, state["k_cache"], state["v_cache"]) if c["kv"] else (q, state["k_cache"], state["v_cache"])
  if op == "verify":
    return S.verify_draft(state["target"], state["tokens"], state["u"], state["starts"], state["lens"], state["draft"],
                          out=torch.empty_like(state["tokens"], dtype=torch.int32))
  if op == "shared":
    return S.shared_prefix_decode(state["q"], state["k_cache"], state["v_cache"], state["tables"], state["ctx"], c["prefix"],
                                  state["sinks"], state["scale"], c["window"])
  return S.paged_extend(state["q"], state["k_cache"], state["v_cache"], state["tables"], state["ctx"], state["starts"],
                        state["lens"], state["sinks"], state["scale"], c["window"], max_q_len=max(state["q_lens"]),
                        out=torch.empty_like(state["q"]))


# ------------------------------------------------------------------------------------------------ the definition, in 64 bits
def exact(case, seed):
  s = prepare(case, seed)
  if case["op"] == "rope":
    n, hq, hkv, d = case["n"], case["hq"], case["hkv"], case["d"]
    x = s["qkv"].double().view(n, hq + 2 * hkv, d)
    z = torch.polar(torch.full((n, d // 2), float(s["conc"]), dtype=torch.float64, device=DEV),
                    s["pos"].double()[:, None] * s["inv"].double()[None])
    y = torch.complex(x[..., :d // 2].contiguous(), x[..., d // 2:].contiguous()) * z[:, None]      # the pair as a complex number
    y = torch.cat((y.real, y.imag), -1)
    kc, vc = s["k_cache"].double().view(-1, hkv, d), s["v_cache"].double().view(-1, hkv, d)
    rows = (s["slots"] >= 0).nonzero().flatten()
    kc.index_copy_(0, s["slots"][rows].long(), y[rows, hq:hq + hkv])
    vc.index_copy_(0, s["slots"][rows].long(), x[rows, hq + hkv:])
    kc, vc = kc.view_as(s["k_cache"]), vc.view_as(s["v_cache"])
    return (y[:, :hq], y[:, hq:hq + hkv], x[:, hq + hkv:], kc, vc) if case["kv"] else (y[:, :hq], kc, vc)
  if case["op"] == "verify":
    p, u, x = s["target"].cpu(), s["u"].double().tolist(), s["tokens"].tolist()
    qd = s["draft"].cpu() if s["draft"] is not None else None
    out, count, r0 = [-1] * len(x), [], 0
    for n in s["lens"].tolist():
      j = 0
      while j + 1 < n:
        r = r0 + j + 1
        q = float(qd[r, x[r]]) if qd is not None else 1.0
        if not u[r] * q < float(p[r - 1, x[r]]):
          break
        out[r0 + j] = x[r]
        j += 1
      w = p[r0 + j].double()
      if j + 1 < n:
        if qd is not None:
          w = torch.clamp(w - qd[r0 + j + 1].double(), min=0.0)
        else:
          w[x[r0 + j + 1]] = 0.0
        if float(w.sum()) <= 0.0:
          w = p[r0 + j].double()
      below = int((torch.cumsum(w, 0) <= u[r0] * float(w.sum())).sum())
      out[r0 + j] = below if below < w.numel() else int(w.nonzero()[-1])
      count.append(j + 1)
      r0 += n
    return torch.tensor(out, dtype=torch.int32), torch.tensor(count, dtype=torch.int32)
  # attention, one key/value head and one stretch of queries at a time, by the pages in order
  hq, hkv, d, bs, window = case["hq"], case["hkv"], case["d"], case["bs"], case["window"]
  g = hq // hkv
  out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
  r0 = 0
  for i, (n, ctx) in enumerate(zip(s["q_lens"], s["ctx_lens"])):
    pages = s["tables"][i, :(ctx + bs - 1) // bs].long()
    for h in range(hkv):
      k = s["k_cache"][pages, :, h].reshape(-1, d)[:ctx].double()
      v = s["v_cache"][pages, :, h].reshape(-1, d)[:ctx].double()
      for a in range(0, n, 256):
        e = min(n, a + 256)
        q = s["q"][r0 + a:r0 + e, h * g:(h + 1) * g].double()
        sc = torch.einsum("qgd,kd->gqk", q, k) * s["scale"]
        qp = torch.arange(ctx - n + a, ctx - n + e, device=DEV)[:, None]
        kp = torch.arange(ctx, device=DEV)[None]
        seen = (kp <= qp) & (kp > qp - window) if window > 0 else kp <= qp
        sc = torch.where(seen, sc, torch.full_like(sc, NEG))
        if s["sinks"] is not None:
          extra = s["sinks"][h * g:(h + 1) * g].double()[:, None, None].expand(g, e - a, 1)
          pr = torch.softmax(torch.cat((sc, extra), -1), -1)[..., :-1]
        else:
          pr = torch.softmax(sc, -1)
        out[r0 + a:r0 + e, h * g:(h + 1) * g] = torch.einsum("gqk,kd->qgd", pr, v)
    r0 += n
  return out


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def _seen(n, ctx, window):
  """(query, key) pairs of n tokens at the end of a context, and the keys that at least one of them sees."""
  if n == 0:
    return 0, 0
  pairs = sum(min(p + 1, window) if window > 0 else p + 1 for p in range(ctx - n, ctx))
  return pairs, min(ctx, window + n - 1) if window > 0 else ctx


def work(case):
  if case["op"] == "rope":
    n, hq, hkv, d = case["n"], case["hq"], case["hkv"], case["d"]
    live = n * (1 - case["pad"])
    read = n * (hq + 2 * hkv) * d * 2 + n * 12 + d * 2
    write = n * hq * d * 2 + live * 2 * hkv * d * 2 + (n * 2 * hkv * d * 2 if case["kv"] else 0)
    return {"bytes": int(read + write), "flops": n * (hq + hkv) * d * 3}
  q_lens, ctx = _lens(case)
  if case["op"] == "verify":
    b, n = case["b"], sum(q_lens)
    # one row of the target for each sequence, and the draft row beside it where a token failed (about half of the sequences)
    cut = sum(1 for m in q_lens if m > 1) * 0.5
    return {"bytes": int(case["v"] * 4 * (b + (cut if case["dist"] else 0)) + n * 24), "flops": int(case["v"] * 2 * b)}
  hq, hkv, d, window = case["hq"], case["hkv"], case["d"], case["window"]
  pairs = keys = 0
  for n, c in zip(q_lens, ctx):
    a, k = _seen(n, c, window)
    pairs += a
    keys += k
  if case["op"] == "shared":                                             # the prefix's keys count once
    start = [max(0, c - window) if window > 0 else 0 for c in ctx]
    keys = sum(c - max(st, case["prefix"]) for c, st in zip(ctx, start)) + max(0, case["prefix"] - min(start))
  return {"bytes": keys * hkv * d * 4 + 2 * sum(q_lens) * hq * d * 2 + sum(ctx) // case["bs"] * 4, "flops": 4 * pairs * hq * d}
