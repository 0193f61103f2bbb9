"""Device ops of the serving engine, with plain-PyTorch statements of the same maths for CPU tensors and as test oracles:

  kv_store, paged_decode    scatter K/V rows, one query token per sequence     csrc/paged_attention.cu
  rope_append               rotary embedding + cache append in one pass        csrc/rope_append.cu
  paged_extend              several query tokens per sequence                  csrc/paged_extend.cu
  shared_prefix_decode      one token per sequence behind a common prefix      csrc/paged_extend.cu
  verify_draft              accept / redraw drafted tokens                     csrc/verify_draft.cu
"""
from __future__ import annotations

import contextlib
import ctypes
from typing import Optional, Tuple

import torch

from ..ops import _lib as L
from ..ops.tc_gemm import status_buffer


def kv_store(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor) -> None:
  """k, v: [N, Hkv, D] (views into a fused projection are fine: only the last two dims must be dense);
  caches: [num_blocks, block_size, Hkv, D]; slots: [N] int32, negative = skip."""
  N, Hkv, D = k.shape
  if not k.is_cuda:
    ok = slots >= 0
    kc = k_cache.view(-1, Hkv, D)
    vc = v_cache.view(-1, Hkv, D)
    kc[slots[ok].long()] = k[ok]
    vc[slots[ok].long()] = v[ok]
    return
  assert k.stride(2) == 1 and k.stride(1) == D and v.stride(2) == 1 and v.stride(1) == D
  assert k_cache.is_contiguous() and v_cache.is_contiguous() and slots.dtype == torch.int32
  L.check(L.lib().nmoe_kv_store(L.ptr(k), L.ptr(v), L.ptr(k_cache), L.ptr(v_cache), L.ptr(slots), N, Hkv * D,
                                L.c_ll(k.stride(0)), L.c_ll(v.stride(0)), L.stream()), "kv_store")


def paged_decode_reference(q, k_cache, v_cache, block_tables, context_lens, sinks, scale, window=0):
  """fp32 oracle: q [B,Hq,D] against the cached context of each sequence."""
  B, Hq, D = q.shape
  nb, bs, Hkv, _ = k_cache.shape
  g = Hq // Hkv
  out = torch.zeros(B, Hq, D, dtype=torch.float32)
  for b in range(B):
    ctx = int(context_lens[b])
    start = max(0, ctx - window) if window > 0 else 0
    pos = torch.arange(start, ctx)
    slot = block_tables[b, pos // bs].long() * bs + pos % bs
    k = k_cache.view(-1, Hkv, D)[slot].float().cpu().repeat_interleave(g, dim=1)      # [n, Hq, D]
    v = v_cache.view(-1, Hkv, D)[slot].float().cpu().repeat_interleave(g, dim=1)
    s = torch.einsum("hd,nhd->hn", q[b].float().cpu(), k) * scale
    if sinks is not None:
      s = torch.cat((s, sinks.float().cpu().view(Hq, 1)), dim=1)
    p = torch.softmax(s, dim=-1)
    if sinks is not None:
      p = p[:, :-1]
    out[b] = torch.einsum("hn,nhd->hd", p, v)
  return out


def paged_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                 context_lens: torch.Tensor, sinks: Optional[torch.Tensor], scale: float, window: int = 0) -> torch.Tensor:
  """One new token per sequence: q [B,Hq,D] -> [B,Hq,D].  ``context_lens`` counts the current token,
  whose K/V must already be in the cache."""
  if not q.is_cuda:
    return paged_decode_reference(q, k_cache, v_cache, block_tables, context_lens, sinks, scale, window).to(q.dtype)
  B, Hq, D = q.shape
  _, bs, Hkv, _ = k_cache.shape
  q = q.contiguous()
  out = torch.empty_like(q)
  sk = sinks.detach().float().contiguous() if sinks is not None else None
  assert block_tables.dtype == torch.int32 and context_lens.dtype == torch.int32 and block_tables.is_contiguous()
  L.check(L.lib().nmoe_paged_decode(L.ptr(q), L.ptr(k_cache), L.ptr(v_cache), L.ptr(block_tables), L.ptr(context_lens),
                                    L.ptr(sk), L.ptr(out), B, Hq, Hkv, D, bs, block_tables.size(1), int(window),
                                    L.c_float(scale), L.stream()), "paged_decode")
  return out


# ------------------------------------------------------------------ shared pieces of the operators below
def _need(ok: bool, what: str) -> None:
  if not ok:
    raise ValueError(what)


def _on(device: torch.device):
  """Launches go to the current stream of the tensors' own device, whichever device is current."""
  return contextlib.nullcontext() if device.index == torch.cuda.current_device() else torch.cuda.device(device)


_FN = {}


def _fn(name: str, sig: str, result=ctypes.c_int):
  """C entry with its argument types set once (p pointer, i int, l long long, f float): plain numbers can be passed."""
  f = _FN.get(name)
  if f is None:
    f = getattr(L.lib(), name)
    f.argtypes = [{"p": ctypes.c_void_p, "i": ctypes.c_int, "l": ctypes.c_longlong, "f": ctypes.c_float}[c] for c in sig]
    f.restype = result
    _FN[name] = f
  return f


def _p(t: Optional[torch.Tensor]) -> int:
  return 0 if t is None else t.data_ptr()


def _stream() -> int:
  return torch.cuda.current_stream().cuda_stream


def _aligned(t: torch.Tensor) -> bool:
  return t.data_ptr() % 16 == 0


def _check_cache(k_cache: torch.Tensor, v_cache: torch.Tensor, like: torch.Tensor, Hkv: int, D: int) -> None:
  _need(k_cache.dim() == 4 and k_cache.shape == v_cache.shape, "k_cache and v_cache must be [num_blocks, block_size, Hkv, D]")
  _need(k_cache.size(2) == Hkv and k_cache.size(3) == D, f"the cache holds {tuple(k_cache.shape[2:])} heads x dims, expected ({Hkv}, {D})")
  _need(k_cache.is_contiguous() and v_cache.is_contiguous(), "k_cache and v_cache must be contiguous")
  _need(k_cache.dtype == like.dtype and v_cache.dtype == like.dtype, "the cache and the activations must have one dtype")
  _need(k_cache.device == like.device and v_cache.device == like.device, "the cache must be on the activations' device")


def _check_ints(device: torch.device, **tensors: Optional[torch.Tensor]) -> None:
  for name, t in tensors.items():
    if t is not None:
      _need(t.dtype == torch.int32 and t.device == device, f"{name} must be int32 on {device}")


# ------------------------------------------------------------------ rotate and append
def rope_append_reference(qkv, positions, inv_freq, conc, n_heads, n_kv_heads, k_cache=None, v_cache=None, slots=None):
  """Plain statement of ``rope_append`` (angles in fp64, the rest in fp32): rotated q, rotated k, v."""
  N = qkv.size(0)
  D = qkv.size(1) // (n_heads + 2 * n_kv_heads)
  ang = positions.double().unsqueeze(-1) * inv_freq.double()
  cos, sin = (ang.cos().float() * conc).unsqueeze(1), (ang.sin().float() * conc).unsqueeze(1)
  x = qkv.reshape(N, n_heads + 2 * n_kv_heads, D)
  x1, x2 = x[:, :n_heads + n_kv_heads].float().chunk(2, dim=-1)
  qk = torch.cat((x1 * cos - x2 * sin, x2 * cos + x1 * sin), dim=-1).to(qkv.dtype)
  q, k, v = qk[:, :n_heads].contiguous(), qk[:, n_heads:].contiguous(), x[:, n_heads + n_kv_heads:].contiguous()
  if slots is not None:
    ok = slots >= 0
    k_cache.view(-1, n_kv_heads, D)[slots[ok].long()] = k[ok]
    v_cache.view(-1, n_kv_heads, D)[slots[ok].long()] = v[ok]
  return q, k, v


def rope_append(qkv: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, conc: float, n_heads: int, n_kv_heads: int,
                k_cache: Optional[torch.Tensor] = None, v_cache: Optional[torch.Tensor] = None,
                slots: Optional[torch.Tensor] = None, *, need_kv: bool = False
                ) -> Tuple[torch.Tensor, Optional[torch.Tensor], Optional[torch.Tensor]]:
  """Rotates the q and k heads of a fused projection and appends K and V to the paged cache, in one pass.

  qkv [N, (n_heads + 2 n_kv_heads) * D] (q | k | v; rows may be strided), positions [N] int64 or int32, inv_freq [D/2] fp32,
  halves convention (x1 | x2), both halves scaled by ``conc``.  slots [N] int32: cache slot of each token, negative = store
  nothing; the others are distinct.  Returns q [N, n_heads, D] and, with ``need_kv``, rotated k and v [N, n_kv_heads, D]
  (else None).  A slot past the cache is skipped and shows up in ``check_status``."""
  heads = n_heads + 2 * n_kv_heads
  _need(n_heads > 0 and n_kv_heads > 0 and qkv.dim() == 2 and qkv.size(1) % heads == 0, "qkv must be [N, (n_heads + 2 n_kv_heads) * D]")
  N, D = qkv.size(0), qkv.size(1) // heads
  dev = qkv.device
  _need(positions.shape == (N,) and positions.dtype in (torch.int64, torch.int32) and positions.device == dev,
        "positions must be [N] int64 or int32 on qkv's device")
  _need(inv_freq.shape == (D // 2,) and inv_freq.dtype == torch.float32 and D % 2 == 0 and inv_freq.device == dev,
        "inv_freq must be [D/2] fp32 on qkv's device")
  _need((slots is None) == (k_cache is None) == (v_cache is None), "slots, k_cache and v_cache go together")
  if slots is not None:
    _check_cache(k_cache, v_cache, qkv, n_kv_heads, D)
    _check_ints(dev, slots=slots)
    _need(slots.shape == (N,), "slots must be [N]")
  if not qkv.is_cuda:
    q, k, v = rope_append_reference(qkv, positions, inv_freq, conc, n_heads, n_kv_heads, k_cache, v_cache, slots)
    return (q, k, v) if need_kv else (q, None, None)
  _need(qkv.dtype == torch.bfloat16, "the CUDA kernel takes bf16")
  _need(D % 16 == 0 and D <= 512, f"head dim {D}: the kernel takes multiples of 16 up to 512")
  if qkv.stride(1) != 1 or (N > 1 and qkv.stride(0) % 8 != 0) or not _aligned(qkv):
    qkv = qkv.clone(memory_format=torch.contiguous_format)      # odd strides or start: one copy brings the rows to 16-byte boundaries
  positions, inv_freq = positions.contiguous(), inv_freq.contiguous()
  n_slots = 0
  if slots is not None:
    slots = slots.contiguous()
    n_slots = k_cache.size(0) * k_cache.size(1)
    _need(_aligned(k_cache) and _aligned(v_cache), "the cache must start on a 16-byte boundary")
  with _on(dev):
    q = torch.empty(N, n_heads, D, dtype=qkv.dtype, device=dev)
    k = torch.empty(N, n_kv_heads, D, dtype=qkv.dtype, device=dev) if need_kv else None
    v = torch.empty_like(k) if need_kv else None
    L.check(_fn("nmoe_rope_append", "plpipfppplpppiiiipp")(
      _p(qkv), qkv.stride(0) if N > 1 else qkv.size(1), _p(positions), int(positions.dtype == torch.int64), _p(inv_freq), conc, _p(slots), _p(k_cache),
      _p(v_cache), n_slots, _p(q), _p(k), _p(v), N, n_heads, n_kv_heads, D, _p(status_buffer(dev)), _stream()), "rope_append")
  return q, k, v


# ------------------------------------------------------------------ several query tokens per sequence
def paged_extend_reference(q, k_cache, v_cache, block_tables, context_lens, q_starts, q_lens, sinks, scale, window=0, out=None):
  """Plain statement of ``paged_extend`` in fp32, sequence by sequence."""
  N, Hq, D = q.shape
  _, bs, Hkv, _ = k_cache.shape
  g = Hq // Hkv
  out = torch.zeros_like(q) if out is None else out
  for b in range(context_lens.numel()):
    s0, n, ctx = int(q_starts[b]), int(q_lens[b]), int(context_lens[b])
    if n == 0:
      continue
    pos = torch.arange(ctx, device=q.device)
    slot = block_tables[b, pos // bs].long() * bs + pos % bs
    k = k_cache.view(-1, Hkv, D)[slot].float().repeat_interleave(g, dim=1)                # [ctx, Hq, D]
    v = v_cache.view(-1, Hkv, D)[slot].float().repeat_interleave(g, dim=1)
    s = torch.einsum("nhd,khd->hnk", q[s0:s0 + n].float(), k) * scale
    at = torch.arange(ctx - n, ctx, device=q.device).unsqueeze(1)
    seen = pos <= at
    if window > 0:
      seen = seen & (pos > at - window)
    s = s.masked_fill(~seen, float("-inf"))
    sk = torch.full((Hq, n, 1), float("-inf"), device=q.device) if sinks is None else sinks.float().view(Hq, 1, 1).expand(Hq, n, 1)
    p = torch.softmax(torch.cat((s, sk), dim=-1), dim=-1)[..., :-1].nan_to_num(0.0)       # a row that sees nothing gives zeros
    out[s0:s0 + n] = torch.einsum("hnk,khd->nhd", p, v).to(out.dtype)
  return out


def _check_attention(q, k_cache, v_cache, block_tables, context_lens, sinks, scale, window):
  _need(q.dim() == 3, "q must be [N, Hq, D]")
  _need(k_cache.dim() == 4, "k_cache and v_cache must be [num_blocks, block_size, Hkv, D]")
  Hq, D, Hkv, B = q.size(1), q.size(2), k_cache.size(2), context_lens.numel()
  _need(Hkv > 0 and Hq % Hkv == 0, f"{Hq} query heads cannot be grouped over {Hkv} key/value heads")
  _check_cache(k_cache, v_cache, q, Hkv, D)
  _check_ints(q.device, block_tables=block_tables, context_lens=context_lens)
  _need(block_tables.dim() == 2 and block_tables.size(0) == B and context_lens.dim() == 1, "block_tables must be [B, n], context_lens [B]")
  _need(sinks is None or (sinks.shape == (Hq,) and sinks.device == q.device), "sinks must be [Hq] on q's device")
  _need(window >= 0, "window must not be negative")
  _need(scale > 0, "scale must be positive")


def _attention_args(q, k_cache, v_cache, block_tables, sinks):
  """What the kernel asks of its operands beyond the checks above; q and sinks may come back as copies."""
  _need(q.dtype == torch.bfloat16, "the CUDA kernel takes bf16")
  _need(q.size(2) in (64, 128), f"head dim {q.size(2)}: the kernel takes 64 and 128")
  _need(_aligned(k_cache) and _aligned(v_cache), "the cache must start on a 16-byte boundary")
  _need(block_tables.stride(1) == 1 or block_tables.size(1) <= 1, "the rows of block_tables must be dense")
  if q.stride(2) != 1 or q.stride(1) != q.size(2) or (q.size(0) > 1 and q.stride(0) % 8 != 0) or not _aligned(q):
    q = q.clone(memory_format=torch.contiguous_format)
  if sinks is not None:
    sinks = sinks.detach()
    sinks = sinks.contiguous() if sinks.dtype in (torch.bfloat16, torch.float32) else sinks.float().contiguous()
  return q, sinks


def _attend(what, q, k_cache, v_cache, block_tables, context_lens, q_starts, q_lens, sinks, out, scale, window, max_q_len, prefix_len):
  """The launch behind ``paged_extend`` and ``shared_prefix_decode`` (on q's device)."""
  N, Hq, D = q.shape
  sizes = N, context_lens.numel(), Hq, k_cache.size(2), D
  need = _fn("nmoe_paged_extend_workspace", "iiiiiiiiii", ctypes.c_longlong)(
    *sizes, k_cache.size(1), block_tables.size(1), max_q_len, window, prefix_len)
  # partial results (O, m, l) where the keys of a row are split over more CTAs than exchange them directly
  work = torch.empty(need, dtype=torch.float32, device=q.device) if need else None
  L.check(_fn("nmoe_paged_extend", "plppplppppipiiiiiiiiiifiplpp")(
    _p(q), q.stride(0), _p(k_cache), _p(v_cache), _p(block_tables), block_tables.stride(0), _p(context_lens), _p(q_starts),
    _p(q_lens), _p(sinks), int(sinks is not None and sinks.dtype == torch.float32), _p(out), *sizes, k_cache.size(1), k_cache.size(0),
    block_tables.size(1), max_q_len, window, scale, prefix_len, _p(work), need, _p(status_buffer(q.device)), _stream()),
    what, 2 if need else 1)


def paged_extend(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                 context_lens: torch.Tensor, q_starts: torch.Tensor, q_lens: torch.Tensor, sinks: Optional[torch.Tensor],
                 scale: float, window: int = 0, *, max_q_len: Optional[int] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
  """Attention of ``q_lens[b]`` new tokens per sequence over the paged cache, which already holds their K/V.

  q [N, Hq, D]: the tokens of sequence b are rows q_starts[b] .. q_starts[b] + q_lens[b] - 1 (sequences do not overlap; gaps
  are fine); its token j stands at position context_lens[b] - q_lens[b] + j and sees the keys at or before it, of those the
  last ``window`` if that is positive.  sinks [Hq]: a logit per head that only enters the denominator.  A token that sees no
  key gives zeros.  Rows of no sequence are zero in the result, or left as they were in ``out`` [N, Hq, D].
  ``max_q_len``: an upper bound of q_lens known to the host (default N); with a tight one fewer empty blocks are launched.
  Lengths or pages outside their tensors are skipped and show up in ``check_status``."""
  _check_attention(q, k_cache, v_cache, block_tables, context_lens, sinks, scale, window)
  N, Hq, D = q.shape
  B = context_lens.numel()
  _check_ints(q.device, q_starts=q_starts, q_lens=q_lens)
  _need(q_starts.shape == (B,) and q_lens.shape == (B,), "q_starts and q_lens must be [B]")
  max_q_len = N if max_q_len is None else int(max_q_len)
  _need(max_q_len >= 0, "max_q_len must not be negative")
  if out is not None:
    _need(out.shape == q.shape and out.dtype == q.dtype and out.device == q.device and out.is_contiguous(), "out must be contiguous and like q")
  if not q.is_cuda:
    return paged_extend_reference(q, k_cache, v_cache, block_tables, context_lens, q_starts, q_lens, sinks, scale, window, out)
  q, sinks = _attention_args(q, k_cache, v_cache, block_tables, sinks)
  context_lens, q_starts, q_lens = context_lens.contiguous(), q_starts.contiguous(), q_lens.contiguous()
  with _on(q.device):
    out = torch.zeros(N, Hq, D, dtype=q.dtype, device=q.device) if out is None else out
    _need(_aligned(out), "out must start on a 16-byte boundary")
    _attend("paged_extend", q, k_cache, v_cache, block_tables, context_lens, q_starts, q_lens, sinks, out, scale, window,
            min(max_q_len, N), 0)
  return out


# ------------------------------------------------------------------ a batch behind one prefix
def shared_prefix_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                         context_lens: torch.Tensor, prefix_len: int, sinks: Optional[torch.Tensor], scale: float,
                         window: int = 0) -> torch.Tensor:
  """``paged_decode`` for a batch whose sequences all start with the same ``prefix_len`` tokens: their keys and values are
  read once for the whole batch, through the first sequence's pages, instead of once per sequence.

  q [B, Hq, D] -> [B, Hq, D]; block_tables [B, n] hold every sequence's whole table (prefix pages included; where the prefix
  ends inside a page, each table may have its own copy of that page).  ``context_lens`` counts the current token; a sequence
  with a context of 0 (a padding row) gives zeros, one shorter than the prefix sees its part of it."""
  _check_attention(q, k_cache, v_cache, block_tables, context_lens, sinks, scale, window)
  B, Hq, D = q.shape
  _need(context_lens.numel() == B, "q must hold one token per sequence")
  _need(0 <= prefix_len <= block_tables.size(1) * k_cache.size(1), "prefix_len must lie within the block tables")
  if not q.is_cuda:
    one = torch.ones_like(context_lens)
    return paged_extend_reference(q, k_cache, v_cache, block_tables, context_lens, torch.cumsum(one, 0) - 1,
                                  torch.minimum(one, context_lens), sinks, scale, window)
  q, sinks = _attention_args(q, k_cache, v_cache, block_tables, sinks)
  context_lens = context_lens.contiguous()
  with _on(q.device):
    out = torch.empty(B, Hq, D, dtype=q.dtype, device=q.device)
    _attend("shared_prefix_decode", q, k_cache, v_cache, block_tables, context_lens, None, None, sinks, out, scale, window, 1,
            prefix_len)
  return out


# ------------------------------------------------------------------ drafted tokens
def verify_draft_reference(target_probs, tokens, uniforms, q_starts, q_lens, draft_probs=None, out=None):
  """Plain statement of ``verify_draft`` in fp64."""
  out = torch.full((tokens.numel(),), -1, dtype=torch.int32) if out is None else out
  n_out = torch.zeros(q_lens.numel(), dtype=torch.int32)
  u = uniforms.double()
  for b, (s0, n) in enumerate(zip(q_starts.tolist(), q_lens.tolist())):
    if n == 0:
      continue
    j = 1
    while j < n:
      x = int(tokens[s0 + j])
      qx = 1.0 if draft_probs is None else float(draft_probs[s0 + j, x])
      if not float(u[s0 + j]) * qx < float(target_probs[s0 + j - 1, x]):
        break
      j += 1
    p = target_probs[s0 + j - 1].double()
    w = p
    if j < n:
      if draft_probs is None:
        w = p.clone()
        w[int(tokens[s0 + j])] = 0.0
      else:
        w = (p - draft_probs[s0 + j].double()).clamp_(min=0.0)
      if not float(w.sum()) > 0.0:
        w = p
    c = w.cumsum(0)
    hit = ((c > float(u[s0]) * float(w.sum())) & (w > 0)).nonzero()
    pos = (w > 0).nonzero()
    new = int(hit[0]) if hit.numel() else int(pos[-1]) if pos.numel() else w.numel() - 1
    out[s0:s0 + n] = -1
    out[s0:s0 + j - 1] = tokens[s0 + 1:s0 + j].to(torch.int32)
    out[s0 + j - 1] = new
    n_out[b] = j
  return out, n_out


def verify_draft(target_probs: torch.Tensor, tokens: torch.Tensor, uniforms: torch.Tensor, q_starts: torch.Tensor,
                 q_lens: torch.Tensor, draft_probs: Optional[torch.Tensor] = None, *, out: Optional[torch.Tensor] = None
                 ) -> Tuple[torch.Tensor, torch.Tensor]:
  """Accepts or redraws drafted tokens so that the emitted ones are distributed as draws from the target.

  The rows are those of the step that scored them: sequence b owns rows q_starts[b] .. + q_lens[b] - 1, ``tokens`` [N] holds
  its last known token in the first and the drafted ones behind it, ``target_probs`` [N, V] fp32 the target's probabilities
  AFTER each row's token.  ``draft_probs`` [N, V] fp32: row r = the distribution that the token at row r was drawn from (the
  first row of a sequence is not read); None = looked-up tokens, drawn with certainty.  ``uniforms`` [N] fp32 in [0, 1): row r
  decides over the token at row r (it passes while u * q(x) < p(x)), the first row's number over the one that is drawn: from
  max(p - q, 0) at the first token that fails, from the last row's p if none does.  Rows need not add up to 1; entries are
  finite and not negative.

  Returns (out [N] int32: the emitted tokens from row q_starts[b] on, -1 behind them; n_out [B] int32: how many, at least 1
  for a sequence with rows).  Rows of no sequence are -1, or left as they were in a given ``out``.  A drafted token outside
  the vocabulary fails and shows up in ``check_status``."""
  _need(target_probs.dim() == 2 and target_probs.size(1) > 0, "target_probs must be [N, V]")
  N, V = target_probs.shape
  B, dev = q_lens.numel(), target_probs.device
  _need(target_probs.dtype == torch.float32, "target_probs must be fp32")
  _need(draft_probs is None or (draft_probs.shape == (N, V) and draft_probs.dtype == torch.float32 and draft_probs.device == dev),
        "draft_probs must be like target_probs")
  _need(tokens.shape == (N,) and tokens.dtype in (torch.int64, torch.int32) and tokens.device == dev, "tokens must be [N] int64 or int32")
  _need(uniforms.shape == (N,) and uniforms.dtype == torch.float32 and uniforms.device == dev, "uniforms must be [N] fp32")
  _check_ints(dev, q_starts=q_starts, q_lens=q_lens, out=out)
  _need(q_starts.shape == (B,) and q_lens.shape == (B,), "q_starts and q_lens must be [B]")
  _need(out is None or (out.shape == (N,) and out.is_contiguous()), "out must be a contiguous [N]")
  if not target_probs.is_cuda:
    return verify_draft_reference(target_probs, tokens, uniforms, q_starts, q_lens, draft_probs, out)
  if target_probs.stride(1) != 1 and V > 1:
    target_probs = target_probs.contiguous()
  if draft_probs is not None and draft_probs.stride(1) != 1 and V > 1:
    draft_probs = draft_probs.contiguous()
  tokens, uniforms, q_starts, q_lens = tokens.contiguous(), uniforms.contiguous(), q_starts.contiguous(), q_lens.contiguous()
  with _on(dev):
    out = torch.full((N,), -1, dtype=torch.int32, device=dev) if out is None else out
    n_out = torch.empty(B, dtype=torch.int32, device=dev)
    L.check(_fn("nmoe_verify_draft", "plplpippppp" + "iiipp")(
      _p(target_probs), target_probs.stride(0), _p(draft_probs), 0 if draft_probs is None else draft_probs.stride(0), _p(tokens),
      int(tokens.dtype == torch.int64), _p(uniforms), _p(q_starts), _p(q_lens), _p(out), _p(n_out), N, B, V,
      _p(status_buffer(dev)), _stream()), "verify_draft")
  return out, n_out
