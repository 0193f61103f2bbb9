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
import functools
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
# A decode step calls these once a layer with a few microseconds of device work each, so the checks are written to cost
# little where they pass: attributes are read once, messages are built only on the way out.
_HERE = contextlib.nullcontext()


def _on(device: torch.device):
  """Launches go to the current stream of the tensors' own device, whichever device is current."""
  return _HERE if device.index == torch.cuda.current_device() else torch.cuda.device(device)


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


def _stream(device: torch.device) -> int:
  return torch._C._cuda_getCurrentRawStream(device.index)       # torch.cuda.current_stream builds a Stream object every time


@functools.lru_cache(maxsize=1024)
def _attend_plan(N: int, *sizes: int) -> Tuple[int, int]:
  """Floats of partial results and number of launches of a call of these sizes; a function of the sizes alone."""
  return (_fn("nmoe_paged_extend_workspace", "iiiiiiiiii", ctypes.c_longlong)(N, *sizes),
          _fn("nmoe_paged_extend_launches", "iiiiiiiii")(*sizes))


def _check_cache(k_cache: torch.Tensor, v_cache: torch.Tensor, like: torch.Tensor, Hkv: int, D: int) -> None:
  shape, dt, dev = k_cache.shape, like.dtype, like.device
  if len(shape) != 4 or shape != v_cache.shape:
    raise ValueError("k_cache and v_cache must be [num_blocks, block_size, Hkv, D]")
  if shape[2] != Hkv or shape[3] != D:
    raise ValueError(f"the cache holds {tuple(shape[2:])} heads x dims, expected ({Hkv}, {D})")
  if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
    raise ValueError("k_cache and v_cache must be contiguous")
  if k_cache.dtype != dt or v_cache.dtype != dt:
    raise ValueError("the cache and the activations must have one dtype")
  if k_cache.device != dev or v_cache.device != dev:
    raise ValueError("the cache must be on the activations' device")
  if like.is_cuda and (k_cache.data_ptr() | v_cache.data_ptr()) % 16 != 0:
    raise ValueError("the cache must start on a 16-byte boundary")


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
  """Whether the stretches of memory from the first to the last element of two non-empty tensors meet."""
  def span(t):
    first = t.data_ptr()
    return first, first + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()
  (a0, a1), (b0, b1) = span(a), span(b)
  return a0 < b1 and b0 < a1


def _check_int32(t: torch.Tensor, device: torch.device, what: str) -> None:
  if t.dtype != torch.int32 or t.device != device:
    raise ValueError(f"{what} must be int32 on {device}")


def _report(device: torch.device, where: int, a: int, b: int = 0) -> None:
  """An index that a plain statement skips, in the status record of its device (code 2, as the kernels write it)."""
  rec = status_buffer(device)
  if int(rec[0]) == 0:
    rec.copy_(torch.tensor([2, where, a, b]).clamp(-2 ** 31, 2 ** 31 - 1))


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
    past = (slots >= k_cache.size(0) * k_cache.size(1)).nonzero()
    if past.numel():
      _report(qkv.device, 1000, int(past[0]), int(slots[past[0]]))
    ok = (slots >= 0) & (slots < k_cache.size(0) * k_cache.size(1))
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
  if n_heads <= 0 or n_kv_heads <= 0 or qkv.dim() != 2 or qkv.size(1) % heads != 0:
    raise ValueError("qkv must be [N, (n_heads + 2 n_kv_heads) * D]")
  N, width = qkv.shape
  D, dev = width // heads, qkv.device
  if positions.shape != (N,) or positions.dtype not in (torch.int64, torch.int32) or positions.device != dev:
    raise ValueError("positions must be [N] int64 or int32 on qkv's device")
  if inv_freq.shape != (D // 2,) or inv_freq.dtype != torch.float32 or D % 2 != 0 or inv_freq.device != dev:
    raise ValueError("inv_freq must be [D/2] fp32 on qkv's device")
  n_slots = 0
  if slots is None or k_cache is None or v_cache is None:
    if not (slots is None and k_cache is None and v_cache is None):
      raise ValueError("slots, k_cache and v_cache go together")
  else:
    _check_cache(k_cache, v_cache, qkv, n_kv_heads, D)
    _check_int32(slots, dev, "slots")
    if slots.shape != (N,):
      raise ValueError("slots must be [N]")
    slots = slots.contiguous()
    n_slots = k_cache.size(0) * k_cache.size(1)
  if not qkv.is_cuda:
    q, k, v = rope_append_reference(qkv, positions, inv_freq, conc, n_heads, n_kv_heads, k_cache, v_cache, slots)
    return (q, k, v) if need_kv else (q, None, None)
  if qkv.dtype != torch.bfloat16:
    raise ValueError("the CUDA kernel takes bf16")
  if D % 16 != 0 or D > 512:
    raise ValueError(f"head dim {D}: the kernel takes multiples of 16 up to 512")
  row = qkv.stride(0) if N > 1 else width
  if row % 8 != 0 or qkv.data_ptr() % 16 != 0 or qkv.stride(1) != 1:
    qkv, row = qkv.clone(memory_format=torch.contiguous_format), width    # one copy brings the rows to 16-byte boundaries
  positions, inv_freq = positions.contiguous(), inv_freq.contiguous()
  with _on(dev):
    q = torch.empty((N, n_heads, D), dtype=torch.bfloat16, device=dev)
    k = torch.empty((N, n_kv_heads, D), dtype=torch.bfloat16, device=dev) if need_kv else None
    v = torch.empty_like(k) if need_kv else None
    L.check(_fn("nmoe_rope_append", "plpipfppplpppiiiipp")(
      qkv.data_ptr(), row, positions.data_ptr(), positions.dtype == torch.int64, inv_freq.data_ptr(), conc, _p(slots), _p(k_cache),
      _p(v_cache), n_slots, q.data_ptr(), _p(k), _p(v), N, n_heads, n_kv_heads, D, status_buffer(dev).data_ptr(), _stream(dev)),
      "rope_append")
  return q, k, v


# ------------------------------------------------------------------ several query tokens per sequence
def paged_extend_reference(q, k_cache, v_cache, block_tables, context_lens, q_starts, q_lens, sinks, scale, window=0, out=None,
                           max_q_len=None):
  """Plain statement of ``paged_extend`` in fp32, sequence by sequence."""
  N, Hq, D = q.shape
  num_blocks, bs, Hkv, _ = k_cache.shape
  g = Hq // Hkv
  out = torch.zeros_like(q) if out is None else out
  capacity = block_tables.size(1) * bs
  for b in range(context_lens.numel()):
    s0, n, ctx = int(q_starts[b]), int(q_lens[b]), max(int(context_lens[b]), 0)
    if s0 < 0 or n < 0 or s0 + n > N or (max_q_len is not None and n > max_q_len):
      _report(q.device, 1020, b, s0)
      continue
    if n == 0:
      continue
    if ctx > capacity:
      _report(q.device, 1021, b, ctx)
      ctx = capacity
    first = max(0, ctx - n - window + 1) if window > 0 else 0                             # the oldest key that any of them sees
    pos = torch.arange(first, ctx, device=q.device)
    page = block_tables[b, pos // bs].long()
    there = (page >= 0) & (page < num_blocks)
    if not bool(there.all()):
      _report(q.device, 1022, b)
    slot = torch.where(there, page, 0) * bs + pos % bs
    none = ~there.view(-1, 1, 1)
    k, v = (c.view(-1, Hkv, D)[slot].float().masked_fill(none, 0.0).repeat_interleave(g, dim=1) if num_blocks else
            torch.zeros(ctx - first, Hq, D, device=q.device) for c in (k_cache, v_cache))             # [m, Hq, D]
    s = torch.einsum("nhd,khd->hnk", q[s0:s0 + n].float(), k) * scale
    at = torch.arange(ctx - n, ctx, device=q.device).unsqueeze(1)
    seen = pos <= at
    if window > 0:
      seen = seen & (pos > at - window)
    s = s.masked_fill(~seen, float("-inf"))
    sk = torch.full((Hq, n, 1), float("-inf"), device=q.device) if sinks is None else sinks.float().view(Hq, 1, 1).expand(Hq, n, 1)
    p = torch.softmax(torch.cat((s, sk), dim=-1), dim=-1)[..., :-1].masked_fill(~seen.any(-1).unsqueeze(-1), 0.0)
    out[s0:s0 + n] = torch.einsum("hnk,khd->nhd", p, v).to(out.dtype)
  return out


def _check_attention(q, k_cache, v_cache, block_tables, context_lens, sinks, scale, window):
  """Checks what both attention operators ask for; q and sinks come back as the kernel takes them."""
  if q.dim() != 3:
    raise ValueError("q must be [N, Hq, D]")
  if k_cache.dim() != 4:
    raise ValueError("k_cache and v_cache must be [num_blocks, block_size, Hkv, D]")
  N, Hq, D = q.shape
  Hkv, dev = k_cache.size(2), q.device
  if Hkv == 0 or Hq % Hkv != 0:
    raise ValueError(f"{Hq} query heads cannot be grouped over {Hkv} key/value heads")
  _check_cache(k_cache, v_cache, q, Hkv, D)
  _check_int32(block_tables, dev, "block_tables")
  _check_int32(context_lens, dev, "context_lens")
  if context_lens.dim() != 1 or block_tables.dim() != 2 or block_tables.size(0) != context_lens.size(0):
    raise ValueError("block_tables must be [B, n], context_lens [B]")
  if sinks is not None and (sinks.shape != (Hq,) or sinks.device != dev):
    raise ValueError("sinks must be [Hq] on q's device")
  if not 0 <= window < 2 ** 31:
    raise ValueError("window must not be negative, nor pass 32 bits")
  if not scale > 0:
    raise ValueError("scale must be positive")
  if not q.is_cuda:
    return q, sinks
  if q.dtype != torch.bfloat16:
    raise ValueError("the CUDA kernel takes bf16")
  if D != 64 and D != 128:
    raise ValueError(f"head dim {D}: the kernel takes 64 and 128")
  if block_tables.size(1) > 1 and block_tables.stride(1) != 1:
    raise ValueError("the rows of block_tables must be dense")
  if not q.is_contiguous() and (q.stride(2) != 1 or q.stride(1) != D or q.stride(0) % 8 != 0) or q.data_ptr() % 16 != 0:
    q = q.clone(memory_format=torch.contiguous_format)
  if sinks is not None:
    sinks = sinks.detach().contiguous()
    if sinks.dtype != torch.bfloat16 and sinks.dtype != torch.float32:
      sinks = sinks.float()
  return q, sinks


def _attend(what, q, k_cache, v_cache, block_tables, context_lens, q_starts, q_lens, sinks, out, scale, window, max_q_len, prefix_len):
  """The launch behind ``paged_extend`` and ``shared_prefix_decode`` (on q's device)."""
  N, Hq, D = q.shape
  num_blocks, block_size, Hkv, _ = k_cache.shape
  B, width, dev = context_lens.size(0), block_tables.size(1), q.device
  need, launches = _attend_plan(N, B, Hq, Hkv, D, block_size, width, max_q_len, window, prefix_len)
  # partial results (O, m, l) where the keys of a row are split over more CTAs than exchange them directly
  work = torch.empty((need,), dtype=torch.float32, device=dev) if need else None
  L.check(_fn("nmoe_paged_extend", "plppplppppipiiiiiiiiiifiplpp")(
    q.data_ptr(), q.stride(0), k_cache.data_ptr(), v_cache.data_ptr(), block_tables.data_ptr(), block_tables.stride(0),
    context_lens.data_ptr(), _p(q_starts), _p(q_lens), _p(sinks), sinks is not None and sinks.dtype == torch.float32, out.data_ptr(),
    N, B, Hq, Hkv, D, block_size, num_blocks, width, max_q_len, window, scale, prefix_len, _p(work), need,
    status_buffer(dev).data_ptr(), _stream(dev)), what, launches)


def paged_extend(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                 context_lens: torch.Tensor, q_starts: torch.Tensor, q_lens: torch.Tensor, sinks: Optional[torch.Tensor],
                 scale: float, window: int = 0, *, max_q_len: Optional[int] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
  """Attention of ``q_lens[b]`` new tokens per sequence over the paged cache, which already holds their K/V.

  q [N, Hq, D]: the tokens of sequence b are rows q_starts[b] .. q_starts[b] + q_lens[b] - 1 (sequences do not overlap; gaps
  are fine); its token j stands at position context_lens[b] - q_lens[b] + j and sees the keys at or before it, of those the
  last ``window`` if that is positive.  sinks [Hq]: a logit per head that only enters the denominator.  A token that sees no
  key gives zeros, a context below 0 counts as 0.  Rows of no sequence are zero in the result, or left as they were in ``out``
  [N, Hq, D] (which may be q itself).  K and V of the positions before ``context_lens[b]`` (within the window of the first new token) are finite; what else the pages hold does not matter.
  ``max_q_len``: an upper bound of q_lens known to the host (default N); with a tight one fewer empty blocks are launched.  Where it
  is one token, or at most 128 rows of a KV head (max_q_len * Hq / Hkv), the result is rounded once, as that of ``paged_decode``; beyond, in prompts,
  the probabilities are rounded to bf16 before they meet the values, as in dense attention.
  Sequences whose rows lie outside q or exceed ``max_q_len`` are skipped, contexts longer than their table are cut, pages
  outside the cache count as zeros: all three show up in ``check_status``."""
  given = q
  q, sinks = _check_attention(q, k_cache, v_cache, block_tables, context_lens, sinks, scale, window)
  dev, N = q.device, q.size(0)
  _check_int32(q_starts, dev, "q_starts")
  _check_int32(q_lens, dev, "q_lens")
  if q_starts.shape != context_lens.shape or q_lens.shape != context_lens.shape:
    raise ValueError("q_starts and q_lens must be [B]")
  max_q_len = N if max_q_len is None else int(max_q_len)
  if max_q_len < 0:
    raise ValueError("max_q_len must not be negative")
  if out is not None and (out.shape != given.shape or out.dtype != given.dtype or out.device != dev or not out.is_contiguous()):
    raise ValueError("out must be contiguous and like q")
  if out is not None and N > 0 and (out.data_ptr() != given.data_ptr() or not given.is_contiguous()) and _overlap(out, given):
    raise ValueError("out must be q itself or not overlap it: rows are written while others are read")
  if not q.is_cuda:
    return paged_extend_reference(q, k_cache, v_cache, block_tables, context_lens, q_starts, q_lens, sinks, scale, window, out, max_q_len)
  if out is not None and out.data_ptr() % 16 != 0:
    raise ValueError("out must start on a 16-byte boundary")
  with _on(dev):
    if out is None:
      out = torch.zeros(q.shape, dtype=q.dtype, device=dev)
    _attend("paged_extend", q, k_cache, v_cache, block_tables, context_lens.contiguous(), q_starts.contiguous(), q_lens.contiguous(),
            sinks, out, scale, window, min(max_q_len, N), 0)
  return out


# ------------------------------------------------------------------ a batch behind one prefix
def shared_prefix_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                         context_lens: torch.Tensor, prefix_len: int, sinks: Optional[torch.Tensor], scale: float,
                         window: int = 0) -> torch.Tensor:
  """``paged_decode`` for a batch whose sequences all start with the same ``prefix_len`` tokens: their keys and values are
  read once for the whole batch, through the pages of the first sequence that has them all, instead of once per sequence.

  q [B, Hq, D] -> [B, Hq, D]; block_tables [B, n] hold every sequence's whole table (prefix pages included; where the prefix
  ends inside a page, each table may have its own copy of that page).  ``context_lens`` counts the current token; a sequence
  with a context of 0 (a padding row) gives zeros, one shorter than the prefix sees its part of it."""
  q, sinks = _check_attention(q, k_cache, v_cache, block_tables, context_lens, sinks, scale, window)
  if context_lens.size(0) != q.size(0):
    raise ValueError("q must hold one token per sequence")
  if not 0 <= prefix_len <= block_tables.size(1) * k_cache.size(1):
    raise ValueError("prefix_len must lie within the block tables")
  if not q.is_cuda:
    one = torch.ones_like(context_lens)
    return paged_extend_reference(q, k_cache, v_cache, block_tables, context_lens, torch.cumsum(one, 0) - 1,
                                  context_lens.clamp(0, 1), sinks, scale, window)
  with _on(q.device):
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    _attend("shared_prefix_decode", q, k_cache, v_cache, block_tables, context_lens.contiguous(), None, None, sinks, out, scale, window,
            1, prefix_len)
  return out


# ------------------------------------------------------------------ drafted tokens
def verify_draft_reference(target_probs, tokens, uniforms, q_starts, q_lens, draft_probs=None, out=None):
  """Plain statement of ``verify_draft`` in fp64."""
  out = torch.full((tokens.numel(),), -1, dtype=torch.int32) if out is None else out
  n_out = torch.zeros(q_lens.numel(), dtype=torch.int32)
  u = uniforms.double()
  N, V = target_probs.shape
  for b, (s0, n) in enumerate(zip(q_starts.tolist(), q_lens.tolist())):
    if s0 < 0 or n < 0 or s0 + n > N:
      _report(tokens.device, 1010, b, s0)
      continue
    if n == 0:
      continue
    j = 1
    while j < n:
      x = int(tokens[s0 + j])
      if not 0 <= x < V:
        _report(tokens.device, 1011, s0 + j, x)
        break
      qx = 1.0 if draft_probs is None else float(draft_probs[s0 + j, x])
      if not float(u[s0 + j]) * qx < float(target_probs[s0 + j - 1, x]):
        break
      j += 1
    p = target_probs[s0 + j - 1].double()
    w = p
    if j < n:
      if draft_probs is None:
        w = p.clone()
        if 0 <= int(tokens[s0 + j]) < V:
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
  the vocabulary fails, a sequence whose rows lie outside the inputs is skipped with a count of 0; both show up in ``check_status``."""
  if target_probs.dim() != 2 or not 0 < target_probs.size(1) <= 2 ** 30:
    raise ValueError("target_probs must be [N, V], V up to 2^30")
  N, V = target_probs.shape
  dev = target_probs.device
  if target_probs.dtype != torch.float32:
    raise ValueError("target_probs must be fp32")
  if draft_probs is not None and (draft_probs.shape != (N, V) or draft_probs.dtype != torch.float32 or draft_probs.device != dev):
    raise ValueError("draft_probs must be like target_probs")
  if tokens.shape != (N,) or tokens.dtype not in (torch.int64, torch.int32) or tokens.device != dev:
    raise ValueError("tokens must be [N] int64 or int32 on target_probs' device")
  if uniforms.shape != (N,) or uniforms.dtype != torch.float32 or uniforms.device != dev:
    raise ValueError("uniforms must be [N] fp32 on target_probs' device")
  _check_int32(q_starts, dev, "q_starts")
  _check_int32(q_lens, dev, "q_lens")
  if q_starts.dim() != 1 or q_starts.shape != q_lens.shape:
    raise ValueError("q_starts and q_lens must be [B]")
  if out is not None:
    _check_int32(out, dev, "out")
    if out.shape != (N,) or not out.is_contiguous():
      raise ValueError("out must be a contiguous [N]")
    if N > 0 and _overlap(out, tokens):
      raise ValueError("out must not overlap tokens, which are read while it is written")
  if not target_probs.is_cuda:
    return verify_draft_reference(target_probs, tokens, uniforms, q_starts, q_lens, draft_probs, out)
  if target_probs.stride(1) != 1 and V > 1:
    target_probs = target_probs.contiguous()
  if draft_probs is not None and draft_probs.stride(1) != 1 and V > 1:
    draft_probs = draft_probs.contiguous()
  tokens, uniforms, q_starts, q_lens = tokens.contiguous(), uniforms.contiguous(), q_starts.contiguous(), q_lens.contiguous()
  with _on(dev):
    out = torch.full((N,), -1, dtype=torch.int32, device=dev) if out is None else out
    n_out = torch.empty(q_lens.shape, dtype=torch.int32, device=dev)
    L.check(_fn("nmoe_verify_draft", "plplpippppp" + "iiipp")(
      target_probs.data_ptr(), target_probs.stride(0), _p(draft_probs), 0 if draft_probs is None else draft_probs.stride(0),
      tokens.data_ptr(), tokens.dtype == torch.int64, uniforms.data_ptr(), q_starts.data_ptr(), q_lens.data_ptr(), out.data_ptr(),
      n_out.data_ptr(), N, q_lens.size(0), V, status_buffer(dev).data_ptr(), _stream(dev)), "verify_draft")
  return out, n_out
