"""Continuous-batching inference engine over the paged KV cache.

  eng = Engine(model, max_seq_len=4096, max_batch=128)
  sid = eng.add(prompt_tokens, max_new_tokens=64)
  while not eng.idle:
      logits, ids = eng.step()            # one prefill batch or one decode step
      for row, sid in zip(logits, ids):
          tok = int(row.argmax())
          eng.update(sid, tok, finished=tok in stop_tokens)

Each ``step`` either admits waiting requests (as many as fit in the batch and in the cache; their
prompts are prefilled together, minus any prefix already in the cache) or advances every running
sequence by one token.  ``generate`` wraps the loop for greedy / top-k sampling; ``hidden_states``
runs prompts through the first layers only (the probe / judge taps of the curation stack).

Two things shorten decoding.  Blocks that every running sequence has in common (a grading rubric, a
few-shot header) are attended to once per step for the whole batch (steps in which nobody has drafts).  And with ``draft_tokens`` > 0
``generate`` lets each sequence propose that many tokens per step by looking its last tokens up in
its own text (answers that quote their prompt, structured output); one pass scores them all and
those that fit are kept.  Greedy output is what it would be without drafts (on the GPU as far as the
rounding of two kernels leaves near-ties alone), sampled output has the same distribution.

Behavioural counterpart: ``BatchedGenerator`` (nmoe/data/model.py:650-790).  Differences: prefix
blocks found in the cache are really attended to during prefill, the host-side batch assembly is
vectorised, and a request that cannot get a cache block is preempted back to the queue instead of
raising.
"""
from __future__ import annotations

import itertools
from collections import deque
from typing import Callable, Deque, Dict, Iterable, List, Optional, Sequence as Seq, Tuple

import numpy as np
import torch

from . import ops as sops
from .kv import BlockPool, SeqStatus, Sequence
from .model import CacheView, Transformer


# A shared prefix of fewer tokens is left to paged_decode (of twice as many where a KV head's queries are little work).  Measured on
# 2 to 128 sequences with 16 or 64 tokens of their own, shared form against paged_decode, us.  64/8 heads of 64: 4 sequences, 64
# shared tokens 12.6 against 10.0, 96 ones 12.7 and 12.3, 128 ones 13.3 and 14.4; 128 sequences, 128 shared ones 17.9 against 95.
# Little work: 8/2 heads of 64, 8 sequences, 128 tokens 13.4 against 10.0, 192 ones 14.1 and 12.7, 256 ones 14.4 and 15.8;
# 16/16 heads of 64, 32 sequences, 192 tokens 14.1 against 12.4, 256 ones 14.4 and 14.8.
MIN_SHARED_TOKENS = 128
LITTLE_WORK = 448       # query heads of a KV head times head size


class LookupDraft:
  """Proposes the continuation of the last earlier place where a sequence had its current last 3 (else 2) tokens."""

  def __init__(self):
    self.known = 0                                  # tokens of the last call
    self.seen: Dict[tuple, int] = {}                # n-gram -> index of the token behind its last occurrence

  def propose(self, tokens: List[int], k: int) -> List[int]:
    """``tokens``: the sequence so far; successive calls only append to it."""
    for end in range(max(2, self.known), len(tokens)):       # n-grams that end before tokens[end]
      for n in (2, 3):
        if end >= n:
          self.seen[tuple(tokens[end - n:end])] = end
    self.known = len(tokens)
    for n in (3, 2):
      at = self.seen.get(tuple(tokens[-n:])) if len(tokens) >= n else None
      if at is not None:
        return tokens[at:at + k]
    return []


class Engine:
  def __init__(self, model: Transformer, *, max_seq_len: int = 512, max_batch: int = 32, block_size: int = 16,
               num_blocks: Optional[int] = None, max_prefill_tokens: int = 16384):
    self.model = model
    cfg = model.cfg
    self.device = model.embed.device
    self.max_seq_len, self.max_batch, self.block_size = max_seq_len, max_batch, block_size
    self.max_prefill_tokens = max_prefill_tokens
    per_seq = (max_seq_len + block_size - 1) // block_size
    self.num_blocks = num_blocks or max_batch * per_seq
    shape = (cfg.num_hidden_layers, self.num_blocks, block_size, cfg.num_key_value_heads, cfg.head_dim)
    self.k_cache = torch.zeros(shape, dtype=model.embed.dtype, device=self.device)
    self.v_cache = torch.zeros(shape, dtype=model.embed.dtype, device=self.device)
    self.pool = BlockPool(self.num_blocks, block_size)
    self.waiting: Deque[Sequence] = deque()
    self.running: List[Sequence] = []
    self.finished: Dict[int, Sequence] = {}
    self.drafts: Dict[int, LookupDraft] = {}
    self.steps = {"prefill": 0, "decode": 0, "prefill_tokens": 0, "cached_tokens": 0, "preempted": 0, "drafted": 0, "accepted": 0}

  # ------------------------------------------------------------------ requests
  def add(self, tokens: Seq[int], max_new_tokens: Optional[int] = None) -> int:
    if len(tokens) == 0 or len(tokens) >= self.max_seq_len:
      raise ValueError(f"prompt length {len(tokens)} outside (0, {self.max_seq_len})")
    seq = Sequence(list(tokens), max_new_tokens or (self.max_seq_len - len(tokens)))
    self.waiting.append(seq)
    return seq.seq_id

  @property
  def idle(self) -> bool:
    return not self.waiting and not self.running

  # ------------------------------------------------------------------ scheduling
  def _admit(self) -> List[Sequence]:
    batch: List[Sequence] = []
    budget = self.max_prefill_tokens
    while self.waiting and len(self.running) + len(batch) < self.max_batch:
      seq = self.waiting[0]
      if not self.pool.can_allocate(seq) or (batch and len(seq) > budget):
        break
      self.waiting.popleft()
      self.pool.allocate(seq)
      seq.status = SeqStatus.RUNNING
      budget -= len(seq) - seq.n_cached
      batch.append(seq)
    return batch

  def _preempt_for_space(self) -> None:
    """Decode needs a fresh block for some sequence and none is free: push the youngest running
    sequences back to the queue (their blocks are released; they prefill again later)."""
    def need() -> int:
      return sum(1 for s in self.running if (len(s) - 1) // self.block_size >= len(s.block_table))
    while len(self.running) > 1 and need() > self.pool.n_free:
      victim = self.running.pop()
      self.pool.release(victim)
      victim.status = SeqStatus.WAITING
      self.waiting.appendleft(victim)
      self.steps["preempted"] += 1

  # ------------------------------------------------------------------ one step
  @torch.inference_mode()
  def step(self, **model_kw) -> Optional[Tuple[torch.Tensor, List[int]]]:
    """Returns (next-token logits [n, vocab] fp32, sequence ids) or None when idle."""
    batch = self._admit()
    if batch:
      self.running.extend(batch)
      return self._prefill(batch, **model_kw), [s.seq_id for s in batch]
    if not self.running:
      return None
    self._preempt_for_space()
    if not self.running:
      return None
    return self._decode(self.running), [s.seq_id for s in self.running]

  def _prefill(self, seqs: List[Sequence], **model_kw) -> torch.Tensor:
    bs = self.block_size
    new = [len(s) - s.n_cached for s in seqs]
    S = max(new)
    B = len(seqs)
    ids = torch.zeros(B, S, dtype=torch.long)
    pos = torch.zeros(B, S, dtype=torch.long)
    slots = torch.full((B, S), -1, dtype=torch.int32)
    max_blocks = max(len(s.block_table) for s in seqs)
    tables = torch.zeros(B, max_blocks, dtype=torch.int32)
    for i, s in enumerate(seqs):
      n, c = new[i], s.n_cached
      ids[i, :n] = torch.tensor(s.tokens[c:], dtype=torch.long)
      p = torch.arange(c, c + n)
      pos[i, :n] = p
      bt = torch.tensor(s.block_table, dtype=torch.long)
      tables[i, :len(s.block_table)] = bt.int()
      slots[i, :n] = (bt[p // bs] * bs + p % bs).int()
    dev = self.device
    cache = CacheView(self.k_cache, self.v_cache, slots.to(dev), block_tables=tables.to(dev),
                      prefix_lens=[s.n_cached for s in seqs], block_size=bs)
    out = self.model(ids.to(dev), pos.to(dev), cache=cache, is_prefill=True, **model_kw)
    for s in seqs:
      self.pool.mark_ready(s)
    self.steps["prefill"] += 1
    self.steps["prefill_tokens"] += sum(new)
    self.steps["cached_tokens"] += sum(s.n_cached for s in seqs)
    if isinstance(out, tuple) or out is None:
      return out
    last = torch.tensor([n - 1 for n in new], device=dev)
    return out[torch.arange(B, device=dev), last]

  def _decode(self, seqs: List[Sequence]) -> torch.Tensor:
    dev = self.device
    slots = torch.tensor([self.pool.append_slot(s) for s in seqs], dtype=torch.int32)
    ids = torch.tensor([s.tokens[-1] for s in seqs], dtype=torch.long)
    pos = torch.tensor([len(s) - 1 for s in seqs], dtype=torch.long)
    ctx = torch.tensor([len(s) for s in seqs], dtype=torch.int32)
    tables = self._tables(seqs)
    cache = CacheView(self.k_cache, self.v_cache, slots.to(dev), block_tables=torch.from_numpy(tables).to(dev), context_lens=ctx.to(dev),
                      block_size=self.block_size, shared_len=self._shared_len(tables, int(ctx.min())))
    self.steps["decode"] += 1
    return self.model(ids.to(dev), pos.to(dev), cache=cache, is_prefill=False)

  @staticmethod
  def _tables(seqs: List[Sequence]) -> np.ndarray:
    tables = np.zeros((len(seqs), max(len(s.block_table) for s in seqs)), dtype=np.int32)
    for i, s in enumerate(seqs):
      tables[i, :len(s.block_table)] = s.block_table
    return tables

  def _shared_len(self, tables: np.ndarray, shortest: int) -> int:
    """Leading tokens whose blocks are the same in every table, where that is enough to be worth a pass of its own."""
    if len(tables) < 2:
      return 0
    n_blocks = min(tables.shape[1], (shortest - 1) // self.block_size)        # the block being written is nobody else's
    same = (tables[:, :n_blocks] == tables[:1, :n_blocks]).all(0)
    n = (n_blocks if same.all() else int(same.argmin())) * self.block_size
    cfg = self.model.cfg
    little = cfg.num_attention_heads // cfg.num_key_value_heads * cfg.head_dim < LITTLE_WORK
    return n if n >= MIN_SHARED_TOKENS * (2 if little else 1) else 0

  # ------------------------------------------------------------------ several tokens per step
  def _decode_drafts(self, seqs: List[Sequence], k: int) -> Tuple[torch.Tensor, torch.Tensor, CacheView, List[int]]:
    """One pass over the last token of every sequence and up to ``k`` looked-up ones behind it: (logits [N, vocab], the packed
    input tokens [N], the step's cache view, rows per sequence).  A sequence gets fewer where its budget, its context or the
    free blocks end; where nobody has any the step is a plain decode step, behind a shared prefix if there is one."""
    dev, bs = self.device, self.block_size
    for s in seqs:
      self.pool.append_slot(s)                        # the step itself comes before anybody's drafts
    ids, pos, slots, lens = [], [], [], []
    for s in seqs:
      room = min(k, s.max_new_tokens - s.n_generated - 1, self.max_seq_len - len(s) - 1)
      draft = self.drafts.setdefault(s.seq_id, LookupDraft()).propose(s.tokens, room) if room > 0 else []
      if draft:
        draft = draft[:self.pool.reserve(s, len(draft))]
      first = len(s) - 1
      ids += [s.tokens[-1]] + draft
      pos += range(first, first + 1 + len(draft))
      slots += [self.pool.slot(s, p) for p in range(first, first + 1 + len(draft))]
      lens.append(1 + len(draft))
      self.steps["drafted"] += len(draft)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).to(dev)
    tokens = torch.tensor(ids, dtype=torch.long).to(dev)
    ctx, tables = [len(s) - 1 + n for s, n in zip(seqs, lens)], self._tables(seqs)
    if max(lens) == 1:
      rows = dict(shared_len=self._shared_len(tables, min(ctx)))
    else:
      rows = dict(q_starts=i32(self._starts(lens)), q_lens=i32(lens), max_q_len=max(lens))
    cache = CacheView(self.k_cache, self.v_cache, i32(slots), block_tables=torch.from_numpy(tables).to(dev), context_lens=i32(ctx),
                      block_size=bs, **rows)
    self.steps["decode"] += 1
    return self.model(tokens, torch.tensor(pos, dtype=torch.long).to(dev), cache=cache, is_prefill=False), tokens, cache, lens

  @staticmethod
  def _starts(lens: List[int]) -> List[int]:
    """First row of each sequence where their rows follow one another."""
    return [0] + list(itertools.accumulate(lens[:-1]))

  @torch.inference_mode()
  def step_drafts(self, k: int, *, temperature: float = 0.0, top_k: int = 0, generator: Optional[torch.Generator] = None
                  ) -> Optional[List[Tuple[int, List[int]]]]:
    """``step`` with up to ``k`` looked-up tokens per running sequence, sampling included: (sequence id, emitted tokens) of
    every sequence that moved, at least one token each.  The caller hands them to ``update`` one by one."""
    batch = self._admit()
    if batch:
      self.running.extend(batch)
      logits = self._prefill(batch)
      nxt = self._probs(logits, temperature, top_k)
      nxt = logits.argmax(-1) if nxt is None else torch.multinomial(nxt, 1, generator=generator).squeeze(-1)
      return [(s.seq_id, [t]) for s, t in zip(batch, nxt.tolist())]
    if not self.running:
      return None
    self._preempt_for_space()
    seqs = list(self.running)
    logits, tokens, cache, lens = self._decode_drafts(seqs, k)
    probs = self._probs(logits, temperature, top_k)
    out, row = [], 0
    if probs is None:                                 # greedy: a drafted token passes where it is the likeliest one
      nxt, ids = logits.argmax(-1).tolist(), tokens.tolist()
      for s, n in zip(seqs, lens):
        j = 1
        while j < n and ids[row + j] == nxt[row + j - 1]:
          j += 1
        out.append((s.seq_id, nxt[row:row + j]))
        row += n
    else:
      u = torch.rand(tokens.numel(), device=generator.device if generator is not None else self.device, generator=generator).to(self.device)
      rows = cache.q_starts, cache.q_lens
      if cache.q_lens is None:                        # no drafts: one token each, drawn from its row
        rows = (torch.tensor(x, dtype=torch.int32).to(self.device) for x in (self._starts(lens), lens))
      emitted, count = sops.verify_draft(probs, tokens, u, *rows, out=torch.empty_like(tokens, dtype=torch.int32))
      emitted = emitted.tolist()
      for s, n, j in zip(seqs, lens, count.tolist()):
        out.append((s.seq_id, emitted[row:row + j]))
        row += n
    self.steps["accepted"] += sum(len(t) - 1 for _, t in out)
    return out

  @staticmethod
  def _probs(logits: torch.Tensor, temperature: float, top_k: int) -> Optional[torch.Tensor]:
    """Sampling probabilities, None for greedy."""
    if temperature <= 0:
      return None
    lg = logits / temperature
    if top_k > 0:
      kth = lg.topk(min(top_k, lg.size(-1)), dim=-1).values[:, -1:]
      lg = lg.masked_fill(lg < kth, float("-inf"))
    return torch.softmax(lg, -1)

  def update(self, seq_id: int, token: int, finished: bool = False) -> None:
    for i, s in enumerate(self.running):
      if s.seq_id == seq_id:
        if not finished:
          s.tokens.append(int(token))
        if finished or s.n_generated >= s.max_new_tokens or len(s) >= self.max_seq_len:
          s.status = SeqStatus.FINISHED
          self.pool.release(s)
          self.running.pop(i)
          self.finished[s.seq_id] = s
          self.drafts.pop(s.seq_id, None)
        return
    raise KeyError(f"sequence {seq_id} is not running")

  # ------------------------------------------------------------------ conveniences
  def generate(self, prompts: Iterable[Seq[int]], *, max_new_tokens: int = 64, stop_tokens: Iterable[int] = (),
               temperature: float = 0.0, top_k: int = 0, generator: Optional[torch.Generator] = None,
               on_token: Optional[Callable[[int, int], None]] = None, draft_tokens: int = 0) -> List[List[int]]:
    """Greedy (temperature 0) or top-k sampled completions, in the order of ``prompts``.  ``draft_tokens``: tokens that every
    sequence may look up in its own text and have scored in one step (see the module's first lines)."""
    if draft_tokens < 0:
      raise ValueError("draft_tokens must not be negative")
    stop = set(int(t) for t in stop_tokens)
    order = [self.add(p, max_new_tokens) for p in prompts]
    while not self.idle:
      if draft_tokens > 0:
        moved = self.step_drafts(draft_tokens, temperature=temperature, top_k=top_k, generator=generator)
        if moved is None:
          break
      else:
        res = self.step()
        if res is None:
          break
        logits, ids = res
        probs = self._probs(logits, temperature, top_k)
        nxt = logits.argmax(-1) if probs is None else torch.multinomial(probs, 1, generator=generator).squeeze(-1)
        moved = [(sid, [tok]) for sid, tok in zip(ids, nxt.tolist())]
      for sid, toks in moved:
        for tok in toks:
          if on_token is not None:
            on_token(sid, tok)
          self.update(sid, tok, finished=tok in stop)
          if sid in self.finished:                    # what was drafted behind the end is dropped
            break
    return [self.finished[sid].tokens[self.finished[sid].prompt_len:] for sid in order]

  @torch.inference_mode()
  def hidden_states(self, prompts: List[Seq[int]], up_to_layer: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """Hidden states after ``up_to_layer`` blocks for a batch of prompts, without touching the cache:
    (hidden [B,S,H], mask [B,S])."""
    S = max(len(p) for p in prompts)
    ids = torch.zeros(len(prompts), S, dtype=torch.long)
    mask = torch.zeros(len(prompts), S, dtype=torch.bool)
    for i, p in enumerate(prompts):
      ids[i, :len(p)] = torch.tensor(list(p), dtype=torch.long)
      mask[i, :len(p)] = True
    pos = torch.arange(S).expand(len(prompts), S)
    _, taps = self.model(ids.to(self.device), pos.to(self.device), is_prefill=True, up_to_layer=up_to_layer,
                         return_hidden_states=True, no_logits=True)
    return taps[up_to_layer], mask.to(self.device)
