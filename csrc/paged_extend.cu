// Attention of several new tokens per sequence over the paged cache, on tcgen05: drafted tokens of a decode step, the
// part of a prompt behind a cached prefix, and a whole batch of single tokens over the keys of a prefix they share.
//   out = sum_j softmax_j(scale * q . k_j | sink) * v_j       over the keys j that a token sees
//
// Rows.  The g query heads of a key/value head and the tokens that read the same keys are stacked: row = token * g +
// head of the group, 128 rows to a tile, so every K/V block is read once for all of them.  Each row carries its own
// bounds [lo, hi) of visible keys (causal end, window, shared part); a block that lies inside all of them needs no mask.
//
// Many rows (k_paged_extend), a tile a CTA, 64 keys at a time.  A loader warp (D = 128: one for K, one for V) brings a block's
// rows from their pages, by TMA where whole boxes of keys lie in a page, else with cp.async (16 bytes a lane, any page
// size; 8 prompts: 597 us by TMA where 982 by hand); both leave zeros where the CTA has no keys, so that what lies there cannot
// reach the products.  One thread issues the MMAs, four warps own 32 rows each: running maximum and sum in fp32, P as bf16 back
// to tensor memory as the A operand of P V.  The maximum is raised only when it grows by more than 2^8; the stale one is exact
// after the final division.  The sum l takes the unrounded p.
//
// Roundings of P.  The tensor core multiplies it with bf16 values, so it has to be bf16 too.  Steps of a few tokens (the kernel for
// few rows, lists of one tile or one token, a shared prefix) take it in two parts, its bf16 value and the bf16 value of what that leaves, at
// twice the products of P V: what comes out is rounded once, as paged_decode's results are (which has P in fp32), whichever kernel a
// sequence's step happens to run on.  Error of the result relative to its norm 1.7e-3, with one part 2.4e-3.  Prompts of several
// tiles take one part, as the dense attention of a prompt without a cached prefix does (8 prompts: 597 us, in two parts 795).
//
// A block is a chain of latencies (S, softmax, P V and the way to the next S) in which no unit is busy, so an SM is filled with
// chains: four CTAs for D = 64, whose S has a single buffer to fit tensor memory, two for D = 128.  Code that is run once or
// seldom stays rolled: with the softmax of 64 keys in one piece, 55 % of the instruction cache's request rate was the bound and
// the fourth CTA gained nothing (699 us; loops over 32 keys: 625; loaders and start of a CTA rolled too: 597; three CTAs: 700).
// 8 prompts of 200..1750 new tokens behind 1300..3500 cached ones, 64/8 heads of 64: 597 us, 670 TFLOP/s (over a long run, at
// lower clocks, 632 us; issue slots 55 %, special function unit 64 %, tensor cores 32 %).  What did not help: part of the
// exponentials by polynomial, two warps for 32 rows, two tiles a CTA, 16 keys at a time (631 us), keeping half of the scores
// between maximum and exponentials (679 us).
//
// Few rows (k_paged_few, below): decode steps and drafts, bound by the bytes of K and V.
//
// Few CTAs: the keys are split over the CTAs of a cluster, whose (m, l, O) meet in distributed shared memory: no workspace,
// no atomics, one launch; beyond eight splits over several clusters and a launch that joins their sets.  Shared prefix: one
// launch for the prefix (rows of all sequences, sets to a workspace), a dependent launch for each sequence's own keys that
// starts while the first one drains and joins its rows at the end.  All of it gives the same bits on every run.
#include <cooperative_groups.h>
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "common/ptx.cuh"
#include "common/tensormap.h"

namespace cg = cooperative_groups;

namespace nmoe {

constexpr int PX_BM = 128;            // rows per tile
constexpr int PX_BN = 64;             // keys per block
constexpr uint64_t kPxWaitNs = 2000000000ull;
constexpr float kPxRescale = 8.f;     // log2 units

struct ExtendParams {
  const __nv_bfloat16 *q, *k_cache, *v_cache;
  __nv_bfloat16* out;
  const int *block_tables, *context_lens, *q_starts, *q_lens;    // q_starts / q_lens null: one token per sequence
  const void* sinks;
  // partial results of another launch: row (token * hq + head): O (unnormalised) and (m, l), m in log2 units
  float *part_o, *part_ml;
  StatusRecord* status;
  long long q_stride, bt_stride;
  int n_rows, n_seqs, hq, hkv, group, block_size, block_shift, num_blocks, capacity, max_q_len, window, sinks_fp32;
  int key_begin, key_end;             // only keys in [key_begin, key_end) count here
  int flat;                           // 1: the tokens of all sequences are one list that reads the pages of one of them
  int splits, groups;                 // the keys of a row list are divided over groups x splits CTAs, splits = a cluster
  int sorted;                         // 1: lists by falling context
  int part_mode;                      // 0 none, 1 write partial results (one set per group), 2 join those of the launch before
  int n_sets;                         // sets of partial results to join
  int tma_rows;                       // keys of a TMA box, 0: the page size does not allow it
  long long set_rows;                 // rows of a set
  float scale_log2;
};

NMOE_DEVICE uint64_t px_timer() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
NMOE_DEVICE bool px_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = px_timer();
  uint32_t it = 0;
  while (!mbar_try_wait(bar, parity)) {
    if ((++it & 255u) == 0) {
      if (*abort_flag) return false;
      if (px_timer() - t0 > kPxWaitNs) return false;
    }
  }
  return true;
}
NMOE_DEVICE bool px_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
NMOE_DEVICE void px_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
NMOE_DEVICE void px_tmem_st_x16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
NMOE_DEVICE float px_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// three-input maximum and two fp32 operations per instruction (sm_100)
NMOE_DEVICE float px_max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
NMOE_DEVICE uint64_t px_pack(float a, float b) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
NMOE_DEVICE void px_unpack(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
NMOE_DEVICE uint64_t px_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
NMOE_DEVICE uint64_t px_add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// two probabilities as bf16 values and, in a second pair, what these leave of them: together they hold 2^-16 of each
NMOE_DEVICE void px_split(float a, float b, uint32_t& high, uint32_t& rest) {
  high = pack_bf16x2(a, b);
  const float2 h = unpack_bf16x2(high);
  rest = pack_bf16x2(a - h.x, b - h.y);
}
NMOE_DEVICE void px_cp16(uint32_t dst, const void* src, uint32_t bytes) {      // bytes 0: the 16 bytes become zero
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
NMOE_DEVICE void px_cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
NMOE_DEVICE void px_cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
NMOE_DEVICE void px_launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
NMOE_DEVICE void px_wait_prior_grid() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// x / g for x below g + 128 and 2^22, from 1 / g: (x + 1/2) / g is at least 1 / (2 g) from a whole number
NMOE_DEVICE int px_div(int x, float inv_g) { return static_cast<int>((static_cast<float>(x) + 0.5f) * inv_g); }

// floor(n * i / of) for i <= of: where the share of unit i starts (a 64-bit division only where 32 bits do not hold it)
NMOE_DEVICE int px_share(int n, int i, int of) {
  if (of == 1) return i == 0 ? 0 : n;
  if (n < 0x7fffffff / (of + 1)) return static_cast<int>(static_cast<unsigned>(n * i) / static_cast<unsigned>(of));
  return static_cast<int>(static_cast<long long>(n) * i / of);
}

// Rows of one list: its first row, its number of tokens (0 where the lengths are out of range) and its context.
NMOE_DEVICE void px_list(const ExtendParams& p, int b, bool speaker, int& start, int& n, int& ctx) {
  start = 0;
  n = p.n_seqs;
  ctx = 0;
  if (p.flat) return;
  start = p.q_starts != nullptr ? p.q_starts[b] : b;
  n = p.q_lens != nullptr ? p.q_lens[b] : 1;
  ctx = p.context_lens[b];
  if (start < 0 || n < 0 || start > p.n_rows || n > p.n_rows - start || n > p.max_q_len) {
    if (speaker) report_status(p.status, kStatusBadIndex, 1020, b, start);
    n = 0;
  } else if (ctx > p.capacity) {
    if (speaker) report_status(p.status, kStatusBadIndex, 1021, b, ctx);
    ctx = p.capacity;
  }
  ctx = max(ctx, 0);                                             // a negative length is none: positions must not wrap below
}
// The list of blocks with index z: the z-th longest context where one wave of CTAs does not hold them all, so that the long
// ones start first and the short ones fill the end (64 drafted steps: 102 -> 74 us).  Every CTA ranks the contexts for itself,
// as numbers that also hold the index, so that no two are the same and one comparison does (contexts from 2^23 on count alike).
constexpr int PX_SORT_MOST = 256;
template <int kThreads>
NMOE_DEVICE int px_nth_longest(const ExtendParams& p, int z, int* s_key) {         // s_key: PX_SORT_MOST + 1 words of scratch
  constexpr int kEach = (PX_SORT_MOST + kThreads - 1) / kThreads;
  const int n4 = (p.n_seqs + 3) / 4;
  int key[kEach];
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int t = threadIdx.x + k * kThreads;
    const bool in = t < p.n_seqs;
    const int len = in && !(p.q_lens != nullptr && p.q_lens[t] <= 0) ? min(max(p.context_lens[t], 0), 0x7fffff) : 0;
    key[k] = in ? len * PX_SORT_MOST + (PX_SORT_MOST - 1 - t) : -1;
    if (t < 4 * n4) s_key[t] = key[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int t = threadIdx.x + k * kThreads;
    if (t >= p.n_seqs) break;
    int rank = 0;
    for (int u = 0; u < n4; ++u) {
      const int4 v = reinterpret_cast<const int4*>(s_key)[u];
      rank += (v.x > key[k]) + (v.y > key[k]) + (v.z > key[k]) + (v.w > key[k]);
    }
    if (rank == z) s_key[PX_SORT_MOST] = t;
  }
  __syncthreads();
  const int which = s_key[PX_SORT_MOST];
  __syncthreads();                                               // the scratch may be used for something else
  return which;
}
// Whose pages hold the keys of a list that all sequences share: the first sequence that reaches its end (a padding row does
// not), else the longest.  By a whole warp.
NMOE_DEVICE int px_owner(const ExtendParams& p, int lane) {
  int best = 0, most = -1;
  for (int t0 = 0; t0 < p.n_seqs; t0 += 32) {
    const int t = t0 + lane, c = t < p.n_seqs ? p.context_lens[t] : -1;
    const unsigned all = __ballot_sync(0xffffffffu, t < p.n_seqs && c >= p.key_end);
    if (all != 0) return t0 + __ffs(all) - 1;
    if (c > most) { most = c; best = t; }
  }
  const int top = __reduce_max_sync(0xffffffffu, most);
  return __reduce_min_sync(0xffffffffu, most == top ? best : 0x7fffffff);
}
// Keys [lo, hi) that a token of the list sees.
NMOE_DEVICE void px_bounds(const ExtendParams& p, int tok, int n, int ctx, bool speaker, int& lo, int& hi) {
  int pos = ctx - n + tok;
  if (p.flat) {
    const int c = p.context_lens[tok];
    if (c > p.capacity && speaker) report_status(p.status, kStatusBadIndex, 1021, tok, c);
    pos = min(max(c, 0), p.capacity) - 1;
  }
  lo = max(p.window > 0 ? max(0, max(pos, 0) - p.window + 1) : 0, p.key_begin);    // before position 0: stays within 32 bits
  hi = min(pos + 1, p.key_end);
}
NMOE_DEVICE float px_sink(const ExtendParams& p, int h) {         // log2 units
  if (p.sinks == nullptr) return -INFINITY;
  return 1.4426950408889634f * (p.sinks_fp32 ? static_cast<const float*>(p.sinks)[h]
                                             : __bfloat162float(static_cast<const __nv_bfloat16*>(p.sinks)[h]));
}

NMOE_DEVICE void px_store(__nv_bfloat16* dst, float4 a, float f) {
  *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(a.x * f, a.y * f), pack_bf16x2(a.z * f, a.w * f));
}
// what scales a sum relative to `top` to the result: 1 / (sum + sink's part); no key: zeros; a NaN in q stays one
NMOE_DEVICE float px_factor(float top, float sum, float sink) {
  const float high = fmaxf(top, sink), e = px_exp2(top - high);
  return sum != 0.f ? e / (sum * e + px_exp2(sink - high)) : 0.f;
}
NMOE_DEVICE void px_axpy(float4& y, float w, float4 x) { y.x += w * x.x; y.y += w * x.y; y.z += w * x.z; y.w += w * x.w; }
// Sum of (m, l, O) pieces relative to a common maximum, 4 columns a thread.
struct PxSum {
  float top, sum;
  float4 acc;
  NMOE_DEVICE void start(float t) {
    top = t;
    sum = 0.f;
    acc = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  NMOE_DEVICE void add(float2 ml, float4 a) {
    const float w = px_exp2(ml.x - top);
    sum += w * ml.y;
    px_axpy(acc, w, a);
  }
  // the sets first, first + step, ... of a row, kAtOnce of them on their way; rows without keys hold zeros
  template <int D, int kAtOnce>
  NMOE_DEVICE void add_sets(const ExtendParams& p, long long row, int c, int first, int step) {
    for (int s0 = first; s0 < p.n_sets; s0 += kAtOnce * step) {
      float2 ml[kAtOnce];
      float4 x[kAtOnce];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const int s = s0 + u * step;
        ml[u] = make_float2(0.f, 0.f);
        if (s < p.n_sets) {
          ml[u] = __ldcg(reinterpret_cast<const float2*>(p.part_ml) + s * p.set_rows + row);
          x[u] = __ldcg(reinterpret_cast<const float4*>(p.part_o + (s * p.set_rows + row) * D) + c);
        }
      }
      float high = top;
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u)
        if (ml[u].y != 0.f) high = fmaxf(high, ml[u].x);
      const float w = px_exp2(top - high);
      top = high;
      sum *= w;
      acc.x *= w; acc.y *= w; acc.z *= w; acc.w *= w;
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u)
        if (ml[u].y != 0.f) add(ml[u], x[u]);
    }
  }
  NMOE_DEVICE void store(__nv_bfloat16* dst, float sink) const { px_store(dst, acc, px_factor(top, sum, sink)); }
};

// Joins what the kS CTAs of a cluster hold for the rows row0 .. row0 + n_valid (sx [rows][D] fp32 in 16-byte pieces swizzled
// by row, s_ml [rows][2]) and, in part_mode 2, the sets of the launch before.  Every CTA takes a run of the rows: a thread a
// row works out what each part counts for (s_w, [rows][kS + 3]), then all threads sum the columns, with the loads of several
// sums in flight, since a remote read takes some hundred cycles (doing both per column took 7 us where this takes 3).
template <int D, int kThreads, int kS>
NMOE_DEVICE void px_join_of(const ExtendParams& p, const float* sx, const float* s_ml, float* s_w, int start, int row0, int n_valid, int hk, int unit) {
  cg::cluster_group cl = cg::this_cluster();
  constexpr int kW = kS + 3;                                     // weights, maximum, sum, row of the result
  const int rank = unit % kS, group = unit / kS, g = p.group;
  if (kS > 1) cl.sync();
  else __syncthreads();
  const int per = (n_valid + kS - 1) / kS;
  const int ra = rank * per, n_mine = max(min(n_valid, ra + per) - ra, 0);
  auto of = [&](const float* at, int s) -> const float* { return kS > 1 ? cl.map_shared_rank(const_cast<float*>(at), s) : at; };
  for (int i = threadIdx.x; i < n_mine; i += kThreads) {
    const int r = ra + i, rr = row0 + r, tok = rr / g, h = hk * g + rr - tok * g;
    const long long row = static_cast<long long>(start + tok) * p.hq + h;
    float2 ml[kS];
#pragma unroll
    for (int s = 0; s < kS; ++s) ml[s] = *reinterpret_cast<const float2*>(of(s_ml + 2 * r, s));
    float top = -1e30f, sum = 0.f, w[kS], f = 1.f;
#pragma unroll
    for (int s = 0; s < kS; ++s)
      if (ml[s].y != 0.f) top = fmaxf(top, ml[s].x);
#pragma unroll
    for (int s = 0; s < kS; ++s) {
      w[s] = ml[s].y != 0.f ? px_exp2(ml[s].x - top) : 0.f;
      sum += w[s] * ml[s].y;
    }
    if (p.part_mode == 0) f = px_factor(top, sum, px_sink(p, h));
    else if (p.part_mode == 1) reinterpret_cast<float2*>(p.part_ml)[group * p.set_rows + row] = make_float2(top, sum);
#pragma unroll
    for (int s = 0; s < kS; ++s) s_w[i * kW + s] = w[s] * f;
    s_w[i * kW + kS] = top;
    s_w[i * kW + kS + 1] = sum;
    s_w[i * kW + kS + 2] = __int_as_float(static_cast<int>(row));
  }
  if (p.part_mode == 2) px_wait_prior_grid();
  __syncthreads();
  constexpr int kCols = D / 4, kItems = kS <= 2 ? 4 : kS == 4 ? 2 : 1;             // up to eight pieces of 16 bytes on their way
  const int n_items = n_mine * kCols;
  for (int i0 = threadIdx.x; i0 < n_items; i0 += kThreads * kItems) {
    float4 x[kItems][kS];
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      const int i = min(i0 + k * kThreads, n_items - 1), r = ra + i / kCols, c = i % kCols;
#pragma unroll
      for (int s = 0; s < kS; ++s) x[k][s] = reinterpret_cast<const float4*>(of(sx + r * D, s))[c ^ (r & 7)];
    }
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      const int i = i0 + k * kThreads, c = i % kCols;
      if (i >= n_items) break;
      const float* w = s_w + i / kCols * kW;
      const long long row = __float_as_int(w[kS + 2]);
      PxSum t;
      t.start(w[kS]);
      t.sum = w[kS + 1];
#pragma unroll
      for (int s = 0; s < kS; ++s) px_axpy(t.acc, w[s], x[k][s]);
      if (p.part_mode == 0) {
        px_store(p.out + row * D + c * 4, t.acc, 1.f);
      } else if (p.part_mode == 1) {
        reinterpret_cast<float4*>(p.part_o + (group * p.set_rows + row) * D)[c] = t.acc;
      } else {
        t.add_sets<D, 4>(p, row, c, 0, 1);
        t.store(p.out + row * D + c * 4, px_sink(p, static_cast<int>(row % p.hq)));
      }
    }
  }
  if (kS > 1) cl.sync();                                         // nobody leaves while its rows may still be read
}
template <int D, int kThreads>
NMOE_DEVICE void px_join(const ExtendParams& p, const float* sx, const float* s_ml, float* s_w, int start, int row0, int n_valid, int hk, int unit) {
  switch (p.splits) {
    case 1: px_join_of<D, kThreads, 1>(p, sx, s_ml, s_w, start, row0, n_valid, hk, unit); break;
    case 2: px_join_of<D, kThreads, 2>(p, sx, s_ml, s_w, start, row0, n_valid, hk, unit); break;
    case 4: px_join_of<D, kThreads, 4>(p, sx, s_ml, s_w, start, row0, n_valid, hk, unit); break;
    default: px_join_of<D, kThreads, 8>(p, sx, s_ml, s_w, start, row0, n_valid, hk, unit); break;
  }
}

// Layout of shared memory.  The exchange of partial results reuses the stages (O as fp32, 16-byte pieces swizzled by row).
template <int D>
struct PxSmem {
  static constexpr int kCtas = D == 64 ? 4 : 2;            // of an SM: all of tensor memory, 128 and 256 columns each
  static constexpr int kBufs = D == 64 ? 1 : 2;            // S buffers of 64 columns
  static constexpr int kLoaders = D == 64 ? 1 : 2;         // warps; with one more four CTAs have no registers
  static constexpr int kThreads = 4 * 32 + 32 + 32 * kLoaders;
  static constexpr int kStages = 2;                        // of K and of V
  static constexpr int kQ = PX_BM * D * 2;
  static constexpr int kKV = PX_BN * D * 2;                // a stage of one of them
  static constexpr int kRing = 2 * kStages * kKV;
  static constexpr int kExchange = PX_BM * (D + 2) * 4;
  static constexpr int kBody = kRing > kExchange ? kRing : kExchange;
  static constexpr int kBytes = kQ + kBody + 256 + 1024;
  static constexpr uint32_t kTmemCols = kBufs * PX_BN + D;
};

template <int D, bool kDirect, bool kFine>
__global__ void __launch_bounds__(PxSmem<D>::kThreads, PxSmem<D>::kCtas)
k_paged_extend(const ExtendParams p, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v) {
  using SM = PxSmem<D>;
  constexpr int kStages = SM::kStages, kBufs = SM::kBufs;
  constexpr int kLag = kStages - 1;          // see the loaders
  constexpr int kThreads = SM::kThreads;
  constexpr int kMmaWarp = 4;
  constexpr uint32_t kTmemO = kBufs * PX_BN;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sKV = sQ + SM::kQ;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sKV + SM::kBody);
  uint64_t* kv_full = bars;                  // [K, V][kStages]
  uint64_t* kv_empty = kv_full + 2 * kStages;
  uint64_t* s_full = kv_empty + 2 * kStages; // [kBufs]
  uint64_t* p_full = s_full + kBufs;         // [kBufs]
  uint64_t* pv_done = p_full + kBufs;
  uint64_t* o_full = pv_done + 1;
  uint64_t* q_full = o_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(q_full + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // the keys are divided over units = groups x splits CTAs, the splits of a group being a cluster
  const int units = p.splits * p.groups, unit = static_cast<int>(blockIdx.x) % units;
  const int n_tiles_x = static_cast<int>(gridDim.x) / units;
  // tiles with the longest contexts (the last ones of a prompt) first: better tail
  const int tile_x = n_tiles_x - 1 - static_cast<int>(blockIdx.x) / units;
  const int hk = blockIdx.y, b = p.flat ? 0 : p.sorted ? px_nth_longest<kThreads>(p, blockIdx.z, reinterpret_cast<int*>(sKV)) : blockIdx.z, g = p.group;

  int start, n, ctx;
  px_list(p, b, tile_x == 0 && unit == 0 && hk == 0 && threadIdx.x == 0, start, n, ctx);
  const int row0 = tile_x * PX_BM;                               // first row of this CTA's tile
  const float inv_g = 1.f / static_cast<float>(g);
  const int n_valid = min(PX_BM, n * g - row0);                  // rows that exist
  if (n_valid <= 0) {                                            // uniform over the cluster
    if (p.part_mode == 1) px_launch_dependents();
    if (p.part_mode == 2) px_wait_prior_grid();
    return;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2 * kStages; ++i) { mbar_init(&kv_full[i], 1); mbar_init(&kv_empty[i], 1); }
    for (int i = 0; i < kBufs; ++i) { mbar_init(&s_full[i], 1); mbar_init(&p_full[i], (n_valid + 31) / 32); }
    mbar_init(pv_done, 1);
    mbar_init(o_full, 1);
    mbar_init(q_full, 4);
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(tmem_slot, SM::kTmemCols);
    tmem_relinquish();
  }
  // keys that the tile sees, worked out by every warp for itself
  int k_begin = 0x7fffffff, k_end = 0;
  {
    const int tok_a = row0 / g, tok_b = (row0 + n_valid - 1) / g;
    if (p.flat) {
      for (int t = tok_a + lane; t <= tok_b; t += 32) {
        int from, to;
        px_bounds(p, t, n, ctx, false, from, to);
        if (from < to) { k_begin = min(k_begin, from); k_end = max(k_end, to); }
      }
      k_begin = __reduce_min_sync(0xffffffffu, k_begin);
      k_end = __reduce_max_sync(0xffffffffu, k_end);
    } else {                                                     // both bounds grow from token to token
      int skip;
      px_bounds(p, tok_a, n, ctx, false, k_begin, skip);
      px_bounds(p, tok_b, n, ctx, false, skip, k_end);
    }
  }
  // blocks start on a box of keys, so that all but the first and the last are whole boxes
  const int k_from = p.tma_rows > 0 && k_end > k_begin ? k_begin - k_begin % p.tma_rows : k_begin;
  const int n_blocks_all = k_end > k_begin ? (k_end - k_from + PX_BN - 1) / PX_BN : 0;
  const int blk0 = px_share(n_blocks_all, unit, units), n_blk = px_share(n_blocks_all, unit + 1, units) - blk0;
  const int key0 = n_blk > 0 ? k_from + blk0 * PX_BN : 0;        // first key of this CTA

  // What a loader looks up: a page and a place in it; they become a row only when the block's turn comes, so that nothing waits
  // for the page table meanwhile.  -1: zeros, -2: no such page.
  struct Spot { int page, in_page; };
  const int rows = p.tma_rows, n_box = rows > 0 ? PX_BN / rows : 0;
  const int* table = nullptr;
  Spot next[2];
  auto whole = [&](int i) -> bool {
    const int k0 = key0 + i * PX_BN;
    return rows > 0 && k0 >= k_begin && k0 + PX_BN <= k_end;
  };
  auto spot_of = [&](int key) -> Spot {
    if (key < k_begin || key >= k_end) return {-1, -1};
    const int pi = p.block_shift >= 0 ? key >> p.block_shift : key / p.block_size;
    return {__ldg(table + pi), key - pi * p.block_size};
  };
  auto look_up = [&](int i) {                                    // this lane's box, or its two keys, of block i
    next[0] = next[1] = {-1, -1};
    if (i >= n_blk) return;
    const int k0 = key0 + i * PX_BN;
    if (whole(i)) {
      if (lane < n_box) next[0] = spot_of(k0 + lane * rows);
    } else {
      next[0] = spot_of(k0 + lane);
      next[1] = spot_of(k0 + 32 + lane);
    }
  };
  if (warp > kMmaWarp) {
    table = p.block_tables + (p.flat ? px_owner(p, lane) : b) * p.bt_stride;
    look_up(0);
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  // every CTA holds its tensor memory before a dependent launch may ask for some
  if (p.part_mode == 1) px_launch_dependents();
  const uint32_t tmem_base = *tmem_slot;
  // Row r of the tile lies in lane r + 32 * turn of tensor memory (modulo 128), the turn differing between the CTAs of an
  // SM: the busy warps of tiles with few rows then sit on different schedulers.
  const int turn = static_cast<int>((tmem_base & 511u) / SM::kTmemCols) * (4 / SM::kBufs / 2 + 1) & 3;
  const int quad_row = (((warp & 3) - turn) & 3) * 32, my_row = quad_row + lane;         // softmax threads: row of the tile
  const bool softmax_warp = warp < kMmaWarp && quad_row < n_valid;
  int lo = 0, hi = 0;                                            // bounds of this thread's row
  if (warp < kMmaWarp) {
    // rows of Q, 128-byte swizzle, K-major; rows that do not exist are zero
    const int tok0 = row0 / g, rem0 = row0 - tok0 * g, c = threadIdx.x % (D / 8);
    const uint32_t dst = smem_u32(sQ) + (c >> 3) * (PX_BM * 128);
#pragma unroll 2
    for (int r = threadIdx.x / (D / 8); r < PX_BM; r += 128 / (D / 8)) {
      const bool in = r < n_valid;
      const int dt = in ? px_div(rem0 + r, inv_g) : 0, h = hk * g + (in ? rem0 + r - dt * g : 0);
      px_cp16(dst + ((r + 32 * turn) & 127) * 128 + (((c & 7) ^ (r & 7)) << 4),
              p.q + (start + tok0 + dt) * p.q_stride + static_cast<long long>(h) * D + c * 8, in ? 16u : 0u);
    }
    px_cp_commit();
    px_cp_wait<0>();
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(q_full);
    if (softmax_warp && my_row < n_valid)
      px_bounds(p, (row0 + my_row) / g, n, ctx, hk == 0 && unit == 0 && (row0 + my_row) % g == 0, lo, hi);
  }

  bool ok = true;
  float m = -1e30f, l = 0.f;
  if (warp > kMmaWarp) {
    // ------------------------------------------------------------ loaders
    // Where pages hold whole boxes of 4 to 64 keys, a block without keys outside [k_begin, k_end) comes by TMA, a box a
    // lane.  Other blocks are copied by hand: every lane looks up two of the 64 keys (a block ahead, so
    // that the page table's latency is covered) and the warp shares the rows by shuffle; such copies are announced in order
    // once they have landed, normally kLag blocks after they were asked for, all at once when the ring is full, since what
    // would make room may be waiting for one of them.
    constexpr int kChunks = D / 8, kRowsPass = 32 / kChunks;
    // K (0) and V (1) by a warp each, or both by one
    const int kv0 = SM::kLoaders == 2 ? warp - kMmaWarp - 1 : 0, kv1 = SM::kLoaders == 2 ? kv0 + 1 : 2;
    const int c = lane % kChunks, rp = lane / kChunks;
    const long long row_bytes = static_cast<long long>(p.hkv) * D * 2, piece = (static_cast<long long>(hk) * D + c * 8) * 2;
    auto row_of = [&](Spot s) -> int {
      return s.in_page < 0 ? -1 : s.page < 0 || s.page >= p.num_blocks ? -2 : s.page * p.block_size + s.in_page;
    };
    bool bad = false;
    int told = 0, st = 0;                                        // blocks announced so far; stage
    uint32_t ph = 1;
    auto announce = [&](int upto) {                              // this thread's copies of the blocks before upto have landed
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0)
        for (int t = told; t < upto; ++t)
          for (int kv = kv0; kv < kv1; ++kv) mbar_arrive(&kv_full[kv * kStages + t % kStages]);
      told = upto;
    };
    for (int i = 0; i < n_blk && ok; ++i) {
      int mine[2] = {row_of(next[0]), row_of(next[1])};
      bool boxes = whole(i);
      if (boxes && __any_sync(0xffffffffu, mine[0] == -2)) {     // a bad page among boxes: its keys become zeros
        boxes = false;
        mine[0] = row_of(spot_of(key0 + i * PX_BN + lane));
        mine[1] = row_of(spot_of(key0 + i * PX_BN + 32 + lane));
      }
      bad = bad || mine[0] == -2 || mine[1] == -2;
      look_up(i + 1);
      if (boxes && told < i) { px_cp_wait<0>(); announce(i); }
      for (int kv = kv0; kv < kv1; ++kv) {
        uint64_t *full = &kv_full[kv * kStages + st], *empty = &kv_empty[kv * kStages + st];
        if (!__all_sync(0xffffffffu, px_test(empty, ph))) {
          if (told < i) { px_cp_wait<0>(); announce(i); }
          ok = px_wait(empty, ph, abort_flag);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) { if (lane == 0) report_status(p.status, kStatusWaitTimeout, 1030, i, kv); *abort_flag = 1; break; }
        }
        uint8_t* slot = sKV + (kv * kStages + st) * SM::kKV;
        if (boxes) {
          const CUtensorMap* map = kv ? &tm_v : &tm_k;
          if (lane == 0) mbar_expect_tx(full, SM::kKV);
          __syncwarp();
          if (lane < n_box) {                                    // a box a lane
#pragma unroll
            for (int d = 0; d < D / 64; ++d) tma_load_2d(slot + d * (PX_BN * 128) + lane * rows * 128, map, full, hk * D + d * 64, mine[0]);
          }
          __syncwarp();
        } else {
          const uint8_t* src = reinterpret_cast<const uint8_t*>(kv ? p.v_cache : p.k_cache) + piece;
          const uint32_t dst = smem_u32(slot);
#pragma unroll 4
          for (int s = 0; s < PX_BN / kRowsPass; ++s) {
            const int r = s * kRowsPass + rp;
            const int row = __shfl_sync(0xffffffffu, mine[s >= PX_BN / kRowsPass / 2], r & 31);
            px_cp16(dst + (c >> 3) * (PX_BN * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4), src + max(row, 0) * row_bytes, row >= 0 ? 16u : 0u);
          }
        }
      }
      if (!ok) break;
      if (boxes) {
        told = i + 1;
      } else {
        px_cp_commit();
        if (i - kLag >= told) { px_cp_wait<kLag>(); announce(i - kLag + 1); }
      }
      if (++st == kStages) { st = 0; ph ^= 1; }
    }
    px_cp_wait<0>();
    if (ok && told < n_blk) announce(n_blk);
    if (bad) report_status(p.status, kStatusBadIndex, 1022, b, 0);
  } else if (warp == kMmaWarp) {
    // ------------------------------------------------------------ MMA issue
    if (elect_one()) {
      constexpr uint32_t idesc_s = make_idesc_bf16(PX_BM, PX_BN, 0, 0);
      constexpr uint32_t idesc_pv = make_idesc_bf16(PX_BM, D, 0, 1);
      const uint64_t qa = make_smem_desc(smem_u32(sQ), 0, 1024, kSwizzle128B);
      const uint64_t k_desc = make_smem_desc(smem_u32(sKV), 0, 1024, kSwizzle128B);
      const uint64_t v_desc = make_smem_desc(smem_u32(sKV + kStages * SM::kKV), PX_BN * 128, 1024, kSwizzle128B);
      int k_st = 0, v_st = 0;
      uint32_t k_ph = 0, v_ph = 0;
      auto wait_for = [&](uint64_t* bar, uint32_t ph, int site, int i) -> bool {
        if (px_wait(bar, ph, abort_flag)) return true;
        report_status(p.status, kStatusWaitTimeout, site, i, 0);
        *abort_flag = 1;
        return false;
      };
      auto issue_s = [&](int i) {                                // S = Q K^T of block i, whose keys are there
        const uint64_t ka = k_desc + static_cast<uint64_t>(k_st * SM::kKV >> 4);
        const uint32_t d = tmem_base + (i % kBufs) * PX_BN;
#pragma unroll
        for (int j = 0; j < D / 16; ++j)
          mma_f16_ss(d, qa + (((j >> 2) * (PX_BM * 128) + (j & 3) * 32) >> 4), ka + (((j >> 2) * (PX_BN * 128) + (j & 3) * 32) >> 4),
                     idesc_s, j != 0 ? 1u : 0u);
        mma_commit(&s_full[i % kBufs]);
        mma_commit(&kv_empty[k_st]);
        if (++k_st == kStages) { k_st = 0; k_ph ^= 1; }
      };
      bool good = n_blk > 0 && wait_for(q_full, 0, 1039, 0) && wait_for(&kv_full[0], 0, 1031, 0);
      if (good) { tc_fence_after_sync(); issue_s(0); }
      for (int i = 0; good && i < n_blk; ++i) {
        const bool more = i + 1 < n_blk;
        // what is known to come in time is waited for first: only P is on the way from S to S
        if (more) { good = wait_for(&kv_full[k_st], k_ph, 1031, i + 1); if (!good) break; }
        if (kBufs == 2 && more) { tc_fence_after_sync(); issue_s(i + 1); }
        good = wait_for(&kv_full[kStages + v_st], v_ph, 1038, i) && wait_for(&p_full[i % kBufs], (i / kBufs) & 1, 1032, i);
        if (!good) break;
        tc_fence_after_sync();
        const uint64_t va = v_desc + static_cast<uint64_t>(v_st * SM::kKV >> 4);
        const uint32_t a_t = tmem_base + (i % kBufs) * PX_BN;
#pragma unroll
        for (int j = 0; j < PX_BN / 16; ++j) {
          const uint64_t v16 = va + ((j * 2048) >> 4);
          if constexpr (kFine) {                                 // 32 keys: 16 columns of P, 16 of what its rounding left
            const uint32_t a16 = a_t + (j >> 1) * 32 + (j & 1) * 8;
            px_mma_ts(tmem_base + kTmemO, a16, v16, idesc_pv, (i | j) != 0 ? 1u : 0u);
            px_mma_ts(tmem_base + kTmemO, a16 + 16, v16, idesc_pv, 1u);
          } else {
            px_mma_ts(tmem_base + kTmemO, a_t + j * 8, v16, idesc_pv, (i | j) != 0 ? 1u : 0u);
          }
        }
        if (!more) mma_commit(o_full);
        else if (kBufs == 2) mma_commit(pv_done);
        // one buffer: S goes over P once P V has read it (the tensor core takes the products in order)
        mma_commit(&kv_empty[kStages + v_st]);
        if (kBufs == 1 && more) issue_s(i + 1);
        if (++v_st == kStages) { v_st = 0; v_ph ^= 1; }
      }
    }
    __syncwarp();
  } else if (softmax_warp) {
    // ------------------------------------------------------------ softmax, 32 rows a warp
    const uint32_t lane_addr = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tmem_o = tmem_base + kTmemO + lane_addr;
    const bool mine = my_row < n_valid;
    // bounds inside which no row of this warp needs a mask
    int w_lo = mine ? lo : 0, w_hi = mine ? hi : 0x7fffffff;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      w_lo = max(w_lo, __shfl_xor_sync(0xffffffffu, w_lo, o));
      w_hi = min(w_hi, __shfl_xor_sync(0xffffffffu, w_hi, o));
    }
    for (int i = 0; i < n_blk; ++i) {
      const int bf = i % kBufs;
      const uint32_t s_addr = tmem_base + lane_addr + bf * PX_BN;
      ok = px_wait(&s_full[bf], (i / kBufs) & 1, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) { if (lane == 0) report_status(p.status, kStatusWaitTimeout, 1033, i, 0); *abort_flag = 1; break; }
      tc_fence_after_sync();
      // S in halves of 32 keys, the first read twice: 80 registers a thread hold no more
      const int k0 = key0 + i * PX_BN;
      const bool edge = k0 < w_lo || k0 + PX_BN > w_hi;
      uint32_t r[32];
      auto half = [&](int hf) {
        tmem_ld_32x32b_x32(s_addr + hf * 32, r);
        tmem_ld_wait();
      };
      if (edge) {                                                            // masked scores go back, so that what follows stays short
#pragma unroll 1
        for (int hf = 0; hf < 2; ++hf) {
          half(hf);
          const int from = lo - k0 - hf * 32, to = hi - k0 - hf * 32;
#pragma unroll
          for (int t = 0; t < 32; ++t)
            if (t < from || t >= to) r[t] = 0xff800000u;                     // -inf
          tmem_st_32x32b_x32(s_addr + hf * 32, r);
        }
        tmem_st_wait();
      }
      float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};           // four chains: one would be 32 latencies long
#pragma unroll 1
      for (int hf = 0; hf < 2; ++hf) {
        half(hf);
#pragma unroll
        for (int t = 0; t < 32; t += 2)
          mx4[(t >> 1) & 3] = px_max3(mx4[(t >> 1) & 3], __uint_as_float(r[t]), __uint_as_float(r[t + 1]));
      }
      const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
      const float m_cand = fmaxf(m, mx * p.scale_log2);
      bool grow = m_cand - m > kPxRescale;
      if (i == 0) { grow = false; m = m_cand; }
      if (__any_sync(0xffffffffu, grow)) {
        if (kBufs == 2) {                                                    // O is final for the blocks before (one buffer: S says so)
          ok = px_wait(pv_done, (i - 1) & 1, abort_flag);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) { if (lane == 0) report_status(p.status, kStatusWaitTimeout, 1034, i, 0); *abort_flag = 1; break; }
          tc_fence_after_sync();
        }
        float alpha = 1.f;
        if (grow) { alpha = px_exp2(m - m_cand); m = m_cand; l *= alpha; }
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          tmem_ld_32x32b_x32(tmem_o + c * 32, o);
          tmem_ld_wait();
#pragma unroll
          for (int t = 0; t < 32; ++t) o[t] = __float_as_uint(__uint_as_float(o[t]) * alpha);
          tmem_st_32x32b_x32(tmem_o + c * 32, o);
        }
        tmem_st_wait();
      }
      const uint64_t sc2 = px_pack(p.scale_log2, p.scale_log2), nm2 = px_pack(-m, -m);
      uint64_t rs2[2] = {0, 0};                                              // pairs of partial sums, both halves 0.f
      auto exps = [&](uint32_t (&pk)[16]) {
#pragma unroll
        for (int t = 0; t < 32; t += 2) {
          float x0, x1;
          px_unpack(px_fma2(px_pack(__uint_as_float(r[t]), __uint_as_float(r[t + 1])), sc2, nm2), x0, x1);
          const float p0 = px_exp2(x0), p1 = px_exp2(x1);
          rs2[(t >> 1) & 1] = px_add2(rs2[(t >> 1) & 1], px_pack(p0, p1));
          if constexpr (kFine) px_split(p0, p1, pk[t >> 1], r[t >> 1]);
          else pk[t >> 1] = pack_bf16x2(p0, p1);
        }
      };
#pragma unroll 1
      for (int hf = 0; hf < 2; ++hf) {
        uint32_t pk[16];
        half(hf);
        exps(pk);
        if constexpr (kFine) {
          px_tmem_st_x16(s_addr + hf * 32, pk);                  // over the scores that were just read
          px_tmem_st_x16(s_addr + hf * 32 + 16, r);
        } else {
          px_tmem_st_x16(s_addr + hf * 16, pk);
        }
      }
      float sa, sb;
      px_unpack(px_add2(rs2[0], rs2[1]), sa, sb);
      l += sa + sb;
      tmem_st_wait();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[bf]);
    }
    // The end of the last P V has a barrier of its own: pv_done alternates its parity with every block, and when a
    // warp gets here it may still be two phases behind (P V of the block before runs after S of the last one) or done.
    if (ok && n_blk > 0) {
      ok = px_wait(o_full, 0, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) { if (lane == 0) report_status(p.status, kStatusWaitTimeout, 1035, 0, 0); *abort_flag = 1; }
    }
    tc_fence_after_sync();
  }
  if (*abort_flag) {
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);            // copies and MMAs in flight end before memory is given up
  }

  // ---------------------------------------------------------------- results
  float* sx = reinterpret_cast<float*>(sKV);                     // [PX_BM][D], 16-byte pieces swizzled by row
  float* s_ml = sx + PX_BM * D;                                  // [PX_BM][2]
  if (!kDirect) __syncthreads();                                  // every MMA of the CTA is done: the stages are free
  if (softmax_warp) {
    const uint32_t tmem_o = tmem_base + kTmemO + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    float f = 1.f;
    __nv_bfloat16* orow = nullptr;
    if (kDirect && my_row < n_valid) {
      const int rr = row0 + my_row, tok = rr / g, h = hk * g + rr - tok * g;
      f = px_factor(m, l, px_sink(p, h));
      orow = p.out + (static_cast<long long>(start + tok) * p.hq + h) * D;
    }
#pragma unroll 1
    for (int c = 0; c < D / 32; ++c) {
      uint32_t o[32];
      if (n_blk > 0) {
        tmem_ld_32x32b_x32(tmem_o + c * 32, o);
        tmem_ld_wait();
      } else {
#pragma unroll
        for (int t = 0; t < 32; ++t) o[t] = 0u;
      }
      if (kDirect) {
        if (my_row < n_valid) {
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            int4 v;
            uint32_t* vv = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              vv[e] = pack_bf16x2(__uint_as_float(o[8 * t + 2 * e]) * f, __uint_as_float(o[8 * t + 2 * e + 1]) * f);
            if (f == 0.f) v = make_int4(0, 0, 0, 0);
            reinterpret_cast<int4*>(orow + c * 32)[t] = v;
          }
        }
      } else if (my_row < n_valid) {
#pragma unroll
        for (int t = 0; t < 8; ++t)
          reinterpret_cast<uint4*>(sx + my_row * D)[(c * 8 + t) ^ (my_row & 7)] =
              make_uint4(o[4 * t], o[4 * t + 1], o[4 * t + 2], o[4 * t + 3]);
      }
    }
    if (!kDirect && my_row < n_valid) reinterpret_cast<float2*>(s_ml)[my_row] = make_float2(m, l);
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, SM::kTmemCols);
  }
  if constexpr (!kDirect) px_join<D, kThreads>(p, sx, s_ml, reinterpret_cast<float*>(sQ), start, row0, n_valid, hk, unit);
}

// ------------------------------------------------------------------------------------------------------------------
// Few rows (up to 40): the same attention where a tile of 128 would be mostly empty, as in decode steps.  It is bound by
// the bytes of K and V, so the matrix work goes where its results are easy to use: with keys as the rows of the warp-wide
// mma and 8 query rows as its columns, S^T = K Q^T and O^T += V^T P^T waste nothing at 8 rows, every lane exponentiates
// its own share (a tcgen05 tile gives a whole row of 64 keys to one lane: 1350 cycles a block for one busy warp), and no
// barrier is needed.  Each of four warps streams its own tiles of 16 or 32 keys through a ring of its own,
// with its own running maximum, sum and O; they meet once at the end.  P^T turns from accumulator to operand layout with
// movmatrix, in its two parts; the maximum is raised only when some key beats it by 2^8, which one vote a tile finds out.
// 64 sequences with 1..5 tokens over 300..4096 keys, 64/8 heads of 64: 70 us, 3.7 TB/s (62 with P in one part, when the stream
// itself ran at 5.5 TB/s; 73 with 40 rows for every list; the rest is 5 us of start-up latencies a CTA and the last wave).  Equal
// shares of all keys for 296 CTAs, with pieces joined afterwards, took 95 us: a start-up for every piece, and heads of one page no
// longer read together.
template <int D, int NT>
struct PxFew {
  static constexpr int kWarps = 4, kThreads = 128;
  // CTAs of an SM, as registers allow; the rings share what shared memory there is
  static constexpr int kCtas = D == 64 ? (NT == 1 ? 4 : NT == 2 ? 3 : 2) : (NT == 1 ? 3 : 2);
  static constexpr int kTile = kCtas > 2 || D == 128 ? 16 : 32;          // keys per tile
  static constexpr int kKV = kTile * D * 2;
  static constexpr int kRows = 8 * NT;
  static constexpr int kOStride = D + 4;                   // floats; a warp leaves its O in its ring
  static constexpr int kJoined = kRows * (D + 2 + kWarps) * 4;
  static constexpr int kRingMost = ((232448 / kCtas - 1024 - 128 - kJoined) / kWarps) & ~127;
  static constexpr int kStages = kRingMost / (2 * kKV) < 6 ? kRingMost / (2 * kKV) : 6;
  static constexpr int kRing = kStages * 2 * kKV;          // of a warp
  static_assert(kStages >= 2 && kRows * kOStride * 4 + kRows * 8 <= kRing, "O of a warp fits its ring");
  static constexpr int kBytes = kWarps * kRing + kJoined + 128;
};

NMOE_DEVICE void px_ldm(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
NMOE_DEVICE void px_ldm_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
NMOE_DEVICE uint32_t px_transpose(uint32_t v) {            // of an 8x8 matrix of 16-bit values over the warp
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
  return d;
}
NMOE_DEVICE void px_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// one list, its rows in NT columns of 8; F: the layout of the kernel it runs in
template <int D, int NT, typename F>
NMOE_DEVICE void px_few_list(const ExtendParams& p, uint8_t* smem, int b, int start, int n, int ctx, int n_valid) {
  constexpr int kTile = F::kTile, kStages = F::kStages, MT = kTile / 16, KS = D / 16;
  const float inv_g = 1.f / static_cast<float>(p.group);
  float* sx = reinterpret_cast<float*>(smem + F::kWarps * F::kRing);       // [rows][D], joined over the warps
  float* s_ml = sx + F::kRows * D;
  float* s_w = s_ml + F::kRows * 2;                                        // [rows][warps] what each warp's part counts for
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int units = p.splits * p.groups, unit = blockIdx.x, hk = blockIdx.y, g = p.group;
  const int* table = p.block_tables + (p.flat ? px_owner(p, lane) : b) * p.bt_stride;

  // keys of the list, and the bounds inside which no row needs a mask
  int k_begin, k_end, w_lo, w_hi;
  if (!p.flat) {                                                 // both bounds grow from token to token
    px_bounds(p, 0, n, ctx, false, k_begin, w_hi);
    px_bounds(p, n - 1, n, ctx, false, w_lo, k_end);
  } else {
    k_begin = w_hi = 0x7fffffff;
    k_end = w_lo = 0;
    for (int t = lane; t < n; t += 32) {
      int lo, hi;
      px_bounds(p, t, n, ctx, hk == 0 && unit == 0 && warp == 0, lo, hi);
      w_lo = max(w_lo, lo);
      w_hi = min(w_hi, hi);
      if (lo < hi) { k_begin = min(k_begin, lo); k_end = max(k_end, hi); }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      k_begin = min(k_begin, __shfl_xor_sync(0xffffffffu, k_begin, o));
      k_end = max(k_end, __shfl_xor_sync(0xffffffffu, k_end, o));
      w_lo = max(w_lo, __shfl_xor_sync(0xffffffffu, w_lo, o));
      w_hi = min(w_hi, __shfl_xor_sync(0xffffffffu, w_hi, o));
    }
  }
  const int tiles_all = k_end > k_begin ? (k_end - k_begin + kTile - 1) / kTile : 0;
  const int tile0 = px_share(tiles_all, unit, units), n_tiles = px_share(tiles_all, unit + 1, units) - tile0;
  const int n_mine = n_tiles > warp ? (n_tiles - warp + F::kWarps - 1) / F::kWarps : 0;      // tiles warp, warp + 4, ...
  const int key0 = (tiles_all > 0 ? k_begin : 0) + (tile0 + warp) * kTile;

  // loads: a lane looks one key up, the warp shares the addresses; a tile ahead, so that the lookup's latency is covered
  constexpr int kChunks = D / 8, kRowsPass = 32 / kChunks;
  const uint32_t ring = smem_u32(smem + warp * F::kRing);
  const long long row_bytes = static_cast<long long>(p.hkv) * D * 2, piece = (static_cast<long long>(hk) * D + lane % kChunks * 8) * 2;
  bool bad = false;
  auto look_up = [&](int i) -> int {                             // cache row of this lane's key in tile i, -1: zeros, -2: no such page
    const int key = key0 + i * F::kWarps * kTile + lane;
    if (lane >= kTile || i >= n_mine || key >= k_end) return -1;
    const int pi = p.block_shift >= 0 ? key >> p.block_shift : key / p.block_size;
    const int page = __ldg(table + pi);
    return page < 0 || page >= p.num_blocks ? -2 : page * p.block_size + (key - pi * p.block_size);
  };
  int ahead[kStages];
#pragma unroll
  for (int i = 0; i < kStages; ++i) ahead[i] = look_up(i);       // all the first tiles at once
  const bool direct = p.splits == 1 && p.part_mode == 0;         // nothing to join but the warps
  const int my_tok = px_div(threadIdx.x, inv_g);                 // thread r has the sink of row r ready for the end
  const float my_sink = direct && threadIdx.x < n_valid ? px_sink(p, hk * g + threadIdx.x - my_tok * g) : -INFINITY;
  // Q^T as B operands: column = row of the list, k = dims
  uint32_t qf[KS][NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = nt * 8 + (lane >> 2);
    const bool in = r < n_valid;
    const int tok = in ? r / g : 0, h = hk * g + (in ? r - tok * g : 0);
    const __nv_bfloat16* src = p.q + (start + tok) * p.q_stride + static_cast<long long>(h) * D + (lane & 3) * 2;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int e = 0; e < 2; ++e) qf[ks][nt][e] = in ? __ldg(reinterpret_cast<const uint32_t*>(src + ks * 16 + e * 8)) : 0u;
  }

  auto load = [&](int i, int row_of) {                           // asks for tile i (past the last one: an empty group)
    if (i < n_mine) {
      bad = bad || row_of == -2;
      const int c = lane % kChunks;
      const uint32_t kd = ring + (i % kStages) * (2 * F::kKV);
      const uint8_t *ksrc = reinterpret_cast<const uint8_t*>(p.k_cache) + piece, *vsrc = reinterpret_cast<const uint8_t*>(p.v_cache) + piece;
#pragma unroll
      for (int s = 0; s < kTile / kRowsPass; ++s) {
        const int r = s * kRowsPass + lane / kChunks;
        const int row = __shfl_sync(0xffffffffu, row_of, r);
        const long long from = max(row, 0) * row_bytes;
        const uint32_t bytes = row >= 0 ? 16u : 0u, o = r * (D * 2) + ((c ^ (r & 7)) << 4);
        px_cp16(kd + o, ksrc + from, bytes);
        px_cp16(kd + F::kKV + o, vsrc + from, bytes);
      }
    }
    px_cp_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) load(i, ahead[i]);
  int next = ahead[kStages - 1];

  float o[KS][NT][4], m[NT][2], l[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[ks][nt][e] = 0.f;
    m[nt][0] = m[nt][1] = -1e30f;
    l[nt][0] = l[nt][1] = 0.f;
  }
  // rows that ldmatrix reads for this lane: K as stored, V transposed
  const int kr = lane & 15, kc = lane >> 4;                      // key, 16-byte piece of the 16 dims
  const int vr = (lane & 7) + ((lane >> 4) << 3), vc = (lane >> 3) & 1;

  for (int i = 0; i < n_mine; ++i) {
    load(i + kStages - 1, next);
    next = look_up(i + kStages);
    px_cp_wait<kStages - 1>();
    __syncwarp();                                                // every lane's copies of tile i are there
    const uint32_t ks_addr = ring + (i % kStages) * (2 * F::kKV), vs_addr = ks_addr + F::kKV;
    float s[MT][NT][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[mt][nt][e] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        uint32_t a[4];
        const int r = mt * 16 + kr;
        px_ldm(ks_addr + r * (D * 2) + (((ks * 2 + kc) ^ (r & 7)) << 4), a);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) px_mma(s[mt][nt], a, qf[ks][nt][0], qf[ks][nt][1]);
      }
    }
    const int k0 = key0 + i * F::kWarps * kTile;
    if (k0 < w_lo || k0 + kTile > w_hi) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = nt * 8 + (lane & 3) * 2 + e;
          const int tok = px_div(r, inv_g);
          int lo = 0, hi = 0;
          if (r < n_valid) px_bounds(p, tok, n, ctx, false, lo, hi);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            const int ka = k0 + mt * 16 + (lane >> 2);
            if (ka < lo || ka >= hi) s[mt][nt][e] = -INFINITY;
            if (ka + 8 < lo || ka + 8 >= hi) s[mt][nt][2 + e] = -INFINITY;
          }
        }
    }
    float mx[NT][2];
    bool grow = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float v = fmaxf(s[0][nt][e], s[0][nt][2 + e]);
        if (MT == 2) v = px_max3(v, s[MT - 1][nt][e], s[MT - 1][nt][2 + e]);
        mx[nt][e] = v * p.scale_log2;
        grow = grow || mx[nt][e] > m[nt][e] + kPxRescale;
      }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float v = mx[nt][e];
#pragma unroll
          for (int w = 4; w < 32; w <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, w));
          const float up = fmaxf(m[nt][e], v), alpha = px_exp2(m[nt][e] - up);
          m[nt][e] = up;
          l[nt][e] *= alpha;
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) { o[ks][nt][e] *= alpha; o[ks][nt][2 + e] *= alpha; }
        }
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      uint32_t pf[NT][2], pr[NT][2];                             // P as a bf16 value and what it leaves, both as operands
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float e4[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) e4[e] = px_exp2(fmaf(s[mt][nt][e], p.scale_log2, -m[nt][e & 1]));
        l[nt][0] += e4[0] + e4[2];
        l[nt][1] += e4[1] + e4[3];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t high, rest;
          px_split(e4[2 * h], e4[2 * h + 1], high, rest);
          pf[nt][h] = px_transpose(high);
          pr[nt][h] = px_transpose(rest);
        }
      }
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        uint32_t a[4];
        const int r = mt * 16 + vr;
        px_ldm_t(vs_addr + r * (D * 2) + (((ks * 2 + vc) ^ (r & 7)) << 4), a);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) px_mma(o[ks][nt], a, pf[nt][0], pf[nt][1]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) px_mma(o[ks][nt], a, pr[nt][0], pr[nt][1]);
      }
    }
    __syncwarp();                                                // the stage may be filled again
  }
  px_cp_wait<0>();
  if (bad) report_status(p.status, kStatusBadIndex, 1022, b, 0);
  __syncwarp();

  // every warp leaves its rows in its ring, the CTA joins them
  float* wo = reinterpret_cast<float*>(smem + warp * F::kRing);
  float* wml = wo + F::kRows * F::kOStride;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = nt * 8 + (lane & 3) * 2 + e;
      float v = l[nt][e];
#pragma unroll
      for (int w = 4; w < 32; w <<= 1) v += __shfl_xor_sync(0xffffffffu, v, w);
      if (lane < 4) { wml[2 * r] = m[nt][e]; wml[2 * r + 1] = v; }
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        wo[r * F::kOStride + ks * 16 + (lane >> 2)] = o[ks][nt][e];
        wo[r * F::kOStride + ks * 16 + 8 + (lane >> 2)] = o[ks][nt][2 + e];
      }
    }
  __syncthreads();
  if (const int r = threadIdx.x; r < n_valid) {
    float2 ml[F::kWarps];
    float top = -1e30f, sum = 0.f, w[F::kWarps], f = 1.f;
#pragma unroll
    for (int k = 0; k < F::kWarps; ++k) {
      ml[k] = *reinterpret_cast<const float2*>(smem + k * F::kRing + F::kRows * F::kOStride * 4 + r * 8);
      if (ml[k].y != 0.f) top = fmaxf(top, ml[k].x);
    }
#pragma unroll
    for (int k = 0; k < F::kWarps; ++k) {
      w[k] = ml[k].y != 0.f ? px_exp2(ml[k].x - top) : 0.f;
      sum += w[k] * ml[k].y;
    }
    if (direct) f = px_factor(top, sum, my_sink);
    else reinterpret_cast<float2*>(s_ml)[r] = make_float2(top, sum);
#pragma unroll
    for (int k = 0; k < F::kWarps; ++k) s_w[r * F::kWarps + k] = w[k] * f;
  }
  __syncthreads();
#pragma unroll 2
  for (int i = threadIdx.x; i < n_valid * (D / 4); i += F::kThreads) {
    const int r = i / (D / 4), c = i % (D / 4), tok = px_div(r, inv_g), h = hk * g + r - tok * g;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < F::kWarps; ++k)
      px_axpy(acc, s_w[r * F::kWarps + k], *reinterpret_cast<const float4*>(smem + k * F::kRing + (r * F::kOStride + c * 4) * 4));
    if (direct) px_store(p.out + (static_cast<long long>(start + tok) * p.hq + h) * D + c * 4, acc, 1.f);
    else reinterpret_cast<float4*>(sx + r * D)[c ^ (r & 7)] = acc;
  }
  if (direct) return;
  px_join<D, F::kThreads>(p, sx, s_ml, reinterpret_cast<float*>(smem), start, 0, n_valid, hk, unit);
}

template <int D, int NT>
__global__ void __launch_bounds__(128, PxFew<D, NT>::kCtas) k_paged_few(const ExtendParams p) {
  using F = PxFew<D, NT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~uintptr_t(127));
  const int b = p.flat ? 0 : p.sorted ? px_nth_longest<F::kThreads>(p, blockIdx.z, reinterpret_cast<int*>(smem)) : blockIdx.z;
  int start, n, ctx;
  px_list(p, b, blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0, start, n, ctx);
  const int n_valid = min(F::kRows, n * p.group);                // the host launches this kernel only where all rows fit
  if (n_valid <= 0) {                                            // uniform over the cluster
    if (p.part_mode == 1) px_launch_dependents();
    if (p.part_mode == 2) px_wait_prior_grid();
    return;
  }
  if (p.part_mode == 1) px_launch_dependents();
  if constexpr (NT == 5) {                                       // a list with few of the rows that the longest one may have
    if (n_valid <= 24) { px_few_list<D, 3, F>(p, smem, b, start, n, ctx, n_valid); return; }
  }
  px_few_list<D, NT, F>(p, smem, b, start, n, ctx, n_valid);
}

// Joins the sets of the launches that split the keys over several clusters: D / 4 threads for the columns of a row, kParts of
// such groups for its sets (1 for a few sets and many rows; a CTA a row for the dozens of sets of a single long context,
// which took 32 us one after the other).
template <int D, int kParts>
struct PxJoin {
  static constexpr int kCols = D / 4, kThreads = kParts > 1 ? kCols * kParts : 128, kRows = kThreads / (kCols * kParts);
};
template <int D, int kParts>
__global__ void __launch_bounds__(PxJoin<D, kParts>::kThreads) k_paged_join(const ExtendParams p) {
  using J = PxJoin<D, kParts>;
  const int b = blockIdx.y, c = threadIdx.x % J::kCols, part = kParts > 1 ? threadIdx.x / J::kCols : 0;
  const int i = static_cast<int>(blockIdx.x) * J::kRows + (kParts > 1 ? 0 : threadIdx.x / J::kCols), h = i % p.hq, tok = i / p.hq;
  int start, n, ctx;
  px_list(p, b, false, start, n, ctx);
  px_wait_prior_grid();
  if (tok >= n) return;                                          // the whole CTA where it has one row
  const long long row = static_cast<long long>(start + tok) * p.hq + h;
  PxSum t;
  t.start(-1e30f);
  t.add_sets<D, (kParts > 1 ? 4 : 8)>(p, row, c, part, kParts);
  if constexpr (kParts > 1) {
    __shared__ float4 s_acc[kParts][J::kCols];
    __shared__ float2 s_ml[kParts];
    s_acc[part][c] = t.acc;
    if (c == 0) s_ml[part] = make_float2(t.top, t.sum);
    __syncthreads();
    if (part > 0) return;
    t.start(-1e30f);
#pragma unroll
    for (int q = 0; q < kParts; ++q) t.top = fmaxf(t.top, s_ml[q].x);
#pragma unroll
    for (int q = 0; q < kParts; ++q) t.add(s_ml[q], s_acc[q][c]);
  }
  t.store(p.out + row * D + c * 4, px_sink(p, h));
}

// How a call is cut: which kernel, tiles a list, CTAs the keys of a tile are split over.
struct PxPlan {
  int nt;                 // > 0: the kernel for few rows, 8 * nt of them
  long long tiles, slots;
  int splits, groups;
};

// `lists` row lists of up to `rows` rows that see at most `keys` keys each; groups only where partial sets may be written.
// (Times: those of few_most with P in two parts, the others as they were with one, on both sides of each choice.)
static PxPlan px_plan(int D, int hkv, long long rows, int lists, long long keys, bool may_group) {
  PxPlan q;
  // 64 sequences over 300..4096 keys, D = 64: 40 rows 84 us against 100 in the kernel for many rows, 24 rows 62 against 91 (one
  // context of 100000 keys: 40 rows 65 against 54, 24 rows 49 and 49); D = 128: 16 rows 76 against 74 (99k keys: 44 against 43), 8
  // rows 65 against 74 (42 against 43)
  const int few_most = D == 64 ? 40 : 16;
  q.nt = 0;
  q.tiles = 1;
  // CTAs the GPU holds at once; keys that make a split worth while (few rows, 3 sequences of 900..1000 keys: 8.0 us, with half of
  // that 9.2, with twice as many 9.7; many rows, 4 sequences of 2000..3000 keys: 18.3 us, 24.2 and 20.3)
  long long slots, least;
  if (rows <= few_most) {
    const int t = static_cast<int>((rows + 7) / 8);
    q.nt = t == 4 ? 5 : t;
    slots = 148 * (D == 64 ? (q.nt == 1 ? 4 : q.nt == 2 ? 3 : 2) : (q.nt == 1 ? 3 : 2));
    least = 128;
  } else {
    q.tiles = (rows + PX_BM - 1) / PX_BM;
    slots = D == 64 ? 4 * 148 : 2 * 148;
    least = 4 * PX_BN;
  }
  q.slots = slots;
  const long long base = q.tiles * lists * hkv;
  // Rounded down: a second wave of a few CTAs costs as much as a first one.  (32 sequences of 3000 keys each, 16 rows: 41 us,
  // rounded up 55; of 1000..8000 keys 82 and 64, but the lengths are not known here.)
  long long units = slots / (base > slots ? slots : base);
  const long long worth = keys / least;
  if (units > worth) units = worth;
  if (units < 1) units = 1;
  q.splits = 1;
  // One cluster does up to 8 splits in one launch.  More of them go to clusters of 2 and a launch that joins these: large
  // clusters leave SMs free that do not fill one (99k keys of one sequence: 84 us in clusters of 2, 113 in clusters of 8).
  const int most = may_group && units > 8 ? 2 : 8;
  while (q.splits * 2 <= most && q.splits * 2 <= units) q.splits *= 2;
  q.groups = may_group && units >= 2 * q.splits ? static_cast<int>(units / q.splits) : 1;
  return q;
}

template <auto kern, typename... More>
static cudaError_t px_launch(const ExtendParams& p, dim3 grid, int threads, int smem, bool dependent, cudaStream_t st, const More&... more) {
  static std::atomic<unsigned long long> ready{0};               // of this kernel: devices where its shared memory has been raised
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (smem > 0 && (dev > 63 || !((ready.load() >> dev) & 1))) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    if (dev <= 63) ready.fetch_or(1ull << dev);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  int n = 0;
  if (p.splits > 1) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n].val.clusterDim.x = p.splits; at[n].val.clusterDim.y = 1; at[n].val.clusterDim.z = 1;
    ++n;
  }
  if (dependent) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = at; cfg.numAttrs = n;
  e = cudaLaunchKernelEx(&cfg, kern, p, more...);
  return e == cudaSuccess ? cudaGetLastError() : e;
}

template <int D, int NT>
static cudaError_t px_few(const ExtendParams& p, dim3 grid, cudaStream_t st) {
  return px_launch<k_paged_few<D, NT>>(p, grid, PxFew<D, NT>::kThreads, PxFew<D, NT>::kBytes, p.part_mode == 2, st);
}
template <int D>
static cudaError_t px_many(const ExtendParams& p, dim3 grid, bool fine, cudaStream_t st) {
  // The maps are made for every call: they take a fraction of a microsecond, and nothing is kept by an address.
  CUtensorMap tk{}, tv{};
  const uint64_t inner = static_cast<uint64_t>(p.hkv) * D, rows = static_cast<uint64_t>(p.num_blocks) * p.block_size;
  ExtendParams a = p;
  // Boxes of as many keys as both a page and a block are whole multiples of, from 4 on (8 prompts: boxes of 16 keys 600 us, of 8
  // 629, of 4 759, of 2 1018; by hand 982 to 1048).
  const int low = p.block_size & -p.block_size;
  a.tma_rows = low >= PX_BN ? PX_BN : low >= 4 ? low : 0;
  if (a.tma_rows > 0) {
    const int rc = make_tensor_map_2d(&tk, p.k_cache, kTmaBf16, inner, rows, inner * 2, 64, a.tma_rows, kTmaSwizzle128) |
                   make_tensor_map_2d(&tv, p.v_cache, kTmaBf16, inner, rows, inner * 2, 64, a.tma_rows, kTmaSwizzle128);
    if (rc != 0) a.tma_rows = 0;                                 // then every block is copied by hand
  }
  const int threads = PxSmem<D>::kThreads, smem = PxSmem<D>::kBytes;
  const bool direct = p.splits == 1 && p.part_mode == 0, dependent = p.part_mode == 2;
  if (fine)
    return direct ? px_launch<k_paged_extend<D, true, true>>(a, grid, threads, smem, false, st, tk, tv)
                  : px_launch<k_paged_extend<D, false, true>>(a, grid, threads, smem, dependent, st, tk, tv);
  return direct ? px_launch<k_paged_extend<D, true, false>>(a, grid, threads, smem, false, st, tk, tv)
                : px_launch<k_paged_extend<D, false, false>>(a, grid, threads, smem, dependent, st, tk, tv);
}

template <int D, int kParts>
static cudaError_t px_join_launch(const ExtendParams& p, long long rows, int B, cudaStream_t st) {
  using J = PxJoin<D, kParts>;
  return px_launch<k_paged_join<D, kParts>>(p, dim3(static_cast<unsigned>((rows + J::kRows - 1) / J::kRows), B), J::kThreads, 0, true, st);
}

static int px_run(ExtendParams& p, const PxPlan& q, int D, int lists, cudaStream_t st) {
  if (q.tiles * q.splits * q.groups > 0x3fffffff) return -5;
  p.splits = q.splits;
  p.groups = q.groups;
  p.sorted = !p.flat && lists > 1 && lists <= PX_SORT_MOST && q.tiles * q.splits * q.groups * p.hkv * lists > q.slots;
  const dim3 grid(static_cast<unsigned>(q.tiles) * q.splits * q.groups, p.hkv, lists);
  // steps of a few tokens: P in two parts, see the head of this file
  const bool fine = p.flat || q.tiles == 1 || p.max_q_len == 1;
  cudaError_t e;
  if (D == 64) {
    switch (q.nt) {
      case 0: e = px_many<64>(p, grid, fine, st); break;
      case 1: e = px_few<64, 1>(p, grid, st); break;
      case 2: e = px_few<64, 2>(p, grid, st); break;
      case 3: e = px_few<64, 3>(p, grid, st); break;
      default: e = px_few<64, 5>(p, grid, st); break;
    }
  } else {
    switch (q.nt) {
      case 0: e = px_many<128>(p, grid, fine, st); break;
      case 1: e = px_few<128, 1>(p, grid, st); break;
      default: e = px_few<128, 2>(p, grid, st); break;
    }
  }
  return e == cudaSuccess ? 0 : static_cast<int>(e);
}

// The launches of a call.  One row list a sequence: `own`, and a join where its keys are split over several clusters.  A shared
// prefix: `pre` for its keys, then `own` for each sequence's, whose CTAs join pre's sets.  (Letting own run beside pre and
// joining both in a third launch gained nothing: 128 sequences behind 1504 keys 45 -> 46 us, pre leaves few places free.)
struct PxCall {
  PxPlan own, pre;
  bool shared, join;
  int sets;
};

static PxCall px_call(int B, int Hq, int Hkv, int D, int block_size, int max_blocks, int max_q_len, int window, int prefix_len) {
  const long long capacity = static_cast<long long>(max_blocks) * block_size, seen = prefix_len > 0 ? capacity - prefix_len : capacity;
  const long long reach = window > 0 ? static_cast<long long>(window) + max_q_len : seen, keys = reach < seen ? reach : seen;
  const int g = Hq / Hkv;
  PxCall c{};
  c.shared = prefix_len > 0;
  c.own = px_plan(D, Hkv, static_cast<long long>(max_q_len) * g, B, keys, !c.shared);
  if (c.shared) {
    c.pre = px_plan(D, Hkv, static_cast<long long>(B) * g, 1, prefix_len, true);
    c.sets = c.pre.groups;
  } else {
    c.join = c.own.groups > 1;
    c.sets = c.join ? c.own.groups : 0;
  }
  return c;
}

}  // namespace nmoe

using namespace nmoe;

// Floats of workspace that nmoe_paged_extend needs for a call of these sizes (0: none).
extern "C" long long nmoe_paged_extend_workspace(int n_rows, int B, int Hq, int Hkv, int D, int block_size, int max_blocks,
                                                 int max_q_len, int window, int prefix_len) {
  if (B < 1 || n_rows < 1 || max_q_len < 1 || Hkv < 1 || Hq < Hkv || max_blocks < 0 || block_size < 1) return 0;
  return px_call(B, Hq, Hkv, D, block_size, max_blocks, max_q_len, window, prefix_len).sets * static_cast<long long>(n_rows) * Hq * (D + 2);
}

// Kernels that such a call launches.
extern "C" int nmoe_paged_extend_launches(int B, int Hq, int Hkv, int D, int block_size, int max_blocks, int max_q_len, int window,
                                          int prefix_len) {
  if (B < 1 || max_q_len < 1 || Hkv < 1 || Hq < Hkv || max_blocks < 0 || block_size < 1) return 0;
  const PxCall c = px_call(B, Hq, Hkv, D, block_size, max_blocks, max_q_len, window, prefix_len);
  return 1 + (c.shared ? 1 : 0) + (c.join ? 1 : 0);
}

// q [n_rows, Hq, D] (rows q_stride apart), out [n_rows, Hq, D]; caches [num_blocks, block_size, Hkv, D]; block_tables [B] rows
// of max_blocks entries, bt_stride apart; context_lens, q_starts, q_lens [B].  prefix_len > 0: one token per sequence
// (q_starts, q_lens null) behind that many common keys.  workspace: see above.
extern "C" int nmoe_paged_extend(const void* q, long long q_stride, const void* k_cache, const void* v_cache,
                                 const int* block_tables, long long bt_stride, const int* context_lens,
                                 const int* q_starts, const int* q_lens, const void* sinks, int sinks_fp32, void* out,
                                 int n_rows, int B, int Hq, int Hkv, int D, int block_size, int num_blocks, int max_blocks,
                                 int max_q_len, int window, float scale, int prefix_len, float* workspace,
                                 long long workspace_floats, void* status, cudaStream_t st) {
  if (B == 0 || n_rows == 0 || max_q_len == 0) return 0;
  if (n_rows < 0 || max_q_len < 0 || max_blocks < 0 || num_blocks < 0 || Hkv < 1 || Hkv > 65535 || Hq < Hkv || Hq % Hkv != 0 || block_size < 1 || B < 0 || B > 65535 || !(scale > 0.f)) return -1;
  if (D != 64 && D != 128) return -2;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) |
       reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) % 16 != 0 || (n_rows > 1 && q_stride % 8 != 0)) return -3;
  if (static_cast<long long>(n_rows) * Hq > 0x7fffffffll / (D / 8) - 256 || static_cast<long long>(num_blocks) * block_size > 0x7fffffffll) return -4;
  if (prefix_len > 0 && (q_starts != nullptr || q_lens != nullptr)) return -5;
  if (workspace_floats < nmoe_paged_extend_workspace(n_rows, B, Hq, Hkv, D, block_size, max_blocks, max_q_len, window, prefix_len)) return -6;
  const PxCall c = px_call(B, Hq, Hkv, D, block_size, max_blocks, max_q_len, window, prefix_len);
  ExtendParams p{};
  p.q = static_cast<const __nv_bfloat16*>(q); p.k_cache = static_cast<const __nv_bfloat16*>(k_cache);
  p.v_cache = static_cast<const __nv_bfloat16*>(v_cache); p.out = static_cast<__nv_bfloat16*>(out);
  p.block_tables = block_tables; p.context_lens = context_lens; p.q_starts = q_starts; p.q_lens = q_lens; p.sinks = sinks;
  p.status = static_cast<StatusRecord*>(status); p.q_stride = q_stride; p.bt_stride = bt_stride; p.n_rows = n_rows;
  p.n_seqs = B; p.hq = Hq; p.hkv = Hkv; p.group = Hq / Hkv; p.block_size = block_size; p.num_blocks = num_blocks;
  p.block_shift = -1;
  for (int s = 0; s < 31; ++s)
    if (block_size == 1 << s) p.block_shift = s;
  const long long capacity = static_cast<long long>(max_blocks) * block_size;
  p.capacity = static_cast<int>(capacity < 0x7fffff00ll ? capacity : 0x7fffff00ll);
  p.max_q_len = max_q_len; p.window = window; p.sinks_fp32 = sinks_fp32;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.set_rows = static_cast<long long>(n_rows) * Hq;
  p.n_sets = c.sets;
  p.part_o = workspace;
  p.part_ml = workspace != nullptr ? workspace + p.n_sets * p.set_rows * D : nullptr;
  p.key_end = 0x7fffffff;
  if (c.shared) {
    ExtendParams f = p;
    f.flat = 1; f.part_mode = 1; f.key_end = prefix_len;
    const int rc = px_run(f, c.pre, D, 1, st);
    if (rc != 0) return rc;
    p.key_begin = prefix_len;
    p.part_mode = 2;
  } else if (c.join) {
    p.part_mode = 1;
  }
  const int rc = px_run(p, c.own, D, B, st);
  if (rc != 0 || !c.join) return rc;
  p.splits = 1;
  const long long rows = static_cast<long long>(max_q_len) * Hq;
  cudaError_t e;
  if (p.n_sets > 8) e = D == 64 ? px_join_launch<64, 16>(p, rows, B, st) : px_join_launch<128, 8>(p, rows, B, st);
  else e = D == 64 ? px_join_launch<64, 1>(p, rows, B, st) : px_join_launch<128, 1>(p, rows, B, st);
  return e == cudaSuccess ? 0 : static_cast<int>(e);
}
