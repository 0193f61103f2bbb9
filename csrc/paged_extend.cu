// Attention of several new tokens per sequence over the paged cache, on tcgen05: drafted tokens of a decode step, the
// part of a prompt behind a cached prefix, and a whole batch of single tokens over the keys of a prefix they share.
//   out = sum_j softmax_j(scale * q . k_j | sink) * v_j       over the keys j that a token sees
//
// Rows.  The g query heads of a key/value head and the tokens that read the same keys are stacked: row = token * g +
// head of the group, 128 rows to a tile, so every K/V block is read once for all of them.  Each row carries its own
// bounds [lo, hi) of visible keys (causal end, window, shared part); a block that lies inside all of them needs no mask.
//
// Pipeline of a CTA, 64 keys at a time: four loader warps gather the block's K and V rows from their pages with
// cp.async (16 bytes a lane, any page size, zero fill outside the CTA's keys, so that what lies there cannot reach the
// products), one thread issues the MMAs (S of block i+1 before P V of block i), four warps per tile own 32 rows each:
// running maximum and sum in fp32, P as bf16 back to tensor memory as the A operand of P V.  The running maximum is
// raised only when it grows by more than 2^8; the stale one is exact after the final division.  P is rounded to bf16
// because the tensor core multiplies it with bf16 values; the sum l takes the unrounded p.
//
// Few rows: the keys are split over the CTAs of a cluster, whose (m, l, O) meet in distributed shared memory: no
// workspace, no atomics, one launch, the same bits on every run.  Shared prefix: one launch for the prefix (rows of all
// sequences, partial (m, l, O) to a workspace), a dependent launch for each sequence's own keys that starts while the
// first one drains and joins its rows at the end.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common/ptx.cuh"

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
  int n_rows, n_seqs, hq, hkv, group, block_size, block_shift, num_blocks, max_blocks, max_q_len, window, sinks_fp32;
  int key_begin, key_end;             // only keys in [key_begin, key_end) count here
  int flat;                           // 1: the tokens of all sequences are one list that reads the first sequence's pages
  int splits;                         // CTAs of a cluster = splits of the keys
  int part_mode;                      // 0 none, 1 write partial results, 2 join those of the launch before
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
NMOE_DEVICE void px_cp16(uint32_t dst, const void* src, uint32_t bytes) {      // bytes 0: the 16 bytes become zero
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
NMOE_DEVICE void px_cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
NMOE_DEVICE void px_cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
NMOE_DEVICE void px_launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
NMOE_DEVICE void px_wait_prior_grid() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Layout of shared memory.  D = 64: 4 stages of 16 KB, with one row tile two CTAs fit an SM; D = 128: 32 KB stages,
// one CTA an SM.  The exchange of partial results reuses the stages (O as fp32, 16-byte pieces swizzled by row).
template <int D, int TILES>
struct PxSmem {
  // loader threads: two warps keep the two CTAs of an SM at 8 warps and 128 registers each
  static constexpr int kLoaders = D == 64 && TILES == 1 ? 64 : 128;
  static constexpr int kThreads = 4 * TILES * 32 + 32 + kLoaders;
  static constexpr int kStages = 4;
  static constexpr int kQTile = PX_BM * D * 2;
  static constexpr int kKV = PX_BN * D * 2;                // one of K, V
  static constexpr int kStage = 2 * kKV;
  static constexpr int kRing = kStages * kStage;
  static constexpr int kExchange = TILES * PX_BM * (D + 2) * 4;
  static constexpr int kBody = kRing > kExchange ? kRing : kExchange;
  static constexpr int kBytes = TILES * kQTile + kBody + 256 + 1024;
};

template <int D, int TILES>
__global__ void __launch_bounds__(PxSmem<D, TILES>::kThreads, (D == 64 && TILES == 1) ? 2 : 1)
k_paged_extend(const ExtendParams p) {
  using SM = PxSmem<D, TILES>;
  constexpr int kStages = SM::kStages;
  constexpr int kLag = 2;                    // see the loader
  constexpr int kRows = TILES * PX_BM;
  constexpr int kThreads = SM::kThreads;
  constexpr int kMmaWarp = 4 * TILES;
  constexpr uint32_t kTmemCols = TILES == 1 ? 256 : 512;
  constexpr uint32_t kTmemO = TILES * 128;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sKV = sQ + TILES * SM::kQTile;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sKV + SM::kBody);
  uint64_t* kv_full = bars;                  // [kStages]
  uint64_t* kv_empty = kv_full + kStages;    // [kStages]
  uint64_t* s_full = kv_empty + kStages;     // [tile][buf]
  uint64_t* p_full = s_full + 2 * TILES;     // [tile][buf]
  uint64_t* pv_done = p_full + 2 * TILES;    // [tile]
  uint64_t* o_full = pv_done + TILES;        // [tile]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_full + TILES);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* s_range = reinterpret_cast<int*>(tmem_slot + 2);          // [2] first key, end of keys

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int splits = p.splits, rank = static_cast<int>(blockIdx.x) % splits;
  const int n_tiles_x = static_cast<int>(gridDim.x) / splits;
  // tiles with the longest contexts (the last ones of a prompt) first: better tail
  const int tile_x = n_tiles_x - 1 - static_cast<int>(blockIdx.x) / splits;
  const int hk = blockIdx.y, b = p.flat ? 0 : blockIdx.z, g = p.group;

  // ---------------------------------------------------------------- what this CTA works on
  int start, n, ctx = 0;
  const int capacity = static_cast<int>(min(static_cast<long long>(p.max_blocks) * p.block_size, 0x7fffffffll));
  const bool speaker = tile_x == 0 && rank == 0 && hk == 0 && threadIdx.x == 0;
  bool live = true;
  if (p.flat) {
    start = 0;
    n = p.n_seqs;
  } else {
    start = p.q_starts != nullptr ? p.q_starts[b] : b;
    n = p.q_lens != nullptr ? p.q_lens[b] : 1;
    ctx = p.context_lens[b];
    if (start < 0 || n < 0 || start > p.n_rows || n > p.n_rows - start || n > p.max_q_len) {
      if (speaker) report_status(p.status, kStatusBadIndex, 1020, b, start);
      live = false;
    } else if (ctx > capacity) {
      if (speaker) report_status(p.status, kStatusBadIndex, 1021, b, ctx);
      ctx = capacity;
    }
  }
  const int row0 = tile_x * kRows;                               // first row of this CTA's tiles
  const int n_valid = live ? min(kRows, n * g - row0) : 0;       // rows that exist
  if (n_valid <= 0) {                                            // uniform over the cluster
    if (p.part_mode == 1) px_launch_dependents();
    if (p.part_mode == 2) px_wait_prior_grid();
    return;
  }
  const int* table = p.block_tables + b * p.bt_stride;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) { mbar_init(&kv_full[i], SM::kLoaders / 32); mbar_init(&kv_empty[i], 1); }
    for (int t = 0; t < TILES; ++t) {
      const int rows = min(PX_BM, n_valid - t * PX_BM);
      const int warps = rows > 0 ? (rows + 31) / 32 : 1;
      for (int i = 0; i < 2; ++i) { mbar_init(&s_full[2 * t + i], 1); mbar_init(&p_full[2 * t + i], warps); }
      mbar_init(&pv_done[t], 1);
      mbar_init(&o_full[t], 1);
    }
    s_range[0] = 0x7fffffff;
    s_range[1] = 0;
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  // rows of Q, 128-byte swizzle, K-major; rows that do not exist are zero
  for (int i = threadIdx.x; i < kRows * (D / 8); i += kThreads) {
    const int r = i / (D / 8), c = i % (D / 8), rr = row0 + r;
    int4 v = make_int4(0, 0, 0, 0);
    if (r < n_valid) {
      const int tok = rr / g, h = hk * g + rr - tok * g;
      v = ld_nc_v4(p.q + (start + tok) * p.q_stride + static_cast<long long>(h) * D + c * 8);
    }
    *reinterpret_cast<int4*>(sQ + (r >> 7) * SM::kQTile + (c >> 3) * (PX_BM * 128) + (r & 127) * 128 + (((c & 7) ^ (r & 7)) << 4)) = v;
  }
  fence_proxy_async_smem();
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  // every CTA holds its tensor memory before a dependent launch may ask for some
  if (p.part_mode == 1) px_launch_dependents();

  // bounds of this thread's row
  int lo = 0, hi = 0;
  const int my_row = threadIdx.x;                                // softmax threads: row inside the CTA's tiles
  if (warp < 4 * TILES && my_row < n_valid) {
    const int tok = (row0 + my_row) / g;
    int pos;
    if (p.flat) {
      const int c = p.context_lens[tok];
      if (c > capacity && hk == 0 && rank == 0 && (row0 + my_row) % g == 0) report_status(p.status, kStatusBadIndex, 1021, tok, c);
      pos = min(c, capacity) - 1;
    } else {
      pos = ctx - n + tok;
    }
    lo = max(p.window > 0 ? max(0, pos - p.window + 1) : 0, p.key_begin);
    hi = min(pos + 1, p.key_end);
    if (lo < hi) {
      atomicMin(&s_range[0], lo);
      atomicMax(&s_range[1], hi);
    }
  }
  __syncthreads();
  const int k_begin = s_range[0], k_end = s_range[1];
  const int n_blocks_all = k_end > k_begin ? (k_end - k_begin + PX_BN - 1) / PX_BN : 0;
  const int blk0 = static_cast<int>(static_cast<long long>(n_blocks_all) * rank / splits);
  const int n_blk = static_cast<int>(static_cast<long long>(n_blocks_all) * (rank + 1) / splits) - blk0;
  const int key0 = n_blk > 0 ? k_begin + blk0 * PX_BN : 0;       // first key of this CTA

  bool ok = true;
  float m = -1e30f, l = 0.f;
  if (warp > kMmaWarp) {
    // ------------------------------------------------------------ loaders: K and V rows of a block from their pages
    // Blocks are announced in order once they have landed: normally kLag blocks after they were asked for, all at once
    // when the ring is full, since the block that would make room may be waiting for one of them.
    // Each warp owns kRowsWarp keys of a block; a lane looks one of them up (a block ahead, so that the page table's
    // latency is covered) and the warp shares the addresses by shuffle: a lookup per copied piece took 2500 cycles a block.
    constexpr int kChunks = D / 8, kRowsWarp = PX_BN / (SM::kLoaders / 32), kRowsPass = 32 / kChunks;
    static_assert(kRowsWarp <= 32 && kRowsWarp % kRowsPass == 0, "one lookup per lane");
    const int lw = warp - kMmaWarp - 1;
    const int c = lane % kChunks, rp = lane / kChunks;
    const long long row_elems = static_cast<long long>(p.hkv) * D;
    const long long head_off = static_cast<long long>(hk) * D;
    auto look_up = [&](int i) -> long long {                     // element offset of this lane's key in block i, -1: zeros
      const int key = key0 + i * PX_BN + lw * kRowsWarp + lane;
      if (lane >= kRowsWarp || i >= n_blk || key >= k_end) return -1;
      const int pi = p.block_shift >= 0 ? key >> p.block_shift : key / p.block_size;
      const int page = __ldg(table + pi);
      if (page < 0 || page >= p.num_blocks) return -2;
      return (static_cast<long long>(page) * p.block_size + (key - pi * p.block_size)) * row_elems + head_off;
    };
    long long next = look_up(0);
    bool bad = false;
    int told = 0;                                                // blocks announced so far
    auto announce = [&](int upto) {                              // this thread's copies of the blocks before upto have landed
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0)
        for (int t = told; t < upto; ++t) mbar_arrive(&kv_full[t % kStages]);
      told = upto;
    };
    for (int i = 0; i < n_blk && ok; ++i) {
      const int st = i % kStages;
      const uint32_t empty_ph = ((i / kStages) & 1) ^ 1;
      if (!__all_sync(0xffffffffu, px_test(&kv_empty[st], empty_ph))) {
        if (told < i) { px_cp_wait<0>(); announce(i); }
        ok = px_wait(&kv_empty[st], empty_ph, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) { if (lane == 0) report_status(p.status, kStatusWaitTimeout, 1030, i, 0); *abort_flag = 1; break; }
      }
      const uint32_t kd = smem_u32(sKV + st * SM::kStage), vd = kd + SM::kKV;
      const long long mine = next;
      bad = bad || mine == -2;
      next = look_up(i + 1);
#pragma unroll
      for (int s = 0; s < kRowsWarp / kRowsPass; ++s) {
        const int rw = s * kRowsPass + rp, r = lw * kRowsWarp + rw;
        const long long at = __shfl_sync(0xffffffffu, mine, rw);
        const uint32_t bytes = at >= 0 ? 16 : 0;
        const long long from = at >= 0 ? at + c * 8 : 0;
        const uint32_t o = (c >> 3) * (PX_BN * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4);
        px_cp16(kd + o, p.k_cache + from, bytes);
        px_cp16(vd + o, p.v_cache + from, bytes);
      }
      px_cp_commit();
      if (i - kLag >= told) { px_cp_wait<kLag>(); announce(i - kLag + 1); }
    }
    px_cp_wait<0>();
    if (ok && told < n_blk) announce(n_blk);
    if (bad) report_status(p.status, kStatusBadIndex, 1022, b, 0);
  } else if (warp == kMmaWarp) {
    // ------------------------------------------------------------ MMA issue
    if (elect_one()) {
      constexpr uint32_t idesc_s = make_idesc_bf16(PX_BM, PX_BN, 0, 0);
      constexpr uint32_t idesc_pv = make_idesc_bf16(PX_BM, D, 0, 1);
      auto issue_s = [&](int i) -> bool {
        const int st = i % kStages;
        if (!px_wait(&kv_full[st], (i / kStages) & 1, abort_flag)) { report_status(p.status, kStatusWaitTimeout, 1031, i, 0); *abort_flag = 1; return false; }
        tc_fence_after_sync();
        const uint64_t ka = make_smem_desc(smem_u32(sKV + st * SM::kStage), 0, 1024, kSwizzle128B);
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
          if (t * PX_BM >= n_valid) continue;
          const uint64_t qa = make_smem_desc(smem_u32(sQ + t * SM::kQTile), 0, 1024, kSwizzle128B);
          const uint32_t d = tmem_base + t * 128 + (i & 1) * PX_BN;
#pragma unroll
          for (int j = 0; j < D / 16; ++j)
            mma_f16_ss(d, qa + (((j >> 2) * (PX_BM * 128) + (j & 3) * 32) >> 4), ka + (((j >> 2) * (PX_BN * 128) + (j & 3) * 32) >> 4),
                       idesc_s, j != 0 ? 1u : 0u);
          mma_commit(&s_full[t * 2 + (i & 1)]);
        }
        return true;
      };
      bool good = n_blk > 0 && issue_s(0);
      for (int i = 0; good && i < n_blk; ++i) {
        if (i + 1 < n_blk) { good = issue_s(i + 1); if (!good) break; }
        const int st = i % kStages;
        const uint64_t va = make_smem_desc(smem_u32(sKV + st * SM::kStage + SM::kKV), PX_BN * 128, 1024, kSwizzle128B);
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
          if (t * PX_BM >= n_valid) continue;
          if (!px_wait(&p_full[t * 2 + (i & 1)], (i >> 1) & 1, abort_flag)) { report_status(p.status, kStatusWaitTimeout, 1032, i, t); *abort_flag = 1; good = false; break; }
          tc_fence_after_sync();
          const uint32_t a_t = tmem_base + t * 128 + (i & 1) * PX_BN;
#pragma unroll
          for (int j = 0; j < PX_BN / 16; ++j)
            px_mma_ts(tmem_base + kTmemO + t * D, a_t + j * 8, va + ((j * 2048) >> 4), idesc_pv, (i | j) != 0 ? 1u : 0u);
          mma_commit(i + 1 < n_blk ? &pv_done[t] : &o_full[t]);
        }
        mma_commit(&kv_empty[st]);
      }
    }
    __syncwarp();
  } else if ((warp >> 2) * PX_BM + (warp & 3) * 32 < n_valid) {
    // ------------------------------------------------------------ softmax: warp -> (tile, 32 rows)
    const int tile = warp >> 2;
    const uint32_t lane_addr = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tmem_o = tmem_base + kTmemO + tile * D + lane_addr;
    const bool mine = my_row < n_valid;
    // bounds inside which no row of this warp needs a mask
    int w_lo = mine ? lo : 0, w_hi = mine ? hi : 0x7fffffff;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      w_lo = max(w_lo, __shfl_xor_sync(0xffffffffu, w_lo, o));
      w_hi = min(w_hi, __shfl_xor_sync(0xffffffffu, w_hi, o));
    }
    for (int i = 0; i < n_blk; ++i) {
      const int bf = i & 1;
      const uint32_t s_addr = tmem_base + lane_addr + tile * 128 + bf * PX_BN;
      ok = px_wait(&s_full[tile * 2 + bf], (i >> 1) & 1, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) { if (lane == 0) report_status(p.status, kStatusWaitTimeout, 1033, i, tile); *abort_flag = 1; break; }
      tc_fence_after_sync();
      uint32_t r[PX_BN];
      tmem_ld_32x32b_x32(s_addr, r);
      tmem_ld_32x32b_x32(s_addr + 32, r + 32);
      tmem_ld_wait();
      const int k0 = key0 + i * PX_BN;
      if (k0 < w_lo || k0 + PX_BN > w_hi) {
        const int from = lo - k0, to = hi - k0;
#pragma unroll
        for (int t = 0; t < PX_BN; ++t)
          if (t < from || t >= to) r[t] = 0xff800000u;                       // -inf
      }
      float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};           // four chains: one would be 64 latencies long
#pragma unroll
      for (int t = 0; t < PX_BN; t += 2)
        mx4[(t >> 1) & 3] = px_max3(mx4[(t >> 1) & 3], __uint_as_float(r[t]), __uint_as_float(r[t + 1]));
      const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
      const float m_cand = fmaxf(m, mx * p.scale_log2);
      bool grow = m_cand - m > kPxRescale;
      if (i == 0) { grow = false; m = m_cand; }
      if (__any_sync(0xffffffffu, grow)) {
        ok = px_wait(&pv_done[tile], (i - 1) & 1, abort_flag);               // O is final for the blocks before
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) { if (lane == 0) report_status(p.status, kStatusWaitTimeout, 1034, i, tile); *abort_flag = 1; break; }
        tc_fence_after_sync();
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
      uint64_t rs2[4] = {0, 0, 0, 0};                                        // pairs of partial sums, both halves 0.f
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        uint32_t pk[16];
#pragma unroll
        for (int t = 0; t < 32; t += 2) {
          float x0, x1;
          px_unpack(px_fma2(px_pack(__uint_as_float(r[hf * 32 + t]), __uint_as_float(r[hf * 32 + t + 1])), sc2, nm2), x0, x1);
          const float p0 = px_exp2(x0), p1 = px_exp2(x1);
          rs2[(t >> 1) & 3] = px_add2(rs2[(t >> 1) & 3], px_pack(p0, p1));
          pk[t >> 1] = pack_bf16x2(p0, p1);
        }
        px_tmem_st_x16(s_addr + hf * 16, pk);
      }
      float sa, sb;
      px_unpack(px_add2(px_add2(rs2[0], rs2[1]), px_add2(rs2[2], rs2[3])), sa, sb);
      l += sa + sb;
      tmem_st_wait();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[tile * 2 + bf]);
    }
    // The end of the last P V has a barrier of its own: pv_done alternates its parity with every block, and when a
    // warp gets here it may still be two phases behind (P V of the block before runs after S of the last one) or done.
    if (ok && n_blk > 0) {
      ok = px_wait(&o_full[tile], 0, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) { if (lane == 0) report_status(p.status, kStatusWaitTimeout, 1035, 0, tile); *abort_flag = 1; }
    }
    tc_fence_after_sync();
  }
  if (*abort_flag) {
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);            // copies and MMAs in flight end before memory is given up
  }

  // ---------------------------------------------------------------- results
  const bool softmax_warp = warp < 4 * TILES && (warp >> 2) * PX_BM + (warp & 3) * 32 < n_valid;
  const bool direct = splits == 1 && p.part_mode == 0;
  float* sx = reinterpret_cast<float*>(sKV);                     // [kRows][D], 16-byte pieces swizzled by row
  float* s_ml = sx + kRows * D;                                  // [kRows][2]
  auto sink_of = [&](int h) -> float {                           // log2 units
    if (p.sinks == nullptr) return -INFINITY;
    return 1.4426950408889634f * (p.sinks_fp32 ? static_cast<const float*>(p.sinks)[h]
                                               : __bfloat162float(static_cast<const __nv_bfloat16*>(p.sinks)[h]));
  };
  if (!direct) __syncthreads();                                  // every MMA of the CTA is done: the stages are free
  if (softmax_warp) {
    const uint32_t tmem_o = tmem_base + kTmemO + (warp >> 2) * D + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    float f = 1.f;
    __nv_bfloat16* orow = nullptr;
    if (direct && my_row < n_valid) {
      const int rr = row0 + my_row, tok = rr / g, h = hk * g + rr - tok * g;
      const float sk = sink_of(h), mm = fmaxf(m, sk);
      f = l > 0.f ? px_exp2(m - mm) / (l * px_exp2(m - mm) + px_exp2(sk - mm)) : 0.f;
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
      if (direct) {
        if (my_row < n_valid) {
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            int4 v;
            uint32_t* vv = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              vv[e] = pack_bf16x2(__uint_as_float(o[8 * t + 2 * e]) * f, __uint_as_float(o[8 * t + 2 * e + 1]) * f);
            if (!(f > 0.f)) v = make_int4(0, 0, 0, 0);
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
    if (!direct && my_row < n_valid) reinterpret_cast<float2*>(s_ml)[my_row] = make_float2(m, l);
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, kTmemCols);
  }
  if (direct) return;

  // join the splits (and the launch before): this CTA takes every splits-th run of rows, 8 columns a thread
  cg::cluster_group cl = cg::this_cluster();
  if (splits > 1) cl.sync();
  if (p.part_mode == 2) px_wait_prior_grid();
  const int per = (n_valid + splits - 1) / splits;
  const int ra = rank * per, rb = min(n_valid, ra + per);
  for (int i = threadIdx.x; i < (rb - ra) * (D / 8); i += kThreads) {
    const int r = ra + i / (D / 8), c = i % (D / 8);
    const int rr = row0 + r, tok = rr / g, h = hk * g + rr - tok * g;
    const long long grow = static_cast<long long>(start + tok) * p.hq + h;
    float mm = -1e30f;
    for (int s = 0; s < splits; ++s) {
      const float2 ml = *reinterpret_cast<const float2*>(splits > 1 ? cl.map_shared_rank(s_ml + 2 * r, s) : s_ml + 2 * r);
      if (ml.y > 0.f) mm = fmaxf(mm, ml.x);
    }
    float2 pm = make_float2(0.f, 0.f);
    if (p.part_mode == 2) {
      pm = __ldcg(reinterpret_cast<const float2*>(p.part_ml) + grow);
      if (pm.y > 0.f) mm = fmaxf(mm, pm.x);
    }
    const float sk = p.part_mode == 1 ? -INFINITY : sink_of(h);
    const float top = fmaxf(mm, sk);
    float acc[8], sum = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = 0.f;
    auto add = [&](float4 a, float4 d, float w) {
      acc[0] += w * a.x; acc[1] += w * a.y; acc[2] += w * a.z; acc[3] += w * a.w;
      acc[4] += w * d.x; acc[5] += w * d.y; acc[6] += w * d.z; acc[7] += w * d.w;
    };
    for (int s = 0; s < splits; ++s) {
      const float* xr = sx + r * D;
      const float* mr = s_ml + 2 * r;
      if (splits > 1) { xr = cl.map_shared_rank(xr, s); mr = cl.map_shared_rank(mr, s); }
      const float2 ml = *reinterpret_cast<const float2*>(mr);
      if (!(ml.y > 0.f)) continue;
      const float w = px_exp2(ml.x - top);
      sum += w * ml.y;
      add(reinterpret_cast<const float4*>(xr)[(2 * c) ^ (r & 7)], reinterpret_cast<const float4*>(xr)[(2 * c + 1) ^ (r & 7)], w);
    }
    if (pm.y > 0.f) {
      const float w = px_exp2(pm.x - top);
      sum += w * pm.y;
      const float4* o = reinterpret_cast<const float4*>(p.part_o + grow * D) + 2 * c;
      add(__ldcg(o), __ldcg(o + 1), w);
    }
    if (p.part_mode == 1) {
      float4* o = reinterpret_cast<float4*>(p.part_o + grow * D) + 2 * c;
      o[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
      o[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
      if (c == 0) reinterpret_cast<float2*>(p.part_ml)[grow] = make_float2(top, sum);
    } else {
      const float f = sum > 0.f ? 1.f / (sum + px_exp2(sk - top)) : 0.f;
      int4 v;
      uint32_t* vv = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
      for (int e = 0; e < 4; ++e) vv[e] = pack_bf16x2(acc[2 * e] * f, acc[2 * e + 1] * f);
      *reinterpret_cast<int4*>(p.out + grow * D + c * 8) = v;
    }
  }
  if (splits > 1) cl.sync();                                     // nobody leaves while its rows may still be read
}

template <int D, int TILES>
static cudaError_t px_launch(const ExtendParams& p, int tiles, int z, cudaStream_t st) {
  auto kern = k_paged_extend<D, TILES>;
  // per device, so set at every launch (it only stores a number): a process may use several
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, PxSmem<D, TILES>::kBytes);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles) * p.splits, p.hkv, z);
  cfg.blockDim = dim3(PxSmem<D, TILES>::kThreads);
  cfg.dynamicSmemBytes = PxSmem<D, TILES>::kBytes;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  int n = 0;
  if (p.splits > 1) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n].val.clusterDim.x = p.splits; at[n].val.clusterDim.y = 1; at[n].val.clusterDim.z = 1;
    ++n;
  }
  if (p.part_mode == 2) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = at; cfg.numAttrs = n;
  e = cudaLaunchKernelEx(&cfg, kern, p);
  return e == cudaSuccess ? cudaGetLastError() : e;
}

// Tiles, splits and launch for `lists` row lists of up to `rows` rows each that see at most `keys` keys.
static int px_run(ExtendParams& p, int D, long long rows, int lists, long long keys, cudaStream_t st) {
  // two tiles a CTA halve the K/V traffic; one tile spreads few rows over more SMs
  const long long pairs = (rows + 2 * PX_BM - 1) / (2 * PX_BM);
  const bool two = rows > PX_BM && pairs * lists * p.hkv >= 148;
  const long long tiles = two ? pairs : (rows + PX_BM - 1) / PX_BM;
  if (tiles > (1 << 20)) return -5;
  // split the keys while SMs are free and every split keeps four blocks
  const long long room = (D == 64 && !two) ? 296 : 148;
  int splits = 1;
  while (splits < 8 && tiles * lists * p.hkv * splits * 2 <= room && keys >= static_cast<long long>(splits) * 2 * 4 * PX_BN) splits *= 2;
  p.splits = splits;
  cudaError_t e;
  if (D == 64) e = two ? px_launch<64, 2>(p, static_cast<int>(tiles), lists, st) : px_launch<64, 1>(p, static_cast<int>(tiles), lists, st);
  else e = two ? px_launch<128, 2>(p, static_cast<int>(tiles), lists, st) : px_launch<128, 1>(p, static_cast<int>(tiles), lists, st);
  return e == cudaSuccess ? 0 : static_cast<int>(e);
}

}  // namespace nmoe

using namespace nmoe;

// q [n_rows, Hq, D] (rows q_stride apart), out [n_rows, Hq, D]; caches [num_blocks, block_size, Hkv, D]; block_tables [B] rows
// of max_blocks entries, bt_stride apart; context_lens, q_starts, q_lens [B].  prefix_len < 0: extend.  Otherwise one token
// per sequence (q_starts, q_lens null) behind prefix_len common keys, with a workspace of n_rows * Hq * (D + 2) floats.
extern "C" int nmoe_paged_extend(const void* q, long long q_stride, const void* k_cache, const void* v_cache,
                                 const int* block_tables, long long bt_stride, const int* context_lens,
                                 const int* q_starts, const int* q_lens, const void* sinks, int sinks_fp32, void* out,
                                 int n_rows, int B, int Hq, int Hkv, int D, int block_size, int num_blocks, int max_blocks,
                                 int max_q_len, int window, float scale, int prefix_len, float* workspace, void* status,
                                 cudaStream_t st) {
  if (B == 0 || n_rows == 0 || max_q_len == 0) return 0;
  if (Hkv < 1 || Hkv > 65535 || Hq % Hkv != 0 || block_size < 1 || B < 0 || B > 65535 || !(scale > 0.f)) return -1;
  if (D != 64 && D != 128) return -2;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) |
       reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) % 16 != 0 || (n_rows > 1 && q_stride % 8 != 0)) return -3;
  if (static_cast<long long>(n_rows) * (Hq / Hkv) > 0x7fffffffll - 256) return -4;
  ExtendParams p;
  p.q = static_cast<const __nv_bfloat16*>(q); p.k_cache = static_cast<const __nv_bfloat16*>(k_cache);
  p.v_cache = static_cast<const __nv_bfloat16*>(v_cache); p.out = static_cast<__nv_bfloat16*>(out);
  p.block_tables = block_tables; p.context_lens = context_lens; p.q_starts = q_starts; p.q_lens = q_lens; p.sinks = sinks;
  p.status = static_cast<StatusRecord*>(status); p.q_stride = q_stride; p.bt_stride = bt_stride; p.n_rows = n_rows;
  p.n_seqs = B; p.hq = Hq; p.hkv = Hkv; p.group = Hq / Hkv; p.block_size = block_size; p.num_blocks = num_blocks;
  p.block_shift = -1;
  for (int s = 0; s < 31; ++s)
    if (block_size == 1 << s) p.block_shift = s;
  p.max_blocks = max_blocks; p.max_q_len = max_q_len; p.window = window; p.sinks_fp32 = sinks_fp32;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.part_o = workspace; p.part_ml = workspace ? workspace + static_cast<long long>(n_rows) * Hq * D : nullptr;
  p.key_begin = 0; p.key_end = 0x7fffffff; p.flat = 0; p.part_mode = 0;
  const long long capacity = static_cast<long long>(max_blocks) * block_size;
  long long keys = window > 0 && window + max_q_len < capacity ? window + max_q_len : capacity;
  if (prefix_len <= 0) return px_run(p, D, static_cast<long long>(max_q_len) * p.group, B, keys, st);
  if (workspace == nullptr || q_starts != nullptr || q_lens != nullptr) return -5;
  ExtendParams f = p;
  f.flat = 1; f.part_mode = 1; f.key_end = prefix_len;
  const int rc = px_run(f, D, static_cast<long long>(B) * p.group, 1, prefix_len, st);
  if (rc != 0) return rc;
  p.part_mode = 2; p.key_begin = prefix_len;
  keys = window > 0 && window < capacity - prefix_len ? window : capacity - prefix_len;
  return px_run(p, D, p.group, B, keys, st);
}
