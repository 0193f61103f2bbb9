// Attention of several new tokens per sequence over the paged cache (drafted tokens of a decode step, the part of a
// prompt behind a cached prefix): token j of a sequence stands at position context - q_len + j and sees the keys at or
// before it, within the window, plus an optional learned sink logit per head that only enters the denominator.
//   out = sum_j softmax_j(scale * q . k_j | sink) * v_j
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common/ptx.cuh"

namespace nmoe {

struct ExtendParams {
  const __nv_bfloat16 *q, *k_cache, *v_cache;
  __nv_bfloat16* out;
  const int *block_tables, *context_lens, *q_starts, *q_lens;    // q_starts / q_lens null: one token per sequence
  const void* sinks;
  StatusRecord* status;
  long long q_stride, bt_stride;
  int n_rows, hq, hkv, block_size, num_blocks, max_blocks, max_q_len, window, sinks_fp32;
  float scale_log2;
};

// one warp per (token, query head), keys one after the other, D / 32 dims a lane
template <int D>
__global__ void __launch_bounds__(128) k_paged_extend_rows(const ExtendParams p) {
  constexpr int E = D / 32;
  const int b = blockIdx.z, j = blockIdx.x, h = blockIdx.y * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int start = p.q_starts ? p.q_starts[b] : b, n = p.q_lens ? p.q_lens[b] : 1;
  int ctx = p.context_lens[b];
  const bool first = j == 0 && blockIdx.y == 0 && threadIdx.x == 0;
  if (start < 0 || n < 0 || start > p.n_rows || n > p.n_rows - start || n > p.max_q_len) {
    if (first) report_status(p.status, kStatusBadIndex, 1020, b, start);
    return;
  }
  if (static_cast<long long>(ctx) > static_cast<long long>(p.max_blocks) * p.block_size) {
    if (first) report_status(p.status, kStatusBadIndex, 1021, b, ctx);
    ctx = p.max_blocks * p.block_size;
  }
  if (j >= n || h >= p.hq) return;
  const long long row = start + j;
  const int pos = ctx - n + j, hkv = h / (p.hq / p.hkv);
  float qf[E], acc[E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    qf[i] = __bfloat162float(p.q[row * p.q_stride + h * D + lane * E + i]);
    acc[i] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int t = p.window > 0 ? max(0, pos - p.window + 1) : 0; t <= pos; ++t) {
    const int page = p.block_tables[b * p.bt_stride + t / p.block_size];
    if (page < 0 || page >= p.num_blocks) {
      if (lane == 0) report_status(p.status, kStatusBadIndex, 1022, b, page);
      continue;
    }
    const long long at = ((static_cast<long long>(page) * p.block_size + t % p.block_size) * p.hkv + hkv) * D + lane * E;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) s += qf[i] * __bfloat162float(p.k_cache[at + i]);
    s = warp_sum(s) * p.scale_log2;
    const float mn = fmaxf(m, s), al = exp2f(m - mn), e = exp2f(s - mn);
    l = l * al + e;
#pragma unroll
    for (int i = 0; i < E; ++i) acc[i] = acc[i] * al + e * __bfloat162float(p.v_cache[at + i]);
    m = mn;
  }
  float den = l, f = 1.f;
  if (p.sinks != nullptr) {
    const float sk = 1.4426950408889634f * (p.sinks_fp32 ? static_cast<const float*>(p.sinks)[h]
                                                         : __bfloat162float(static_cast<const __nv_bfloat16*>(p.sinks)[h]));
    const float mn = fmaxf(m, sk);
    if (mn > -INFINITY) { f = exp2f(m - mn); den = l * f + exp2f(sk - mn); }
  }
  const float inv = l > 0.f ? f / den : 0.f;
#pragma unroll
  for (int i = 0; i < E; ++i) p.out[(row * p.hq + h) * D + lane * E + i] = __float2bfloat16(acc[i] * inv);
}

}  // namespace nmoe

using namespace nmoe;

extern "C" int nmoe_paged_extend(const void* q, long long q_stride, const void* k_cache, const void* v_cache,
                                 const int* block_tables, long long bt_stride, const int* context_lens,
                                 const int* q_starts, const int* q_lens, const void* sinks, int sinks_fp32, void* out,
                                 int n_rows, int B, int Hq, int Hkv, int D, int block_size, int num_blocks, int max_blocks,
                                 int max_q_len, int window, float scale, void* status, cudaStream_t st) {
  if (B == 0 || n_rows == 0 || max_q_len == 0) return 0;
  if (Hkv < 1 || Hq % Hkv != 0 || block_size < 1 || B > 65535) return -1;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) |
       reinterpret_cast<uintptr_t>(out)) % 16 != 0 || (n_rows > 1 && q_stride % 8 != 0)) return -3;
  ExtendParams p;
  p.q = static_cast<const __nv_bfloat16*>(q); p.k_cache = static_cast<const __nv_bfloat16*>(k_cache);
  p.v_cache = static_cast<const __nv_bfloat16*>(v_cache); p.out = static_cast<__nv_bfloat16*>(out);
  p.block_tables = block_tables; p.context_lens = context_lens; p.q_starts = q_starts; p.q_lens = q_lens; p.sinks = sinks;
  p.status = static_cast<StatusRecord*>(status); p.q_stride = q_stride; p.bt_stride = bt_stride; p.n_rows = n_rows;
  p.hq = Hq; p.hkv = Hkv; p.block_size = block_size; p.num_blocks = num_blocks; p.max_blocks = max_blocks;
  p.max_q_len = max_q_len; p.window = window; p.sinks_fp32 = sinks_fp32; p.scale_log2 = scale * 1.4426950408889634f;
  const dim3 grid(max_q_len, (Hq + 3) / 4, B);
  if (D == 64) k_paged_extend_rows<64><<<grid, 128, 0, st>>>(p);
  else if (D == 128) k_paged_extend_rows<128><<<grid, 128, 0, st>>>(p);
  else return -2;
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : static_cast<int>(e);
}
