// Rotary embedding and cache append in one pass over the fused q|k|v projection of a serving step:
//   q, k rows   (x1, x2) halves of a head -> conc * (x1 cos a - x2 sin a, x2 cos a + x1 sin a), a = position * inv_freq
//   k, v rows   -> cache slot of their token (slot < 0: padding, nothing is stored); also to dense tensors when asked for
//
// The pass is bound by memory (three flops an element): every input element is read once and every output
// written once, 16 bytes a thread and half-head, no rotated copy in between.  A block takes one token, or four
// where there are enough to fill the GPU, works out their D/2 angles once into shared memory and lets all heads use
// them.  16384 tokens of 64/8 heads of 64 with dense K and V: 60 us, 6.0 TB/s (65 with one token a block); one token or
// 128: 4.3 us, the latency of a launch and two dependent reads.
//
// Angles: position * inv_freq is formed in 64 bits and reduced to [-1/2, 1/2] turns there, so that far
// positions keep the accuracy of near ones (in 32 bits the product alone is off by position * 2^-24 radians);
// sine and cosine of the remainder and the rotation itself are fp32, rounded once to bf16.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common/ptx.cuh"

namespace nmoe {

constexpr int kRopeThreads = 256;
constexpr int kRopeTokens = 4;       // of a block, where that leaves a few blocks for every SM

struct RopeAppendParams {
  const __nv_bfloat16* qkv;          // [N, (Hq + 2 Hkv) * D], rows qkv_stride apart
  const void* positions;             // [N] int64 or int32
  const float* inv_freq;             // [D / 2]
  const int* slots;                  // [N], null = no cache
  __nv_bfloat16 *k_cache, *v_cache;  // [n_slots, Hkv * D]
  __nv_bfloat16 *q_out, *k_out, *v_out;   // [N, H, D]; k_out / v_out may be null
  StatusRecord* status;
  long long qkv_stride, n_slots;
  int n_tokens, hq, hkv, d, pos64, tokens_per_block;
  float conc;
};

__global__ void __launch_bounds__(kRopeThreads) k_rope_append(const RopeAppendParams p) {
  extern __shared__ float2 s_cs[];                       // [tokens_per_block][D / 2] (cos, sin) * conc
  const int half = p.d >> 1, heads = p.hq + 2 * p.hkv;
  const int t0 = blockIdx.x * p.tokens_per_block;
  const int n_tok = min(p.tokens_per_block, p.n_tokens - t0);
  for (int i = threadIdx.x; i < n_tok * half; i += kRopeThreads) {
    const int t = t0 + i / half, f = i % half;
    const double pos = p.pos64 ? static_cast<double>(static_cast<const long long*>(p.positions)[t])
                               : static_cast<double>(static_cast<const int*>(p.positions)[t]);
    const double turns = pos * static_cast<double>(p.inv_freq[f]) * 0.15915494309189533577;    // 1 / (2 pi)
    float sn, cs;
    sincospif(2.f * static_cast<float>(turns - rint(turns)), &sn, &cs);
    s_cs[i] = make_float2(cs * p.conc, sn * p.conc);
  }
  __syncthreads();
  // one unit = 8 dims of the first half of a head and the 8 that rotate with them
  const int per_head = p.d >> 4, per_tok = heads * per_head;
  for (int u = threadIdx.x; u < n_tok * per_tok; u += kRopeThreads) {
    const int lt = u / per_tok, r = u - lt * per_tok, h = r / per_head, c = (r - h * per_head) * 8;
    const int t = t0 + lt;
    const __nv_bfloat16* src = p.qkv + t * p.qkv_stride + static_cast<long long>(h) * p.d + c;
    int4 a = ld_nc_v4(src), b = ld_nc_v4(src + half);
    if (h < p.hq + p.hkv) {
      const float2* cs = s_cs + lt * half + c;
      int* ai = reinterpret_cast<int*>(&a);
      int* bi = reinterpret_cast<int*>(&b);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 x1 = unpack_bf16x2(ai[i]), x2 = unpack_bf16x2(bi[i]), e0 = cs[2 * i], e1 = cs[2 * i + 1];
        ai[i] = pack_bf16x2(x1.x * e0.x - x2.x * e0.y, x1.y * e1.x - x2.y * e1.y);
        bi[i] = pack_bf16x2(x2.x * e0.x + x1.x * e0.y, x2.y * e1.x + x1.y * e1.y);
      }
    }
    if (h < p.hq) {
      __nv_bfloat16* o = p.q_out + (static_cast<long long>(t) * p.hq + h) * p.d + c;
      *reinterpret_cast<int4*>(o) = a;
      *reinterpret_cast<int4*>(o + half) = b;
      continue;
    }
    const bool is_k = h < p.hq + p.hkv;
    const int col = (h - p.hq - (is_k ? 0 : p.hkv)) * p.d + c;
    const long long row = static_cast<long long>(p.hkv) * p.d;
    __nv_bfloat16* dense = is_k ? p.k_out : p.v_out;
    if (dense != nullptr) {
      *reinterpret_cast<int4*>(dense + t * row + col) = a;
      *reinterpret_cast<int4*>(dense + t * row + col + half) = b;
    }
    const int slot = p.slots != nullptr ? p.slots[t] : -1;
    if (slot < 0) continue;
    if (slot >= p.n_slots) { report_status(p.status, kStatusBadIndex, 1000, t, slot); continue; }
    __nv_bfloat16* cache = (is_k ? p.k_cache : p.v_cache) + slot * row + col;
    *reinterpret_cast<int4*>(cache) = a;
    *reinterpret_cast<int4*>(cache + half) = b;
  }
}

}  // namespace nmoe

using namespace nmoe;

// D a multiple of 16 up to 512; every pointer and row stride a multiple of 16 bytes.  slots / caches null: rotate only.
extern "C" int nmoe_rope_append(const void* qkv, long long qkv_stride, const void* positions, int pos64,
                                const float* inv_freq, float conc, const int* slots, void* k_cache, void* v_cache,
                                long long n_slots, void* q_out, void* k_out, void* v_out, int n_tokens, int hq, int hkv,
                                int d, void* status, cudaStream_t st) {
  if (n_tokens == 0) return 0;
  if (n_tokens < 0 || hq < 1 || hkv < 1 || d < 16 || d > 512 || d % 16 != 0 || qkv_stride % 8 != 0) return -1;
  if (slots != nullptr && (k_cache == nullptr || v_cache == nullptr)) return -2;
  uintptr_t bits = 0;
  for (const void* a : {qkv, static_cast<const void*>(k_cache), static_cast<const void*>(v_cache), static_cast<const void*>(q_out),
                        static_cast<const void*>(k_out), static_cast<const void*>(v_out)})
    bits |= reinterpret_cast<uintptr_t>(a);
  if (bits % 16 != 0) return -3;
  RopeAppendParams p;
  p.qkv = static_cast<const __nv_bfloat16*>(qkv); p.positions = positions; p.inv_freq = inv_freq; p.slots = slots;
  p.k_cache = static_cast<__nv_bfloat16*>(k_cache); p.v_cache = static_cast<__nv_bfloat16*>(v_cache);
  p.q_out = static_cast<__nv_bfloat16*>(q_out); p.k_out = static_cast<__nv_bfloat16*>(k_out);
  p.v_out = static_cast<__nv_bfloat16*>(v_out); p.status = static_cast<StatusRecord*>(status);
  p.qkv_stride = qkv_stride; p.n_slots = n_slots; p.n_tokens = n_tokens; p.hq = hq; p.hkv = hkv; p.d = d;
  p.pos64 = pos64; p.conc = conc;
  p.tokens_per_block = n_tokens >= 148 * 8 * 4 ? kRopeTokens : 1;
  k_rope_append<<<(n_tokens + p.tokens_per_block - 1) / p.tokens_per_block, kRopeThreads, p.tokens_per_block * (d / 2) * sizeof(float2), st>>>(p);
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : static_cast<int>(e);
}
