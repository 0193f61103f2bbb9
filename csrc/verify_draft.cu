// Verification of drafted tokens against the target's probabilities, from given random numbers, so that what comes
// out is distributed as if every token had been drawn from the target:
//   drafted token x of row i passes while u_i * q_i(x) < p_{i-1}(x);
//   at the first that fails, one token is drawn from max(p - q, 0) of that position (q = 1 at x for a looked-up token);
//   if all pass, one more is drawn from the last target row.  A sequence without drafted tokens is plain sampling.
// The draw is the first index whose running sum passes u * total.
//
// Products of two fp32 numbers are exact in 64 bits, and the sums are 64-bit too, so the chosen index does not depend
// on how a row is split except where u * total falls within 1e-15 of a border.
//
// One row of V probabilities per sequence (two with a draft distribution) is all that has to be read: bandwidth for
// many sequences, latency for one.  A cluster of CTAs shares a row, each warp owns a contiguous stretch that it reads in
// batches of 512 entries (loads of a batch issued together: entry by entry the loop waited for memory 25 times a
// stretch) and keeps the sum of every step of them; the CTAs' sums meet through distributed shared memory, and the warp
// whose stretch holds the crossing walks one step of it once more from the L2.
// No workspace, no atomics on global memory, the same result for every run.
// 64 sequences, vocabulary 201088, draft distribution: 30 us, 2.4 TB/s (sums 17 us: 64-bit conversions and adds; 13 us of
// dependent reads: lengths, tokens, probabilities, and the crossing).  One sequence: 12.5 us, those latencies alone.
#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common/ptx.cuh"

namespace cg = cooperative_groups;

namespace nmoe {

constexpr int kVerifyThreads = 512;
constexpr int kVerifyWarps = kVerifyThreads / 32;
constexpr int kVerifyMaxCluster = 16;
constexpr int kVerifyBatch = 4;         // groups of 128 entries that a warp reads at once
constexpr int kVerifySteps = 32;        // sums that a warp keeps of its stretch

struct VerifyParams {
  const float* target;        // [N, V], rows target_stride apart
  const float* draft;         // [N, V] or null: row r = what the token at row r was drawn from
  const void* tokens;         // [N] int64 or int32; row q_starts[b] is the last known token, the drafted ones follow
  const float* uniforms;      // [N]
  const int *q_starts, *q_lens;   // [B]
  int* out;                   // [N]: emitted tokens at q_starts[b].., -1 behind them
  int* n_out;                 // [B]
  StatusRecord* status;
  long long target_stride, draft_stride;
  int n_rows, vocab, tok64, vec;
};

NMOE_DEVICE long long verify_token(const VerifyParams& p, int row) {
  return p.tok64 ? static_cast<const long long*>(p.tokens)[row] : static_cast<const int*>(p.tokens)[row];
}
NMOE_DEVICE double verify_warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// weight of one vocabulary entry in the draw
NMOE_DEVICE double verify_weight(float pv, float qv) {
  const double d = static_cast<double>(pv) - static_cast<double>(qv);
  return d > 0.0 ? d : 0.0;
}

__global__ void __launch_bounds__(kVerifyThreads, 2) k_verify_draft(const VerifyParams p) {
  cg::cluster_group cl = cg::this_cluster();
  const int n_cta = cl.num_blocks(), rank = cl.block_rank();
  const int b = blockIdx.x / n_cta;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __shared__ int s_first;
  __shared__ double s_warp[kVerifyWarps], s_step[kVerifyWarps][kVerifySteps];
  __shared__ double s_all[2][kVerifyMaxCluster];        // every CTA's sum, written by the CTAs themselves; one row per attempt
  const int start = p.q_starts[b], n = p.q_lens[b];
  const bool fits = start >= 0 && n >= 0 && start <= p.n_rows && n <= p.n_rows - start;
  if (!fits && rank == 0 && threadIdx.x == 0) report_status(p.status, kStatusBadIndex, 1010, b, start);
  if (!fits || n == 0) {                                // the whole cluster leaves together
    if (rank == 0 && threadIdx.x == 0) p.n_out[b] = 0;
    return;
  }
  cl.barrier_arrive();                                  // waited for below, before anything is written to another CTA
  // how many drafted tokens pass: every CTA of the cluster works it out for itself
  if (threadIdx.x == 0) s_first = n;
  __syncthreads();
  for (int i = 1 + threadIdx.x; i < n; i += kVerifyThreads) {
    const long long x = verify_token(p, start + i);
    bool pass = false;
    if (x >= 0 && x < p.vocab) {
      const double pv = p.target[(start + i - 1) * p.target_stride + x];
      const double qv = p.draft != nullptr ? static_cast<double>(p.draft[(start + i) * p.draft_stride + x]) : 1.0;
      pass = static_cast<double>(p.uniforms[start + i]) * qv < pv;
    } else {
      report_status(p.status, kStatusBadIndex, 1011, start + i, static_cast<int>(x));
    }
    if (!pass) { atomicMin(&s_first, i); break; }
  }
  __syncthreads();
  const int first = s_first;                            // == n when all pass
  const int row = start + first - 1;
  bool cut = first < n;
  const float* tp = p.target + row * p.target_stride;
  const float* dp = nullptr;
  long long hole = -1;                                  // the looked-up token that failed: its weight is max(p - 1, 0) = 0
  if (cut) {
    if (p.draft != nullptr) dp = p.draft + (row + 1) * p.draft_stride;
    else hole = verify_token(p, row + 1);
  }
  // this warp's stretch of the vocabulary, in whole groups of 4
  const int groups = (p.vocab + 3) >> 2, n_warps = n_cta * kVerifyWarps;
  const int per = (groups + n_warps - 1) / n_warps, w = rank * kVerifyWarps + warp;
  const int v0 = min(p.vocab, w * per * 4), v1 = min(p.vocab, (w + 1) * per * 4);
  auto read4 = [&](const float* src, int v, float (&o)[4]) {            // entries v .. v+3, 0 past the end of the stretch
    if (p.vec && v + 4 <= v1) {
      const float4 f = *reinterpret_cast<const float4*>(src + v);
      o[0] = f.x; o[1] = f.y; o[2] = f.z; o[3] = f.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = v + i < v1 ? src[v + i] : 0.f;
    }
  };
  auto weights = [&](int v, const float (&pv)[4], const float (&qv)[4], double (&o)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = v + i == hole ? 0.0 : verify_weight(pv[i], qv[i]);
  };
  constexpr int kBatch = kVerifyBatch * 128;
  const int batches = (per * 4 + kBatch - 1) / kBatch, per_step = (batches + kVerifySteps - 1) / kVerifySteps * kBatch;   // entries
  double total = 0.0;
  int attempt = 0;
  cl.barrier_wait();
  for (;; ++attempt) {
    double sum = 0.0;
    for (int v = v0, step = 0; v < v1; v += per_step, ++step) {
      double mine = 0.0;
      for (int w = v; w < min(v1, v + per_step); w += kBatch) {
        float pv[kVerifyBatch][4], qv[kVerifyBatch][4];
#pragma unroll
        for (int u = 0; u < kVerifyBatch; ++u) read4(tp, w + u * 128 + lane * 4, pv[u]);
        if (dp != nullptr) {
#pragma unroll
          for (int u = 0; u < kVerifyBatch; ++u) read4(dp, w + u * 128 + lane * 4, qv[u]);
        } else {
#pragma unroll
          for (int u = 0; u < kVerifyBatch; ++u) qv[u][0] = qv[u][1] = qv[u][2] = qv[u][3] = 0.f;
        }
#pragma unroll
        for (int u = 0; u < kVerifyBatch; ++u) {
          double o[4];
          weights(w + u * 128 + lane * 4, pv[u], qv[u], o);
          mine += (o[0] + o[1]) + (o[2] + o[3]);
        }
      }
      mine = verify_warp_sum(mine);
      if (lane == 0) s_step[warp][step] = mine;
      sum += mine;
    }
    if (lane == 0) s_warp[warp] = sum;
    __syncthreads();
    if (threadIdx.x < n_cta) {
      double c = 0.0;
      for (int i = 0; i < kVerifyWarps; ++i) c += s_warp[i];
      *cl.map_shared_rank(&s_all[attempt][rank], threadIdx.x) = c;
    }
    cl.sync();
    total = 0.0;
    for (int i = 0; i < n_cta; ++i) total += s_all[attempt][i];
    // nothing left of the difference (the two distributions agree to the last bit): draw from the target itself
    if (!cut || total > 0.0 || attempt == 1) break;
    cut = false; dp = nullptr; hole = -1;
  }
  // the stretch that holds the crossing: the first whose running sum passes u * total, else the last with any weight
  const double goal = static_cast<double>(p.uniforms[start]) * total;
  double before = 0.0, base = 0.0;
  int pick = -1;
  for (int i = 0; i < n_cta; ++i) {
    const double s = s_all[attempt][i];
    if (s > 0.0) { pick = i; base = before; if (before + s > goal) break; }
    before += s;
  }
  if (pick == rank || (pick < 0 && rank == 0)) {
    int pw = -1;
    double run = pick < 0 ? 0.0 : base, wbase = run;
    for (int i = 0; i < kVerifyWarps; ++i) {
      const double s = s_warp[i];
      if (s > 0.0) { pw = i; wbase = run; if (run + s > goal) break; }
      run += s;
    }
    if (pw == warp) {
      __syncwarp();                                     // the step sums of lane 0
      int at_step = 0;
      double run2 = wbase;
      for (int i = 0; v0 + i * per_step < v1; ++i) {
        const double s = s_step[warp][i];
        if (s > 0.0) { at_step = i; wbase = run2; if (run2 + s > goal) break; }
        run2 += s;
      }
      int found = -1, last = -1;
      const int e0 = v0 + at_step * per_step, e1 = min(v1, e0 + per_step);
      for (int v = e0; v < e1 && found < 0; v += kBatch) {
        float pv[kVerifyBatch][4], qv[kVerifyBatch][4];
#pragma unroll
        for (int u = 0; u < kVerifyBatch; ++u) {
          read4(tp, v + u * 128 + lane * 4, pv[u]);
          if (dp != nullptr) read4(dp, v + u * 128 + lane * 4, qv[u]);
          else qv[u][0] = qv[u][1] = qv[u][2] = qv[u][3] = 0.f;
        }
#pragma unroll
        for (int u = 0; u < kVerifyBatch; ++u) {
          if (found >= 0) break;
          const int at = v + u * 128 + lane * 4;
          double o[4];
          weights(at, pv[u], qv[u], o);
          const double mine = (o[0] + o[1]) + (o[2] + o[3]);
          double inc = mine;
#pragma unroll
          for (int k = 1; k < 32; k <<= 1) {
            const double up = __shfl_up_sync(0xffffffffu, inc, k);
            if (lane >= k) inc += up;
          }
          double c = wbase + (inc - mine);
          int hit = -1, tail = -1;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            c += o[i];
            if (o[i] > 0.0) tail = at + i;
            if (hit < 0 && o[i] > 0.0 && c > goal) hit = at + i;
          }
          const unsigned who = __ballot_sync(0xffffffffu, hit >= 0);
          if (who) found = __shfl_sync(0xffffffffu, hit, __ffs(who) - 1);
          const unsigned any = __ballot_sync(0xffffffffu, tail >= 0);
          if (any) last = __shfl_sync(0xffffffffu, tail, 31 - __clz(any));
          wbase += __shfl_sync(0xffffffffu, inc, 31);
        }
      }
      if (lane == 0) p.out[row] = found >= 0 ? found : last;
    } else if (pw < 0 && warp == 0 && lane == 0) {
      p.out[row] = p.vocab - 1;                         // a target row without a positive entry
    }
  }
  if (rank == 0) {
    if (threadIdx.x == 0) p.n_out[b] = first;
    for (int i = threadIdx.x; i < n; i += kVerifyThreads)
      if (i != first - 1) p.out[start + i] = i < first - 1 ? static_cast<int>(verify_token(p, start + i + 1)) : -1;
  }
  cl.sync();                                            // nobody leaves while its sums may still be read
}

}  // namespace nmoe

using namespace nmoe;

extern "C" int nmoe_verify_draft(const float* target, long long target_stride, const float* draft, long long draft_stride,
                                 const void* tokens, int tok64, const float* uniforms, const int* q_starts,
                                 const int* q_lens, int* out, int* n_out, int n_rows, int n_seqs, int vocab, void* status,
                                 cudaStream_t st) {
  if (n_seqs == 0) return 0;
  if (n_seqs < 0 || n_rows < 0 || vocab < 1 || vocab > 1 << 30) return -1;     // indices of a stretch stay within 32 bits
  VerifyParams p;
  p.target = target; p.draft = draft; p.tokens = tokens; p.uniforms = uniforms; p.q_starts = q_starts; p.q_lens = q_lens;
  p.out = out; p.n_out = n_out; p.status = static_cast<StatusRecord*>(status);
  p.target_stride = target_stride; p.draft_stride = draft_stride; p.n_rows = n_rows; p.vocab = vocab; p.tok64 = tok64;
  p.vec = (reinterpret_cast<uintptr_t>(target) | reinterpret_cast<uintptr_t>(draft)) % 16 == 0 &&
          (target_stride | draft_stride) % 4 == 0;
  // As many CTAs a row as keep the batch within two an SM: one sequence 12.4 us with 16 of them, 14.4 with 8, 18.5 with 4, 43 with
  // one; 64 sequences 30 us with 4, 38 with 8, 54 with one.
  int cluster = 1;
  while (cluster < kVerifyMaxCluster && n_seqs * cluster * 2 <= 296 && vocab >= cluster * 2 * 4096) cluster *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(n_seqs) * cluster);
  cfg.blockDim = dim3(kVerifyThreads);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cluster; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
  cfg.attrs = at; cfg.numAttrs = 1;
  cudaError_t e = cudaSuccess;
  if (cluster > 8) e = cudaFuncSetAttribute(k_verify_draft, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, k_verify_draft, p);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? 0 : static_cast<int>(e);
}
