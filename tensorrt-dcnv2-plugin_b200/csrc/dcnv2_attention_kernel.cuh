// dcnv2_attention_kernel.cuh — attention of queries to the states of another sequence.
//
// For query row i of a sequence and its kept states j: s_ij = scale q_i k_j, m = max s, p = exp(s -
// m), out_i = sum p v / sum p, lse_i = m + log sum p; without kept states out = 0, lse = -inf.
//
// One warp per query row: a lane takes every 32nd state of a pass of 32, the running maximum and sum
// are warp-wide, the products with v are accumulated 4 elements per lane.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "dcnv2_wait.cuh"
#include "ptx_sm100.cuh"

namespace dcnv2 {

struct AttnTensor {
  const void* p;
  int64_t sb, st, sh;
};

struct AttnArgs {
  AttnTensor q, k, v, o;
  const int* kv_lens;
  const uint8_t* key_mask;
  int64_t mask_sb;
  float* lse;
  int* err;
  int B, L, S, H, G, D;
  float scale;
};

constexpr int kAttnWarps = 8;

__device__ __forceinline__ float attn_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float attn_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void attn_round(float v, __half& o) { o = __float2half_rn(v); }
__device__ __forceinline__ void attn_round(float v, __nv_bfloat16& o) { o = __float2bfloat16_rn(v); }

template <typename T>
__global__ void __launch_bounds__(kAttnWarps * 32)
    dcnv2_cross_attention_kernel(const __grid_constant__ AttnArgs a) {
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) a.err[blockIdx.x] = 0;
  const int64_t row = int64_t(blockIdx.x) * kAttnWarps + (threadIdx.x >> 5);
  if (row >= int64_t(a.B) * a.L * a.H) return;
  const int h = row % a.H, t = (row / a.H) % a.L, b = row / (int64_t(a.H) * a.L);
  const int g = h / (a.H / a.G);
  const T* q = static_cast<const T*>(a.q.p) + b * a.q.sb + t * a.q.st + h * a.q.sh;
  const T* k = static_cast<const T*>(a.k.p) + b * a.k.sb + g * a.k.sh;
  const T* v = static_cast<const T*>(a.v.p) + b * a.v.sb + g * a.v.sh;
  int n = a.S;
  if (a.kv_lens) n = max(0, min(a.S, a.kv_lens[b]));
  float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int j0 = 0; j0 < n; j0 += 32) {
    const int j = j0 + lane;
    const bool keep = j < n && (!a.key_mask || a.key_mask[b * a.mask_sb + j]);
    float s = -INFINITY;
    if (keep) {
      s = 0.f;
      for (int d = 0; d < a.D; ++d) s = fmaf(attn_f(q[d]), attn_f(k[j * a.k.st + d]), s);
      s *= a.scale;
    }
    float top = s;
    for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    const float mn = fmaxf(m, top), ref = mn == -INFINITY ? 0.f : mn;
    const float f = expf(m - ref), p = keep ? expf(s - ref) : 0.f;
    float sum = p;
    for (int x = 16; x; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    l = l * f + sum;
    m = mn;
    T pr;
    attn_round(p, pr);
    for (int e = 0; e < 4; ++e) acc[e] *= f;
    for (int x = 0; x < 32; ++x) {
      const float px = __shfl_sync(0xffffffffu, attn_f(pr), x);
      if (!__shfl_sync(0xffffffffu, keep, x)) continue;
      for (int e = 0; e < 4; ++e)
        if (lane + 32 * e < a.D)
          acc[e] = fmaf(px, attn_f(v[(j0 + x) * a.v.st + lane + 32 * e]), acc[e]);
    }
  }
  T* o = static_cast<T*>(const_cast<void*>(a.o.p)) + b * a.o.sb + t * a.o.st + h * a.o.sh;
  for (int e = 0; e < 4; ++e)
    if (lane + 32 * e < a.D) attn_round(l != 0.f ? acc[e] / l : 0.f, o[lane + 32 * e]);
  if (a.lse && lane == 0)
    a.lse[(int64_t(b) * a.H + h) * a.L + t] = m == -INFINITY ? -INFINITY : m + logf(l);
}

}  // namespace dcnv2
