// dcnv2_rotary_kernel.cuh — RMS norm of each query and key head and the rotation by its token's
// position, in one pass.
//
// For a head x of D elements: y = x * rsqrt(mean(x^2) + eps) * weight (norm on, else y = x); for
// rotated pair p with elements (e0, e1): out[e0] = y[e0] cos a - y[e1] sin a, out[e1] = y[e1] cos a
// + y[e0] sin a, a = position[axis of p] * freq[p]; the elements behind the rotated ones keep y.
//
// Work split: a head's D/2 pairs are cut into chunks of VEC pairs, one lane per chunk (two vector
// loads of VEC elements), a power of two of lanes per head, so the norm is a shuffle reduction and
// a warp reads whole heads side by side. The elements behind the rotated ones are taken as pairs
// too (first half, second half) with cos = 1, sin = 0. A block takes a few tokens; the cosines and
// sines of a token are computed once into shared memory and used by all of its heads, while the
// block's first loads are in flight.
//
// Angles: turns = position * (freq / 2 pi) in fp64, minus the nearest integer, then sincospif of
// the fraction. In fp32 the product alone would be off by position * freq * 2^-24 radians (0.006 at
// position 100000); the fp64 product keeps 2^-53 of it. Everything else is fp32, rounded once.
//
// Bound: HBM (every element read once and written once).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "ptx_sm100.cuh"

namespace dcnv2 {

constexpr int kRotThreads = 256;
constexpr int kRotBatch = 2;         // heads per lane group with loads in flight at once
constexpr int kRotMaxPairs = 128;    // head_dim <= 256

struct RotaryTensor {
  const void* in;
  void* out;
  const void* weight;                // [D] or null
  int64_t sb, st, sh;                // strides of in: batch, token, head (elements)
  int64_t ob, ot, oh;                // strides of out
};

struct RotaryArgs {
  RotaryTensor t[2];                 // queries, keys
  const int* pos;                    // [batch][tokens][axes]
  const float* freqs;                // [rot_pairs]
  int64_t pos_sb;                    // batch stride of pos (0: shared)
  int rows, tokens;                  // rows = batch * tokens
  int q_heads, heads;                // heads = q_heads + k_heads
  int D, pairs, rot_pairs, axes;     // pairs = D / 2
  int chunks;                        // lanes' work: pairs / VEC
  int group, group_shift;            // lanes per head
  int rows_per_block;
  int norm, interleaved;
  float eps, inv_d;
  uint32_t pair_axis[kRotMaxPairs / 16];  // 2 bits per rotated pair
};

template <typename T> __device__ __forceinline__ float rot_load(T v);
template <> __device__ __forceinline__ float rot_load(float v) { return v; }
template <> __device__ __forceinline__ float rot_load(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float rot_load(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <typename T> __device__ __forceinline__ T rot_round(float v);
template <> __device__ __forceinline__ float rot_round(float v) { return v; }
template <> __device__ __forceinline__ __half rot_round(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 rot_round(float v) {
  return __float2bfloat16_rn(v);
}

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) RotVec {
  T v[VEC];
};

// Element offsets of the two vectors of chunk c: the pairs' first and second elements, or, for
// interleaved pairs, the lower and upper half of 2 * VEC neighbouring elements. `behind`: the
// chunk's pairs lie behind the rotated ones.
template <int VEC>
__device__ __forceinline__ void rot_chunk(const RotaryArgs& a, int c, int& lo, int& hi,
                                          bool& behind) {
  const int p = c * VEC;
  behind = p >= a.rot_pairs;
  if (a.interleaved) {
    lo = 2 * p;
    hi = lo + VEC;
  } else if (!behind) {
    lo = p;
    hi = p + a.rot_pairs;
  } else {
    lo = p + a.rot_pairs;
    hi = lo + (a.pairs - a.rot_pairs);
  }
}

// VEC pairs per chunk; a lane takes up to NC chunks of a head.
template <typename T, int VEC, int NC>
__global__ void __launch_bounds__(kRotThreads)
    dcnv2_qk_norm_rotary_kernel(const __grid_constant__ RotaryArgs args) {
  using V = RotVec<T, VEC>;
  extern __shared__ float2 trig[];  // [rows_per_block][rot_pairs] (cos, sin)
  const int row0 = static_cast<int>(blockIdx.x) * args.rows_per_block;
  const int n_rows = min(args.rows_per_block, args.rows - row0);
  const int lane = static_cast<int>(threadIdx.x) & (args.group - 1);
  const int n_items = n_rows * args.heads;
  const int step = kRotThreads >> args.group_shift;

  ptx::griddep_launch_dependents();
  ptx::griddep_wait();

  V lo[kRotBatch][NC], hi[kRotBatch][NC];
  auto fetch = [&](int item0) {
#pragma unroll
    for (int u = 0; u < kRotBatch; ++u) {
      const int item = item0 + u * step;
      if (item >= n_items) break;
      const int r = item / args.heads, h = item - r * args.heads;
      const int row = row0 + r, b = row / args.tokens, t = row - b * args.tokens;
      const RotaryTensor& x = args.t[h >= args.q_heads];
      const T* p = static_cast<const T*>(x.in) + b * x.sb + t * x.st +
                   (h >= args.q_heads ? h - args.q_heads : h) * x.sh;
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        const int c = lane + n * args.group;
        if (c < args.chunks) {
          int el, eh;
          bool behind;
          rot_chunk<VEC>(args, c, el, eh, behind);
          lo[u][n] = *reinterpret_cast<const V*>(p + el);
          hi[u][n] = *reinterpret_cast<const V*>(p + eh);
        }
      }
    }
  };

  int item0 = static_cast<int>(threadIdx.x) >> args.group_shift;
  fetch(item0);

  for (int i = threadIdx.x; i < n_rows * args.rot_pairs; i += kRotThreads) {
    const int r = i / args.rot_pairs, p = i - r * args.rot_pairs;
    const int row = row0 + r, b = row / args.tokens, t = row - b * args.tokens;
    const int axis = (args.pair_axis[p >> 4] >> (2 * (p & 15))) & 3;
    const int pos = __ldg(args.pos + b * args.pos_sb + static_cast<int64_t>(t) * args.axes + axis);
    double turns = static_cast<double>(pos) *
                   (static_cast<double>(__ldg(args.freqs + p)) * 0.15915494309189533577);
    turns -= rint(turns);
    float s, c;
    sincospif(2.0f * static_cast<float>(turns), &s, &c);
    trig[i] = make_float2(c, s);
  }
  __syncthreads();

  // every lane of a warp takes the same number of turns, so that the shuffles see whole warps
  for (; __any_sync(0xffffffffu, item0 < n_items); item0 += kRotBatch * step) {
#pragma unroll
    for (int u = 0; u < kRotBatch; ++u) {
      const int item = item0 + u * step;
      const bool live = item < n_items;
      const int r = live ? item / args.heads : 0, h = live ? item - r * args.heads : 0;
      const RotaryTensor& x = args.t[h >= args.q_heads];
      float scale = 1.f;
      if (args.norm) {
        float sum = 0.f;
#pragma unroll
        for (int n = 0; n < NC; ++n)
          if (live && lane + n * args.group < args.chunks)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              const float a = rot_load<T>(lo[u][n].v[i]), b = rot_load<T>(hi[u][n].v[i]);
              sum = fmaf(a, a, fmaf(b, b, sum));
            }
        for (int m = args.group >> 1; m > 0; m >>= 1)
          sum += __shfl_xor_sync(0xffffffffu, sum, m);
        scale = rsqrtf(fmaf(sum, args.inv_d, args.eps));
      }
      if (!live) continue;
      const int row = row0 + r, b = row / args.tokens, t = row - b * args.tokens;
      T* o = static_cast<T*>(x.out) + b * x.ob + t * x.ot +
             (h >= args.q_heads ? h - args.q_heads : h) * x.oh;
      const T* w = static_cast<const T*>(x.weight);
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        const int c = lane + n * args.group;
        if (c >= args.chunks) continue;
        int el, eh;
        bool behind;
        rot_chunk<VEC>(args, c, el, eh, behind);
        float y[2 * VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          y[i] = rot_load<T>(lo[u][n].v[i]) * scale;
          y[VEC + i] = rot_load<T>(hi[u][n].v[i]) * scale;
        }
        if (w) {
          const V wl = *reinterpret_cast<const V*>(w + el), wh = *reinterpret_cast<const V*>(w + eh);
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            y[i] *= rot_load<T>(wl.v[i]);
            y[VEC + i] *= rot_load<T>(wh.v[i]);
          }
        }
        V ol, oh;
        if (!behind) {
          const float2* cs = trig + r * args.rot_pairs + c * VEC;
          float z[2 * VEC];
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const float2 g = cs[i];
            // pair i of the chunk: (i, VEC + i), or (2 i, 2 i + 1) of the 2 VEC neighbours
            const float e0 = args.interleaved ? y[2 * i] : y[i];
            const float e1 = args.interleaved ? y[2 * i + 1] : y[VEC + i];
            const float f0 = fmaf(e0, g.x, -e1 * g.y), f1 = fmaf(e1, g.x, e0 * g.y);
            if (args.interleaved) { z[2 * i] = f0; z[2 * i + 1] = f1; }
            else { z[i] = f0; z[VEC + i] = f1; }
          }
#pragma unroll
          for (int i = 0; i < 2 * VEC; ++i) y[i] = z[i];
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          ol.v[i] = rot_round<T>(y[i]);
          oh.v[i] = rot_round<T>(y[VEC + i]);
        }
        *reinterpret_cast<V*>(o + el) = ol;
        *reinterpret_cast<V*>(o + eh) = oh;
      }
    }
    fetch(item0 + kRotBatch * step);
  }
}

}  // namespace dcnv2
