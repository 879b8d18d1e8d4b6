// dcnv2_rotary_kernel.cuh — RMS norm of each query and key head and the rotation by its token's
// position, in one pass.
//
// For a head x of D elements: y = x * rsqrt(mean(x^2) + eps) * weight (norm on, else y = x); for
// rotated pair p with elements (e0, e1): out[e0] = y[e0] cos a - y[e1] sin a, out[e1] = y[e1] cos a
// + y[e0] sin a, a = position[axis of p] * freq[p]; the elements behind the rotated ones keep y.
//
// Work split: a head's D/2 pairs are cut into chunks of VEC pairs, one lane per chunk (two vector
// loads of VEC elements), a power of two of lanes per head, so the norm is a shuffle reduction. The
// elements behind the rotated ones are taken as pairs too (first half, second half) with cos = 1,
// sin = 0. A team of lanes (a warp, or a power of two of its lanes when a token has few heads)
// takes a token's heads, kRotHeads per lane and step; its lanes compute the token's cosines and
// sines between them, once for all heads, into shared memory. Every team takes an equal run of
// neighbouring tokens (or, with few tokens, a part of a token's heads) and loads a step ahead.
//
// Angles: turns = position * freq / 2 pi modulo 1 in 64-bit fixed point (the product of the
// position and the fraction freq / 2 pi * 2^64 wraps around whole turns by itself), of which the
// upper 32 bits are the angle. In fp32 the product alone would be off by position * freq * 2^-24
// radians (0.006 at position 100000), in fp64 by position * freq * 2^-53 and more (2^-22 at
// position 2^31 and freq 1). Here freq / 2 pi is taken in two doubles, so that its fraction is
// right to 2^-64 turns (and freq * 2^-107): the error is position times that, at most about 2^-33
// turns for freq below 2^42, and 2^-26 turns of rounding the angle to fp32. fp32 tensors take sincospif
// of it, 16-bit ones the hardware's sine and cosine (absolute error at most 2^-21.1 on [-pi, pi],
// beside the half step of 2^-9 or 2^-12 of the output). Everything else is fp32, rounded once.
//
// Bound: latency, at 16 warps per SM with one step of loads in registers; neither HBM nor a pipe is
// full. Four heads of 128 cost a warp 293 instructions (unpacking, norm, gains, rotation, packing,
// and their share of addresses and cosines), which fill 58 % of the issue slots. Measured: 128 x
// 128 maps of 40 heads of 128, batch 4: 293 us, 4.6 TB/s, 71 % of the copy rate; keys of 5456
// tokens, 8 heads of 32, batch 32: 45 us, 4.0 TB/s; heads of 80 leave 3 of 8 lanes idle: 46 us, 3.2
// TB/s. One to four heads per lane and 8 to 32 warps per SM were measured; two and 16 are fastest.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <climits>
#include <type_traits>

#include "ptx_sm100.cuh"

namespace dcnv2 {

constexpr int kRotWarps = 8;
constexpr int kRotThreads = kRotWarps * 32;
constexpr int kRotResident = 16;     // warps per SM that the registers allow
constexpr int kRotHeads = 2;         // heads of a lane in work at once
constexpr int kRotLane = 16;         // cosines and sines in shared memory per lane of a team
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
  int heads[2];
  int side_shift[2];                 // log2 of the heads side by side in a team
  int steps[2];                      // steps of a unit (the heads a team takes of one token)
  int parts[2];                      // units of a token
  int units[2];                      // blocks of neighbouring units that a warp takes at once
  const int* pos;                    // [batch][tokens][axes]
  const float* freqs;                // [rot_pairs]
  int64_t pos_sb;                    // batch stride of pos (0: shared)
  int rows, tokens;                  // rows = batch * tokens
  int pairs, rot_pairs, axes;        // pairs = D / 2
  int chunks;                        // lanes' work: pairs / VEC
  int group_shift;                   // log2 of the lanes per head
  int norm;
  float eps, inv_d;
  uint32_t pair_axis[kRotMaxPairs / 16];  // 2 bits per rotated pair
};

__device__ __forceinline__ float rot_load(float v) { return v; }
__device__ __forceinline__ float rot_load(__half v) { return __half2float(v); }
__device__ __forceinline__ float rot_load(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void rot_round(float x, float& o) { o = x; }
__device__ __forceinline__ void rot_round(float x, __half& o) { o = __float2half_rn(x); }
__device__ __forceinline__ void rot_round(float x, __nv_bfloat16& o) { o = __float2bfloat16_rn(x); }

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) RotVec {
  T v[VEC];
};

// A vector's fp32 values, and back with one rounding.
template <typename T, int VEC>
__device__ __forceinline__ void rot_unpack(const RotVec<T, VEC>& v, float (&f)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) f[i] = rot_load(v.v[i]);
}
template <int VEC>
__device__ __forceinline__ void rot_unpack(const RotVec<__nv_bfloat16, VEC>& v, float (&f)[VEC]) {
  if constexpr (VEC % 2 == 0) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&v);
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = rot_load(v.v[i]);
  }
}
template <int VEC>
__device__ __forceinline__ void rot_unpack(const RotVec<__half, VEC>& v, float (&f)[VEC]) {
  if constexpr (VEC % 2 == 0) {
    const __half2* w = reinterpret_cast<const __half2*>(&v);
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
      const float2 x = __half22float2(w[i]);
      f[2 * i] = x.x;
      f[2 * i + 1] = x.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = rot_load(v.v[i]);
  }
}
template <typename T, int VEC>
__device__ __forceinline__ RotVec<T, VEC> rot_pack(const float (&f)[VEC]) {
  RotVec<T, VEC> v;
  if constexpr (sizeof(T) == 2 && VEC % 2 == 0) {
    uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i)
      w[i] = ptx::pack16<std::is_same<T, __nv_bfloat16>::value>(f[2 * i], f[2 * i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) rot_round(f[i], v.v[i]);
  }
  return v;
}
// VEC cosines or sines from shared memory.
template <int VEC>
__device__ __forceinline__ void rot_trig(const float* p, float (&f)[VEC]) {
  if constexpr (VEC % 4 == 0) {
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) {
      const float4 q = reinterpret_cast<const float4*>(p)[i];
      f[4 * i] = q.x; f[4 * i + 1] = q.y; f[4 * i + 2] = q.z; f[4 * i + 3] = q.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = p[i];
  }
}

// Element offsets of the two vectors of chunk c: the pairs' first and second elements, or, for
// interleaved pairs, the lower and upper half of 2 * VEC neighbouring elements. `behind`: the
// chunk's pairs lie behind the rotated ones.
template <int VEC, bool INTER>
__device__ __forceinline__ void rot_chunk(const RotaryArgs& a, int c, int& lo, int& hi,
                                          bool& behind) {
  const int p = c * VEC;
  behind = p >= a.rot_pairs;
  if (INTER) {
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

// VEC pairs per chunk; a lane takes up to NC chunks of a head; INTER: interleaved pairs.
template <typename T, int VEC, int NC, bool INTER>
__global__ void __launch_bounds__(kRotThreads, kRotResident / kRotWarps)
    dcnv2_qk_norm_rotary_kernel(const __grid_constant__ RotaryArgs args) {
  using V = RotVec<T, VEC>;
  constexpr int U = kRotHeads;
  extern __shared__ __align__(16) uint8_t rot_smem[];
  // turns per position of each pair, modulo 1, times 2^64 | the pairs' axes | per lane of a warp's
  // team: cosines, sines
  uint64_t* turn_table = reinterpret_cast<uint64_t*>(rot_smem);
  int* axis_table = reinterpret_cast<int*>(turn_table + kRotMaxPairs);
  float* trig = reinterpret_cast<float*>(axis_table + kRotMaxPairs);
  const int warp = static_cast<int>(threadIdx.x) >> 5, lane = static_cast<int>(threadIdx.x) & 31;
  const int group = 1 << args.group_shift;
  const int sub = lane & (group - 1);  // lane of the head

  int el[NC], eh[NC];
  bool used[NC], behind[NC];
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    const int c = sub + n * group;
    used[n] = c < args.chunks;
    rot_chunk<VEC, INTER>(args, used[n] ? c : 0, el[n], eh[n], behind[n]);
  }

  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  for (int p = threadIdx.x; p < args.rot_pairs; p += kRotThreads) {
    // 1 / 2 pi in two doubles; each part's whole turns are left out before it is scaled
    constexpr double kTurnHi = 0x1.45f306dc9c883p-3, kTurnLo = -0x1.6b01ec5417056p-57;
    const double f = __ldg(args.freqs + p);
    double hi = f * kTurnHi, lo = fma(f, kTurnLo, fma(f, kTurnHi, -hi));
    hi -= rint(hi);
    lo -= rint(lo);
    turn_table[p] = static_cast<uint64_t>(__double2ll_rn(hi * 0x1p64)) +
                    static_cast<uint64_t>(__double2ll_rn(lo * 0x1p64));
    axis_table[p] = (args.pair_axis[p >> 4] >> (2 * (p & 15))) & 3;
  }
  __syncthreads();

#pragma unroll 1
  for (int which = 0; which < 2; ++which) {
    // this warp's run of unit blocks of the tensor
    const int n_warps = static_cast<int>(gridDim.x) * kRotWarps;
    const int me = static_cast<int>(blockIdx.x) * kRotWarps + warp;
    // (the keys are dealt from the last warp on, so that few units of both go to different warps)
    const int turn = which ? n_warps - 1 - me : me;
    const int64_t n_units = args.units[which];
    int unit = static_cast<int>(n_units * turn / n_warps);
    const int unit_end = static_cast<int>(n_units * (turn + 1) / n_warps);
    if (unit >= unit_end) continue;
    const RotaryTensor x = args.t[which];
    const int heads = args.heads[which], steps = args.steps[which], parts = args.parts[which];
    const int sshift = args.side_shift[which];
    const int side = lane >> args.group_shift & ((1 << sshift) - 1);
    const int64_t in_head = x.sh << sshift, out_head = x.oh << sshift;  // from one of a lane's heads
                                                                        // to the next
    const int team_shift = args.group_shift + sshift;
    const int team = lane >> team_shift, team_lanes = 1 << team_shift;
    float* cosines = trig + (warp * 32 + (lane & ~(team_lanes - 1))) * kRotLane;
    const int stride = team_lanes * kRotLane / 2;  // from the cosines to the sines

    // a unit block is one unit per team: neighbouring rows, the same part of the heads
    int part, row, b, t;
    {
      const int block = unit / parts;
      part = unit - block * parts;
      row = block * (32 >> team_shift) + team;
      b = row / args.tokens;
      t = row - b * args.tokens;
    }
    const int n_steps = (unit_end - unit) * steps;
    auto next_unit = [&](int& r, int& bb, int& tt, int& pp) {
      if (++pp < parts) return;
      pp = 0;
      r += 32 >> team_shift;
      tt += 32 >> team_shift;
      while (tt >= args.tokens) {
        tt -= args.tokens;
        ++bb;
      }
    };
    // the lane's first head of a unit; beyond the last row none is live
    auto first_head = [&](int r, int pp) {
      return r < args.rows ? ((pp * steps * U) << sshift) + side : INT_MAX / 2;
    };
    V lo[U][NC], hi[U][NC];
    int step = 0;  // of the unit that is loaded next
    int row_in = row, b_in = b, t_in = t, part_in = part, head_in = first_head(row, part);
    const T* src = static_cast<const T*>(x.in) + b * x.sb + t * x.st + head_in * x.sh;
    auto fetch = [&](V (&l)[U][NC], V (&h)[U][NC]) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (head_in < heads) {
#pragma unroll
          for (int n = 0; n < NC; ++n)
            if (used[n]) {
              l[u][n] = *reinterpret_cast<const V*>(src + el[n]);
              h[u][n] = *reinterpret_cast<const V*>(src + eh[n]);
            }
        }
        head_in += 1 << sshift;
        src += in_head;
      }
      if (++step == steps) {
        step = 0;
        next_unit(row_in, b_in, t_in, part_in);
        head_in = first_head(row_in, part_in);
        src = static_cast<const T*>(x.in) + b_in * x.sb + t_in * x.st + head_in * x.sh;
      }
    };
    fetch(lo, hi);

    float gl[NC][VEC], gh[NC][VEC];  // gains of the norm
#pragma unroll
    for (int n = 0; n < NC; ++n) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) gl[n][i] = gh[n][i] = 1.f;
      const T* w = static_cast<const T*>(x.weight);
      if (w && used[n]) {
        rot_unpack(*reinterpret_cast<const V*>(w + el[n]), gl[n]);
        rot_unpack(*reinterpret_cast<const V*>(w + eh[n]), gh[n]);
      }
    }

    int at = 0;  // step of the unit in work
    int head = first_head(row, part);
    T* dst = static_cast<T*>(x.out) + b * x.ob + t * x.ot + head * x.oh;
#pragma unroll 1
    for (int s = 0; s < n_steps; ++s) {
      V nl[U][NC], nh[U][NC];
      if (s + 1 < n_steps) fetch(nl, nh);
      if (at == 0 && args.rot_pairs) {
        __syncwarp();
        const int* pos = args.pos + b * args.pos_sb + static_cast<int64_t>(t) * args.axes;
        if (row < args.rows)
#pragma unroll 1
          for (int p = lane & (team_lanes - 1); p < args.rot_pairs; p += team_lanes) {
            const int64_t at_axis = __ldg(pos + axis_table[p]);
            const uint64_t turns = static_cast<uint64_t>(at_axis) * turn_table[p];
            // the fraction of a turn, in [-1/2, 1/2)
            const float frac = static_cast<float>(static_cast<int32_t>(turns >> 32)) * 0x1p-32f;
            float sn, cs;
            if constexpr (sizeof(T) == 4) sincospif(2.f * frac, &sn, &cs);
            else __sincosf(6.283185307179586f * frac, &sn, &cs);
            cosines[p] = cs;
            cosines[p + stride] = sn;
          }
        __syncwarp();
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float yl[NC][VEC], yh[NC][VEC];
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int n = 0; n < NC; ++n) {
          rot_unpack(lo[u][n], yl[n]);
          rot_unpack(hi[u][n], yh[n]);
          if (used[n])
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              sum[0] = fmaf(yl[n][i], yl[n][i], sum[0]);
              sum[1] = fmaf(yh[n][i], yh[n][i], sum[1]);
            }
        }
        if (args.norm) {
          float q = sum[0] + sum[1];
          for (int m = group >> 1; m > 0; m >>= 1) q += __shfl_xor_sync(0xffffffffu, q, m);
          const float r = rsqrtf(fmaf(q, args.inv_d, args.eps));
#pragma unroll
          for (int n = 0; n < NC; ++n)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              yl[n][i] *= r * gl[n][i];
              yh[n][i] *= r * gh[n][i];
            }
        }
#pragma unroll
        for (int n = 0; n < NC; ++n) {
          if (!behind[n]) {
            const float* cp = cosines + (sub + n * group) * VEC;
            float c[VEC], sn[VEC];
            rot_trig<VEC>(cp, c);
            rot_trig<VEC>(cp + stride, sn);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              // pair i: elements i of both vectors, or neighbours 2 i, 2 i + 1 of 2 VEC
              float& e0 = !INTER ? yl[n][i] : 2 * i < VEC ? yl[n][2 * i % VEC] : yh[n][2 * i % VEC];
              float& e1 = !INTER             ? yh[n][i]
                          : 2 * i + 1 < VEC ? yl[n][(2 * i + 1) % VEC]
                                            : yh[n][(2 * i + 1) % VEC];
              const float f0 = e0, f1 = e1;
              e0 = fmaf(f0, c[i], -f1 * sn[i]);
              e1 = fmaf(f1, c[i], f0 * sn[i]);
            }
          }
          if (head < heads && used[n]) {
            *reinterpret_cast<V*>(dst + el[n]) = rot_pack<T, VEC>(yl[n]);
            *reinterpret_cast<V*>(dst + eh[n]) = rot_pack<T, VEC>(yh[n]);
          }
        }
        head += 1 << sshift;
        dst += out_head;
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int n = 0; n < NC; ++n) {
          lo[u][n] = nl[u][n];
          hi[u][n] = nh[u][n];
        }
      if (++at == steps) {
        at = 0;
        next_unit(row, b, t, part);
        head = first_head(row, part);
        dst = static_cast<T*>(x.out) + b * x.ob + t * x.ot + head * x.oh;
      }
    }
    __syncwarp();  // the other tensor's cosines overwrite these
  }
}

}  // namespace dcnv2
