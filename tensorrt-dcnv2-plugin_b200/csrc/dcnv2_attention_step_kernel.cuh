// dcnv2_attention_step_kernel.cuh — attention of few query rows (single tokens and their grouped
// heads, up to 16 per kv head) to the states of another sequence.
//
// The formulas are those of dcnv2_attention_kernel.cuh. Here every state is read once and used by 16
// rows at most, so the time is that of reading K and V; the work on them only has to keep up. Each
// warp runs by itself: it copies chunks of K and V rows (cp.async, 16 bytes per lane, 16 KB of D = 128
// elements in flight per stage of a warp pair of chunks) into a ring of its own in shared memory,
// multiplies with m16n8k16 MMAs on 16 padded rows, and keeps its own maximum, sum and O in
// registers, so that no barrier stands between the loads. Tensor-memory MMAs would need 128 rows
// (or the states as rows) and barriers between the roles; at these sizes the tensor core is idle
// most of the time either way. The warps' parts are joined in shared memory, those of the CTAs of a
// cluster, which split the states, through distributed shared memory in a fixed order.
//
// States that are not kept are not read: their rows in shared memory are filled with zeros (the
// copy's source size is 0), their scores are -inf; chunks without a kept state cost nothing.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "dcnv2_attention_kernel.cuh"
#include "ptx_sm100.cuh"

namespace dcnv2 {

constexpr int kStepWarps = 4;
constexpr int kStepThreads = kStepWarps * 32;
constexpr int kStepRows = 16;

struct AttnStepArgs {
  AttnTensor q, k, v, o;
  const int* kv_lens;
  const uint8_t* key_mask;
  int64_t mask_sb;
  float* lse;
  int* err;
  int L, S, H, G, D;
  int group, rows;       // rows = L * group <= 16
  int split;             // CTAs of a cluster along the states
  float scale;
};

// Chunk of states a warp takes at a time: KEYS rows of DP elements of K and of V.
template <int DP>
struct StepLayout {
  static constexpr int kKeys = DP == 128 ? 16 : DP == 64 ? 32 : 64;
  static constexpr int kStages = 3;
  static constexpr uint32_t kRow = DP * 2;                        // bytes of a row
  static constexpr uint32_t kTile = kKeys * kRow;                 // 4 KB
  static constexpr uint32_t kStage = 2 * kTile;                   // K, V
  static constexpr uint32_t kWarp = kStages * kStage;             // 24 KB
  static constexpr uint32_t kBytes = kStepWarps * kWarp;
  // at the end, over the rings: fp32 O of each warp [16][DP], then the CTA's; (max, sum) behind
  static constexpr uint32_t kPart = kStepRows * DP * 4;
  static constexpr uint32_t kStats = kBytes;                      // [kStepWarps + 1][16] float2
  static constexpr uint32_t kTotal = kStats + (kStepWarps + 1) * kStepRows * 8;
  static_assert(kPart <= kWarp, "a warp's O fits over its ring");
};

// Byte offset of the 16-byte chunk c of row r: the chunk index is mixed with the row so that the 8
// rows of an ldmatrix tile lie in different banks.
template <int DP>
__device__ __forceinline__ uint32_t step_at(int r, int c) {
  constexpr int kChunks = DP / 8;
  const int mix = kChunks >= 8 ? r & 7 : (r >> 1) & 3;  // rows of 64 bytes: two per 128-byte line
  return static_cast<uint32_t>(r) * (DP * 2) + (static_cast<uint32_t>(c ^ mix) << 4);
}

// Copies a chunk's rows j0 .. j0 + kKeys - 1 of both tensors; rows whose bit is not set, and elements
// from D on, are filled with zeros.
template <int DP>
__device__ __forceinline__ void step_load(uint32_t dst, const uint16_t* k, const uint16_t* v,
                                          int64_t kst, int64_t vst, int j0, uint64_t keep, int D,
                                          int lane) {
  using LY = StepLayout<DP>;
  constexpr int kChunks = DP / 8, kRowsAtOnce = 32 / kChunks;
  const int c = lane % kChunks;
  const bool inside = c * 8 < D;
#pragma unroll
  for (int i = 0; i < LY::kKeys / kRowsAtOnce; ++i) {
    const int r = i * kRowsAtOnce + lane / kChunks;
    const bool take = inside && ((keep >> r) & 1);
    const int64_t j = take ? j0 + r : 0;
    const uint32_t at = dst + step_at<DP>(r, c);
    ptx::cp_async_16(at, k + j * kst + (inside ? c * 8 : 0), take);
    ptx::cp_async_16(at + LY::kTile, v + j * vst + (inside ? c * 8 : 0), take);
  }
}

template <int DP, bool BF16>
__global__ void __launch_bounds__(kStepThreads)
    dcnv2_attention_step_kernel(const __grid_constant__ AttnStepArgs args) {
  using LY = StepLayout<DP>;
  constexpr int KEYS = LY::kKeys, NS = LY::kStages;
  constexpr int NT = KEYS / 8;       // score tiles of 8 states
  constexpr int KT = DP / 16;        // k-steps of the scores
  constexpr int OT = DP / 8;         // output tiles of 8 elements
  extern __shared__ __align__(128) uint8_t step_smem[];
  const uint32_t base = ptx::smem_addr(step_smem);
  const int warp = static_cast<int>(threadIdx.x) >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(blockIdx.x) % args.split;
  const int unit = static_cast<int>(blockIdx.x) / args.split;
  const int g = unit % args.G, b = unit / args.G;
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  if (threadIdx.x == 0) args.err[blockIdx.x] = 0;  // nothing here waits without end

  int len = args.S;
  if (args.kv_lens) len = max(0, min(len, __ldg(args.kv_lens + b)));
  // the states are dealt to the warps of the cluster in runs of whole chunks
  const int chunks = (len + KEYS - 1) / KEYS;
  const int warps = args.split * kStepWarps, me = rank * kStepWarps + warp;
  const int c0 = static_cast<int>(static_cast<int64_t>(chunks) * me / warps);
  const int c1 = static_cast<int>(static_cast<int64_t>(chunks) * (me + 1) / warps);
  const uint16_t* k = static_cast<const uint16_t*>(args.k.p) + b * args.k.sb + g * args.k.sh;
  const uint16_t* v = static_cast<const uint16_t*>(args.v.p) + b * args.v.sb + g * args.v.sh;
  const uint8_t* mask = args.key_mask ? args.key_mask + b * args.mask_sb : nullptr;
  const uint32_t ring = base + warp * LY::kWarp;

  // bits of the kept states of a chunk; the lane's mask bytes are fetched a chunk ahead
  uint8_t ahead[2] = {0, 0};
  auto fetch_mask = [&](int chunk) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int r = x * 32 + lane, j = chunk * KEYS + r;
      ahead[x] = mask && chunk < c1 && r < KEYS && j < len ? __ldg(mask + j) : 0;
    }
  };
  auto keep_bits = [&](int chunk) -> uint64_t {
    const int left = len - chunk * KEYS;
    uint64_t bits = left >= KEYS ? (KEYS == 64 ? ~0ull : (1ull << KEYS) - 1) : (1ull << left) - 1;
    if (mask) {
      const uint64_t lo = __ballot_sync(0xffffffffu, ahead[0] != 0);
      const uint64_t hi = KEYS > 32 ? __ballot_sync(0xffffffffu, ahead[1] != 0) : 0;
      bits &= lo | hi << 32;
    }
    return bits;
  };
  uint64_t kept[NS];  // of the chunks in the ring
  int next = c0;      // chunk that is loaded next
  auto load = [&](int stage) -> uint64_t {
    uint64_t bits = 0;
    if (next < c1) {
      if (mask) {
        bits = keep_bits(next);
        fetch_mask(next + 1);
      } else {
        bits = keep_bits(next);
      }
      if (bits)
        step_load<DP>(ring + stage * LY::kStage, k, v, args.k.st, args.v.st, next * KEYS, bits,
                      args.D, lane);
      ++next;
    }
    ptx::cp_async_commit();
    return bits;
  };
  if (mask) fetch_mask(c0);
#pragma unroll
  for (int s = 0; s < NS - 1; ++s) kept[s] = load(s);

  // Q fragments: rows g4 and g4 + 8 of the quad's lane group, 16 elements per k-step
  const int g4 = lane >> 2, t4 = lane & 3;
  uint32_t qf[KT][4];
#pragma unroll
  for (int x = 0; x < KT; ++x)
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const int r = g4 + (y & 1) * 8, d = x * 16 + (y >> 1) * 8 + t4 * 2;
      const int tok = r / args.group, h = g * args.group + r - tok * args.group;
      qf[x][y] = r < args.rows && d < args.D
                     ? __ldg(reinterpret_cast<const uint32_t*>(
                           static_cast<const uint16_t*>(args.q.p) + b * args.q.sb +
                           tok * args.q.st + h * args.q.sh + d))
                     : 0u;
    }
  const float c = args.scale * kLog2e;
  const float shift = BF16 ? 0.f : 7.f;  // as in the tiled kernel
  float m_ref[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  float o[OT][4];
#pragma unroll
  for (int x = 0; x < OT; ++x)
#pragma unroll
    for (int y = 0; y < 4; ++y) o[x][y] = 0.f;

  int stage = 0;
  for (int chunk = c0; chunk < c1; ++chunk) {
    ptx::cp_async_wait<NS - 2>();
    __syncwarp();
    uint64_t bits = kept[0];
#pragma unroll
    for (int s = 0; s + 2 < NS; ++s) kept[s] = kept[s + 1];
    const uint32_t kt = ring + stage * LY::kStage, vt = kt + LY::kTile;
    // the stage that was used last is free: its readers are this warp's lanes, behind the barrier
    kept[NS - 2] = load((stage + NS - 1) % NS);
    stage = stage + 1 == NS ? 0 : stage + 1;
    if (!bits) continue;

    float s[NT][4];
#pragma unroll
    for (int x = 0; x < NT; ++x)
#pragma unroll
      for (int y = 0; y < 4; ++y) s[x][y] = 0.f;
#pragma unroll
    for (int x = 0; x < KT; ++x)
#pragma unroll
      for (int y = 0; y < NT; y += 2) {
        // four 8x8 tiles: states 8 y .. 8 y + 15 (lanes 0-15: chunk 2 x, 16-31: chunk 2 x + 1)
        uint32_t f[4];
        ptx::ldmatrix_x4(f, kt + step_at<DP>(y * 8 + (lane & 15), 2 * x + (lane >> 4)));
        ptx::mma_16816<BF16>(s[y], qf[x], f[0], f[2]);
        ptx::mma_16816<BF16>(s[y + 1], qf[x], f[1], f[3]);
      }
    if (bits != (KEYS == 64 ? ~0ull : (1ull << KEYS) - 1)) {
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int y = 0; y < 4; ++y)
          if (!((bits >> (x * 8 + t4 * 2 + (y & 1))) & 1)) s[x][y] = -INFINITY;
    }
    // per row half (rows g4, g4 + 8): the chunk's maximum over the quad
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float top = fmaxf(s[0][2 * r], s[0][2 * r + 1]);
#pragma unroll
      for (int x = 1; x < NT; ++x) top = fmaxf(top, fmaxf(s[x][2 * r], s[x][2 * r + 1]));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const float m = fmaxf(m_ref[r], top);
      if (__any_sync(0xffffffffu, (m - m_ref[r]) * c > kAttnLazy)) {
        const float fac = m == m_ref[r] ? 1.f : ptx::ex2((m_ref[r] - m) * c);
        l[r] *= fac;
        m_ref[r] = m;
#pragma unroll
        for (int x = 0; x < OT; ++x) {
          o[x][2 * r] *= fac;
          o[x][2 * r + 1] *= fac;
        }
      }
      const float neg = (m_ref[r] == -INFINITY ? 0.f : -m_ref[r] * c) + shift;
#pragma unroll
      for (int x = 0; x < NT; ++x) {
        s[x][2 * r] = ptx::ex2(fmaf(s[x][2 * r], c, neg));
        s[x][2 * r + 1] = ptx::ex2(fmaf(s[x][2 * r + 1], c, neg));
        l[r] += s[x][2 * r] + s[x][2 * r + 1];
      }
    }
#pragma unroll
    for (int x = 0; x < KEYS / 16; ++x) {
      // the score fragments of two state tiles are the A fragment of one k-step
      uint32_t p[4];
      p[0] = ptx::pack16<BF16>(s[2 * x][0], s[2 * x][1]);
      p[1] = ptx::pack16<BF16>(s[2 * x][2], s[2 * x][3]);
      p[2] = ptx::pack16<BF16>(s[2 * x + 1][0], s[2 * x + 1][1]);
      p[3] = ptx::pack16<BF16>(s[2 * x + 1][2], s[2 * x + 1][3]);
#pragma unroll
      for (int y = 0; y < OT; y += 2) {
        uint32_t f[4];
        ptx::ldmatrix_x4_trans(f, vt + step_at<DP>(x * 16 + (lane & 15), y + (lane >> 4)));
        ptx::mma_16816<BF16>(o[y], p, f[0], f[1]);
        ptx::mma_16816<BF16>(o[y + 1], p, f[2], f[3]);
      }
    }
  }
  ptx::cp_async_wait<0>();
  __syncwarp();

  // ------------------------------------------------------------ parts of the warps
  float2* stats = reinterpret_cast<float2*>(step_smem + LY::kStats);
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    if (t4 == 0) stats[warp * kStepRows + g4 + 8 * r] = make_float2(m_ref[r], l[r]);
    float* part = reinterpret_cast<float*>(step_smem + warp * LY::kWarp) + (g4 + 8 * r) * DP;
#pragma unroll
    for (int x = 0; x < OT; ++x)
      *reinterpret_cast<float2*>(part + x * 8 + t4 * 2) =
          make_float2(o[x][2 * r], o[x][2 * r + 1]);
  }
  __syncthreads();
  // joined parts of one row's 4 elements: factors to the common maximum, then the sums
  auto store = [&](int r, int d, float4 acc, float top, float total) {
    const int tok = r / args.group, h = g * args.group + r - tok * args.group;
    const float inv = total == 0.f ? 0.f : 1.f / total;
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(const_cast<void*>(args.o.p)) +
                              b * args.o.sb + tok * args.o.st + h * args.o.sh + d) =
        make_uint2(ptx::pack16<BF16>(acc.x * inv, acc.y * inv),
                   ptx::pack16<BF16>(acc.z * inv, acc.w * inv));
    if (args.lse && d == 0)
      args.lse[(static_cast<int64_t>(b) * args.H + h) * args.L + tok] =
          total == 0.f ? -INFINITY : kLn2 * (top * c - shift + log2f(total));
  };
  const int quads = args.D / 4, items = args.rows * quads;
  for (int x = threadIdx.x; x < items; x += kStepThreads) {
    const int r = x / quads, d = (x - r * quads) * 4;
    float top = -INFINITY, total = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int y = 0; y < kStepWarps; ++y) top = fmaxf(top, stats[y * kStepRows + r].x);
#pragma unroll
    for (int y = 0; y < kStepWarps; ++y) {
      const float2 ml = stats[y * kStepRows + r];
      const float f = ml.x == top ? 1.f : ptx::ex2((ml.x - top) * c);
      const float4 q = *reinterpret_cast<const float4*>(step_smem + y * LY::kWarp +
                                                        (r * DP + d) * 4);
      total = fmaf(ml.y, f, total);
      acc.x = fmaf(q.x, f, acc.x); acc.y = fmaf(q.y, f, acc.y);
      acc.z = fmaf(q.z, f, acc.z); acc.w = fmaf(q.w, f, acc.w);
    }
    if (args.split == 1) {
      store(r, d, acc, top, total);
    } else {
      // over the first warp's part: each place is read and written by this thread alone
      *reinterpret_cast<float4*>(step_smem + (r * DP + d) * 4) = acc;
      if (d == 0) stats[kStepWarps * kStepRows + r] = make_float2(top, total);
    }
  }
  if (args.split > 1) {
    // ---------------------------------------------------------- parts of the CTAs
    ptx::cluster_sync();
    for (int x = rank * kStepThreads + static_cast<int>(threadIdx.x); x < items;
         x += args.split * kStepThreads) {
      const int r = x / quads, d = (x - r * quads) * 4;
      const uint32_t st = base + LY::kStats + (kStepWarps * kStepRows + r) * 8;
      float top = -INFINITY, total = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int y = 0; y < args.split; ++y)
        top = fmaxf(top, ptx::ld_cluster_f2(ptx::mapa_shared(st, y)).x);
#pragma unroll 4
      for (int y = 0; y < args.split; ++y) {
        const float2 ml = ptx::ld_cluster_f2(ptx::mapa_shared(st, y));
        const float4 q = ptx::ld_cluster_f4(ptx::mapa_shared(base + (r * DP + d) * 4, y));
        const float f = ml.x == top ? 1.f : ptx::ex2((ml.x - top) * c);
        total = fmaf(ml.y, f, total);
        acc.x = fmaf(q.x, f, acc.x); acc.y = fmaf(q.y, f, acc.y);
        acc.z = fmaf(q.z, f, acc.z); acc.w = fmaf(q.w, f, acc.w);
      }
      store(r, d, acc, top, total);
    }
    ptx::cluster_sync();  // the parts stay until every CTA has read them
  }
}

}  // namespace dcnv2
