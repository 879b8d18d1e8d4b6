// dcnv2_attention_step_kernel.cuh — attention of few query rows (single tokens and their grouped
// heads, up to 16 per kv head) to the states of another sequence.
//
// The formulas are those of dcnv2_attention_kernel.cuh. Here every state is read once and used
// by 16 rows at most, so the time is that of reading K and V; the work on them only has to keep
// up. Each warp runs by itself: it copies chunks of 4 KB of K and of V (cp.async, 16 bytes per
// lane, two chunks ahead) into a ring of its own in shared memory, multiplies with m16n8k16
// MMAs on 16 padded rows, and keeps its own maximum, sum and O in registers, so that no barrier
// stands between the loads. (Tensor-memory MMAs would need 128 rows and barriers between the
// roles: the tiled kernel takes 88 us where this one takes 32, for 32 x 5456 states, heads of 32;
// at 8 x 60001 states of 8 kv heads of 128 309 and 288.) The warps' parts are joined in
// shared memory; the CTAs of a cluster, which split the states, send theirs to the CTA that
// finishes the element (stores into distributed shared memory, one barrier), which adds them in
// a fixed order.
//
// Bound: HBM; a CTA draws at most about 50 GB/s, whatever it has in flight (64 to 192 KB
// measured), so all SMs have to take part. 8 sequences of up to 60001 states, 8 kv heads of 128
// (1.17 GB): 202 us, 5.8 TB/s, 89 % of the copy rate (213 us, 5.5 TB/s, with inputs that change
// from call to call); all 60001 of each: 288 us, 6.8 TB/s. 32 padded images, heads of 32: 32 us,
// 3.5 TB/s: one CTA per (image, head), two on most SMs, the time that of the fullest images;
// without padding the same 32 us are 5.6 TB/s. One sequence, 8 kv heads, 5456 states: 10.9 us, of
// which 4.3 us are a launch without states and 2 us the join over 16 CTAs.
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
constexpr int kStepMaxSplit = 16;  // CTAs of a cluster

struct AttnStepArgs {
  AttnTensor q, k, v, o;
  const int* kv_lens;
  const uint8_t* key_mask;
  int64_t mask_sb;
  float* lse;
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
  // at the end, over the rings: fp32 O of each warp [16][DP]; behind them the warps' (max, sum),
  // then what the CTAs of the cluster send: (max, sum) of all rows, O of the elements finished here
  static constexpr uint32_t kPart = kStepRows * DP * 4;
  static constexpr uint32_t kStats = kBytes;                      // [kStepWarps][16] float2
  static constexpr uint32_t kSentStats = kStats + kStepWarps * kStepRows * 8;  // [split][16] float2
  static constexpr uint32_t kSent = kSentStats + kStepMaxSplit * kStepRows * 8;
  static constexpr uint32_t kTotal = kSent + kPart + kStepMaxSplit * 16;
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

// The lane's part of copying a chunk: 16-byte piece c of rows r0, r0 + kRowsAtOnce, ...
template <int DP>
struct StepCopy {
  static constexpr int kChunks = DP / 8, kRowsAtOnce = 32 / kChunks;
  static constexpr int kTimes = StepLayout<DP>::kKeys / kRowsAtOnce;
  const uint16_t *k, *v;   // of row r0 of the first chunk
  int64_t kst, vst;        // elements between the lane's rows
  uint32_t r0;
  uint32_t c;
  bool inside;             // the piece lies inside the head

  __device__ __forceinline__ StepCopy(const uint16_t* kp, const uint16_t* vp, int64_t ks, int64_t vs,
                                      int D, int lane)
      : kst(ks * kRowsAtOnce), vst(vs * kRowsAtOnce), r0(lane / kChunks), c(lane % kChunks) {
    inside = static_cast<int>(c) * 8 < D;
    k = kp + r0 * ks + (inside ? c * 8 : 0);
    v = vp + r0 * vs + (inside ? c * 8 : 0);
  }
  // The chunk whose first row is kKeys * chunk behind; rows whose bit is not set, and elements
  // behind the head, are filled with zeros.
  __device__ __forceinline__ void operator()(uint32_t dst, int chunk, uint64_t keep,
                                             bool whole) const {
    const uint16_t* kp = k + static_cast<int64_t>(chunk) * kTimes * kst;
    const uint16_t* vp = v + static_cast<int64_t>(chunk) * kTimes * vst;
#pragma unroll
    for (int i = 0; i < kTimes; ++i) {
      const uint32_t to = dst + step_at<DP>(i * kRowsAtOnce + r0, c);
      const bool take = inside && (whole || ((keep >> (i * kRowsAtOnce + r0)) & 1));
      ptx::cp_async_16(to, take ? kp : k, take);  // (nothing is read where take is false)
      ptx::cp_async_16(to + StepLayout<DP>::kTile, take ? vp : v, take);
      kp += kst;
      vp += vst;
    }
  }
};

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
  if (args.split > 1) ptx::cluster_arrive();  // waited for before anything is sent to a CTA
  ptx::griddep_wait();

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
  constexpr uint64_t kWhole = KEYS == 64 ? ~0ull : (1ull << (KEYS & 63)) - 1;
  uint8_t ahead[2] = {0, 0};
  auto fetch_mask = [&](int chunk) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int r = x * 32 + lane, j = chunk * KEYS + r;
      ahead[x] = chunk < c1 && r < KEYS && j < len ? __ldg(mask + j) : 0;
    }
  };
  const StepCopy<DP> copy(k, v, args.k.st, args.v.st, args.D, lane);
  uint64_t kept[NS];  // of the chunks in the ring
  int next = c0;      // chunk that is loaded next
  auto load = [&](int stage) -> uint64_t {
    uint64_t bits = 0;
    if (next < c1) {
      const int left = len - next * KEYS;
      bits = left >= KEYS ? kWhole : (1ull << left) - 1;
      if (mask) {
        const uint64_t lo = __ballot_sync(0xffffffffu, ahead[0] != 0);
        const uint64_t hi = KEYS > 32 ? __ballot_sync(0xffffffffu, ahead[1] != 0) : 0;
        bits &= lo | hi << 32;
        fetch_mask(next + 1);
      }
      if (bits) copy(ring + stage * LY::kStage, next, bits, bits == kWhole);
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
  const bool upper = args.rows > 8;      // rows 8 to 15 are in use
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

    // two accumulators per score tile (even and odd k-steps), so that MMAs do not wait for one
    // another
    constexpr int CH = KT >= 4 ? 2 : 1;
    float s2[CH][NT][4];
#pragma unroll
    for (int z = 0; z < CH; ++z)
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int y = 0; y < 4; ++y) s2[z][x][y] = 0.f;
#pragma unroll
    for (int x = 0; x < KT; ++x)
#pragma unroll
      for (int y = 0; y < NT; y += 2) {
        // four 8x8 tiles: states 8 y .. 8 y + 15 (lanes 0-15: piece 2 x, 16-31: piece 2 x + 1)
        uint32_t f[4];
        ptx::ldmatrix_x4(f, kt + step_at<DP>(y * 8 + (lane & 15), 2 * x + (lane >> 4)));
        ptx::mma_16816<BF16>(s2[x % CH][y], qf[x], f[0], f[2]);
        ptx::mma_16816<BF16>(s2[x % CH][y + 1], qf[x], f[1], f[3]);
      }
    float (&s)[NT][4] = s2[0];
#pragma unroll
    for (int x = 0; x < NT; ++x)
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        if constexpr (CH == 2) s[x][y] += s2[1][x][y];
        if (bits != kWhole && !((bits >> (x * 8 + t4 * 2 + (y & 1))) & 1)) s[x][y] = -INFINITY;
      }
    // the lane's maximum of rows g4 and g4 + 8; the quad's is needed only where a row's reference
    // has to move
    float top[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      top[r] = fmaxf(s[0][2 * r], s[0][2 * r + 1]);
#pragma unroll
      for (int x = 1; x < NT; ++x) top[r] = fmaxf(top[r], fmaxf(s[x][2 * r], s[x][2 * r + 1]));
    }
    // ((-inf) - (-inf) is NaN, which is not greater)
    if (__any_sync(0xffffffffu, (top[0] - m_ref[0]) * c > kAttnLazy ||
                                    (upper && (top[1] - m_ref[1]) * c > kAttnLazy))) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float m = fmaxf(m_ref[r], top[r]);
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
        const float fac = m == m_ref[r] ? 1.f : ptx::ex2((m_ref[r] - m) * c);
        l[r] *= fac;
        m_ref[r] = m;
#pragma unroll
        for (int x = 0; x < OT; ++x) {
          o[x][2 * r] *= fac;
          o[x][2 * r + 1] *= fac;
        }
      }
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      if (r == 1 && !upper) {  // no such rows: no exponentials
#pragma unroll
        for (int x = 0; x < NT; ++x) s[x][2] = s[x][3] = 0.f;
        continue;
      }
      const float neg = (m_ref[r] == -INFINITY ? 0.f : -m_ref[r] * c) + shift;
      float sum[2] = {0.f, 0.f};
#pragma unroll
      for (int x = 0; x < NT; ++x) {
        s[x][2 * r] = ptx::ex2(fmaf(s[x][2 * r], c, neg));
        s[x][2 * r + 1] = ptx::ex2(fmaf(s[x][2 * r + 1], c, neg));
        sum[x & 1] += s[x][2 * r] + s[x][2 * r + 1];
      }
      l[r] += sum[0] + sum[1];
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
  // element quad x is finished by CTA x % split, as its element quad x / split
  const int quads = args.D / 4, items = args.rows * quads;
  const int mine = (items + args.split - 1) / args.split;
  if (args.split > 1) ptx::cluster_wait();
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
      const int to = x % args.split, at = x / args.split;
      ptx::st_cluster_f4(ptx::mapa_shared(base + LY::kSent + (rank * mine + at) * 16, to), acc);
      if (d == 0)
        for (int y = 0; y < args.split; ++y)
          ptx::st_cluster_f2(
              ptx::mapa_shared(base + LY::kSentStats + (rank * kStepRows + r) * 8, y),
              make_float2(top, total));
    }
  }
  if (args.split > 1) {
    // ---------------------------------------------------------- parts of the CTAs
    ptx::cluster_sync();  // all has arrived; nothing is sent from here on
    const float2* ml_of = reinterpret_cast<const float2*>(step_smem + LY::kSentStats);
    const float4* sent = reinterpret_cast<const float4*>(step_smem + LY::kSent);
    for (int at = threadIdx.x; at < mine && at * args.split + rank < items; at += kStepThreads) {
      const int x = at * args.split + rank, r = x / quads, d = (x - r * quads) * 4;
      float top = -INFINITY, total = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int y = 0; y < args.split; ++y) top = fmaxf(top, ml_of[y * kStepRows + r].x);
      for (int y = 0; y < args.split; ++y) {
        const float2 ml = ml_of[y * kStepRows + r];
        const float4 q = sent[y * mine + at];
        const float f = ml.x == top ? 1.f : ptx::ex2((ml.x - top) * c);
        total = fmaf(ml.y, f, total);
        acc.x = fmaf(q.x, f, acc.x); acc.y = fmaf(q.y, f, acc.y);
        acc.z = fmaf(q.z, f, acc.z); acc.w = fmaf(q.w, f, acc.w);
      }
      store(r, d, acc, top, total);
    }
  }
}

}  // namespace dcnv2
