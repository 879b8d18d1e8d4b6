// dcnv2_attention_kernel.cuh — attention of queries to the states of another sequence, on tensor
// cores, in one pass over the states.
//
// For query row i of a sequence and its kept states j: s_ij = scale q_i k_j, m = max s, p = exp(s -
// m), out_i = sum p v / sum p, lse_i = m + log sum p; without kept states out = 0, lse = -inf.
//
// Rows: the queries of one kv head, token by token, the heads of its group side by side (row r =
// token r / group, head r % group), so that grouped heads fill an MMA's 128 rows together and read
// each state once. States come in tiles of 128. Per tile: S[128 rows, 128 states] = Q K^T into
// tensor memory; each softmax thread owns a row, reads its 128 scores, writes the rounded
// probabilities back as the A operand; O[128, D] += P V accumulates in tensor memory. The running
// maximum is followed lazily: O and the row's sum are rescaled only when it has grown by more than
// 2^8 (probabilities up to 2^8 are as exact as those up to 1, and the sums are fp32), so that most
// tiles touch O only through the MMA.
//
// Two softmax warpgroups alternate, so that one's exponentials overlap the other's MMAs:
//   PAIRED = false  two tiles of 128 rows per CTA, each state tile used by both (many rows);
//   PAIRED = true   one tile of rows, the warpgroups take the even and the odd state tiles (few
//                   rows: single tokens, grouped heads), and their halves are joined at the end.
// A cluster of CTAs may split the states; the parts (fp32 O, maximum, sum) are joined through
// distributed shared memory, every CTA finishing a share of the rows: no second launch, no
// workspace, and the order of the sums is fixed.
//
// Roles (352 threads): warps 0-3 and 4-7 softmax and epilogue, warp 8 producer (kept-state words of
// each tile, TMA of K and V; tiles without a kept state are left out altogether), warp 9 MMA issuer,
// warp 10 zeroes the V rows of states that are not kept (their probability is 0, but 0 * NaN is
// not). Every wait is bounded.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/dcnv2.h"
#include "dcnv2_wait.cuh"
#include "ptx_sm100.cuh"

namespace dcnv2 {

constexpr int kAttnTile = 128;                 // states per tile, rows per MMA
constexpr int kAttnThreads = 11 * 32;
constexpr int kAttnProducerWarp = 8, kAttnMmaWarp = 9, kAttnFixWarp = 10;
constexpr uint32_t kAttnBlockBytes = kAttnTile * 128;  // 128 rows of one 128-byte swizzle block
constexpr float kAttnLazy = 8.f;               // log2 of the growth that rescales
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct AttnTensor {
  const void* p;
  int64_t sb, st, sh;                          // strides: batch, token, head (elements)
};

struct AttnArgs {
  AttnTensor q, o;
  const int* kv_lens;
  const uint8_t* key_mask;
  int64_t mask_sb;
  float* lse;                                  // [B][H][L] or null
  int* err;                                    // one word per CTA
  int L, S, H, G, D;                           // G kv heads
  int group, rows;                             // group = H / G, rows = L * group
  int row_tiles;                               // CTAs along the rows
  int split;                                   // CTAs of a cluster along the states
  int k_batch, k_head, v_batch, v_head;        // 0: the tensor is shared along that axis
  float scale;
  unsigned long long timeout_ns;
};

// Shared-memory layout of an instance (bytes from a 1024-aligned base).
template <int DP, bool PAIRED>
struct AttnLayout {
  static constexpr int kBlocks = DP / 64;                         // swizzle blocks of a row
  static constexpr uint32_t kTileBytes = kBlocks * kAttnBlockBytes;
  static constexpr int kQTiles = PAIRED ? 1 : 2;
  static constexpr int kStages = DP == 128 ? (PAIRED ? 3 : 2) : (PAIRED ? 6 : 4);
  static constexpr int kInfos = kStages + 2;
  static constexpr uint32_t kQ = 0;
  static constexpr uint32_t kK = kQTiles * kTileBytes;
  static constexpr uint32_t kV = kK + kStages * kTileBytes;
  static constexpr uint32_t kInfo = kV + kStages * kTileBytes;    // kInfos x 32 bytes
  static constexpr uint32_t kBars = kInfo + kInfos * 32;
  static constexpr int kNumBars = 5 * kStages + kInfos + 6;
  static constexpr uint32_t kSlot = kBars + kNumBars * 8;         // TMEM address, abort flag
  static constexpr uint32_t kBytes = kSlot + 16;
  // at the end, over K and V: fp32 O of the two warpgroups; over Q: their (maximum, sum)
  static constexpr uint32_t kPart = kK;
  static constexpr uint32_t kPartBytes = kAttnTile * DP * 4;
  static_assert(2 * kPartBytes <= 2 * kStages * kTileBytes, "parts fit over K and V");
  static_assert(2 * kAttnTile * 8 <= kK, "statistics fit over Q");
};
template <int DP, bool PAIRED>
constexpr size_t attn_smem_bytes() {
  return AttnLayout<DP, PAIRED>::kBytes + 1024;  // + alignment slack
}

// Place of the 16-byte chunk c of row r of an fp32 part: chunks are rotated by the row, so that
// threads that own a row each do not meet in one bank.
template <int DP>
__device__ __forceinline__ uint32_t attn_part_at(int r, int c) {
  return static_cast<uint32_t>(r) * (DP * 4) + (static_cast<uint32_t>(c ^ (r & 7)) << 4);
}

template <int DP, bool PAIRED, bool BF16>
__global__ void __launch_bounds__(kAttnThreads, 1)
    dcnv2_cross_attention_kernel(const __grid_constant__ AttnArgs args,
                                 const __grid_constant__ CUtensorMap tmap_k,
                                 const __grid_constant__ CUtensorMap tmap_v) {
  using LY = AttnLayout<DP, PAIRED>;
  constexpr int NS = LY::kStages, NI = LY::kInfos;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const uint32_t base = ptx::smem_addr(smem);
  const int warp = static_cast<int>(threadIdx.x) >> 5, lane = threadIdx.x & 31;
  const uint32_t k_full = base + LY::kBars;            // [NS] K tile landed
  const uint32_t k_empty = k_full + 8 * NS;            // [NS] its products done
  const uint32_t v_full = k_empty + 8 * NS;            // [NS] V tile landed
  const uint32_t v_ready = v_full + 8 * NS;            // [NS] its rows of unkept states zeroed
  const uint32_t v_empty = v_ready + 8 * NS;           // [NS] its products done
  const uint32_t info_full = v_empty + 8 * NS;         // [NI] kept-state words of a tile, or the end
  const uint32_t s_full = info_full + 8 * NI;          // [2] scores of warpgroup w
  const uint32_t p_ready = s_full + 16;                // [2] probabilities of warpgroup w
  const uint32_t q_full = p_ready + 16;
  const uint32_t o_final = q_full + 8;
  uint32_t* slot = reinterpret_cast<uint32_t*>(smem + LY::kSlot);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(slot + 1);
  uint32_t* infos = reinterpret_cast<uint32_t*>(smem + LY::kInfo);  // words 0-3, then 1 = the end
  const WaitCtx wc{args.timeout_ns, args.err + blockIdx.x, abort_flag};

  // blockIdx.x = ((batch * kv heads + kv head) * row_tiles + row tile) * split + rank
  const int rank = static_cast<int>(blockIdx.x) % args.split;
  int rest = static_cast<int>(blockIdx.x) / args.split;
  const int row0 = (rest % args.row_tiles) * (PAIRED ? kAttnTile : 2 * kAttnTile);
  rest /= args.row_tiles;
  const int g = rest % args.G, b = rest / args.G;

  ptx::griddep_launch_dependents();
  if (threadIdx.x == 0) {
    for (int i = 0; i < NS; ++i) {
      ptx::mbar_init(k_full + 8 * i, 1);
      ptx::mbar_init(k_empty + 8 * i, 1);
      ptx::mbar_init(v_full + 8 * i, 1);
      ptx::mbar_init(v_ready + 8 * i, 1);
      ptx::mbar_init(v_empty + 8 * i, 1);
    }
    for (int i = 0; i < NI; ++i) ptx::mbar_init(info_full + 8 * i, 1);
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(s_full + 8 * i, 1);
      ptx::mbar_init(p_ready + 8 * i, 4);
    }
    ptx::mbar_init(q_full, 8);
    ptx::mbar_init(o_final, 1);
    *abort_flag = 0;
    ptx::fence_mbar_init();
  }
  if (warp == kAttnMmaWarp) {
    ptx::tmem_alloc(ptx::smem_addr(slot), 512);
    ptx::tmem_relinquish();
  }
  // the setup above overlaps the tail of the kernel ahead; memory is touched only from here
  ptx::griddep_wait();
  if (threadIdx.x == 0) *wc.err = 0;
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = *slot;
  // tensor memory: scores of warpgroup w at 128 w (the probabilities over their first half), its O
  // at 256 + DP w
  const int w = warp >> 2;  // softmax warpgroup
  const float c = args.scale * kLog2e;
  // fp16 probabilities are scaled by 2^7 (at most 2^15): small ones keep their bits longer
  const float shift = BF16 ? 0.f : 7.f;
  float m_ref = -INFINITY, l = 0.f;  // a softmax thread's row: reference maximum, sum

  if (warp == kAttnProducerWarp) {
    // ------------------------------------------------------------ producer
    int len = args.S;
    if (args.kv_lens) len = max(0, min(len, __ldg(args.kv_lens + b)));
    const int tiles = (len + kAttnTile - 1) / kAttnTile;
    const int t1 = static_cast<int>(static_cast<int64_t>(tiles) * (rank + 1) / args.split);
    int t = static_cast<int>(static_cast<int64_t>(tiles) * rank / args.split);
    const uint8_t* mask = args.key_mask ? args.key_mask + b * args.mask_sb : nullptr;
    uint8_t next[4];  // the lane's mask bytes of the next tile
    auto fetch = [&](int tile) {
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int j = tile * kAttnTile + x * 32 + lane;
        next[x] = tile < t1 && j < len ? __ldg(mask + j) : 0;
      }
    };
    if (mask) fetch(t);
    int i = 0;
    bool ok = true, k_ahead = false;  // k_ahead: K of tile i was started, V was not
    for (; t < t1 && ok; ++t) {
      uint32_t word[4];
      if (mask) {
#pragma unroll
        for (int x = 0; x < 4; ++x) word[x] = __ballot_sync(0xffffffffu, next[x] != 0);
        fetch(t + 1);
        if ((word[0] | word[1] | word[2] | word[3]) == 0) continue;
      } else {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int left = len - t * kAttnTile - x * 32;
          word[x] = left >= 32 ? 0xffffffffu : left <= 0 ? 0u : (1u << left) - 1u;
        }
      }
      const int s = i % NS, at = i % NI;
      const uint32_t ph = static_cast<uint32_t>(i / NS) & 1u;
      if (lane == 0) {
        // this slot's last tile was i - NS - 2; V of tile i - 1 was loaded over i - 1 - NS, whose
        // readers were done
        uint32_t* f = infos + at * 8;
        f[0] = word[0]; f[1] = word[1]; f[2] = word[2]; f[3] = word[3];
        f[4] = 0;
        ptx::mbar_arrive(info_full + 8 * at);
        ok = wait_bar<kSuspend>(k_empty + 8 * s, ph ^ 1u, wc, DCNV2_DEVERR_TIMEOUT_PRODUCER);
        if (ok) {
          ptx::mbar_arrive_expect_tx(k_full + 8 * s, LY::kTileBytes);
          for (int x = 0; x < LY::kBlocks; ++x)
            ptx::tma_load_4d(base + LY::kK + s * LY::kTileBytes + x * kAttnBlockBytes, &tmap_k,
                             x * 64, t * kAttnTile, g * args.k_head, b * args.k_batch,
                             k_full + 8 * s);
          k_ahead = true;
          ok = wait_bar<kSuspend>(v_empty + 8 * s, ph ^ 1u, wc, DCNV2_DEVERR_TIMEOUT_PRODUCER);
        }
        if (ok) {
          ptx::mbar_arrive_expect_tx(v_full + 8 * s, LY::kTileBytes);
          for (int x = 0; x < LY::kBlocks; ++x)
            ptx::tma_load_4d(base + LY::kV + s * LY::kTileBytes + x * kAttnBlockBytes, &tmap_v,
                             x * 64, t * kAttnTile, g * args.v_head, b * args.v_batch,
                             v_full + 8 * s);
          k_ahead = false;
          ++i;
        }
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
      i = __shfl_sync(0xffffffffu, i, 0);
    }
    if (lane == 0) {
      for (int x = 0; x < 2 && ok; ++x) {  // the end, for both warpgroups
        const int at = (i + x) % NI;
        infos[at * 8 + 4] = 1;
        ptx::mbar_arrive(info_full + 8 * at);
      }
      // copies in flight land before the CTA ends or its buffers are used for the parts
      for (int x = i > NS ? i - NS : 0; x < i; ++x) {
        const uint32_t ph = static_cast<uint32_t>(x / NS) & 1u;
        drain_bar(k_full + 8 * (x % NS), ph, wc);
        drain_bar(v_full + 8 * (x % NS), ph, wc);
      }
      if (k_ahead) drain_bar(k_full + 8 * (i % NS), static_cast<uint32_t>(i / NS) & 1u, wc);
    }
  } else if (warp == kAttnMmaWarp) {
    // ------------------------------------------------------------ MMA issuer
    // The warp runs this code as a whole (descriptors and barrier addresses stay in uniform
    // registers); one elected lane issues.
    constexpr uint32_t fmt = BF16 ? ptx::kFmtBf16 : 0;
    const uint32_t id_s = ptx::make_idesc(1, fmt, kAttnTile);
    const uint32_t id_o =
        ptx::make_idesc(1, fmt, static_cast<uint32_t>((args.D + 15) / 16 * 16)) | ptx::kIdescBMn;
    const int d_steps = (args.D + 15) / 16;
    const bool leader = ptx::elect_one();
    const uint64_t q_desc = ptx::sw128_kmajor_desc(base + LY::kQ);
    const uint64_t k_desc = ptx::sw128_kmajor_desc(base + LY::kK);
    const uint64_t v_desc = ptx::sw128_mnmajor_desc(base + LY::kV, kAttnBlockBytes);
    bool ok = wait_bar(q_full, 0, wc, DCNV2_DEVERR_TIMEOUT_MMA);
    // whether tile i exists (its words are there), or the states have ended
    auto exists = [&](int i) {
      ok = ok && wait_bar(info_full + 8 * (i % NI), static_cast<uint32_t>(i / NI) & 1u, wc,
                          DCNV2_DEVERR_TIMEOUT_MMA);
      ok = __all_sync(0xffffffffu, ok);
      return ok && ptx::ld_shared_u32_volatile(base + LY::kInfo + (i % NI) * 32 + 16) == 0;
    };
    auto commit = [&](uint32_t bar) {
      if (leader) ptx::tc_commit(bar);
    };
    auto scores = [&](int i, int wg) {  // S of warpgroup wg from K tile i
      const uint64_t q = q_desc + (PAIRED ? 0 : wg) * (LY::kTileBytes >> 4);
      const uint64_t k = k_desc + (i % NS) * (LY::kTileBytes >> 4);
      const uint32_t d = tmem + kAttnTile * wg;
      if (leader) {
#pragma unroll
        for (int x = 0; x < DP / 16; ++x) {
          const uint32_t off = ((x >> 2) * kAttnBlockBytes + (x & 3) * 32) >> 4;
          if (x < d_steps) ptx::mma_f16(d, q + off, k + off, id_s, x > 0);
        }
        ptx::tc_commit(s_full + 8 * wg);
      }
    };
    auto product = [&](int i, int wg, bool first) {  // O of warpgroup wg += P V tile i
      const uint64_t v = v_desc + (i % NS) * (LY::kTileBytes >> 4);
      const uint32_t d = tmem + 2 * kAttnTile + DP * wg, p = tmem + kAttnTile * wg;
      if (leader) {
#pragma unroll
        for (int x = 0; x < kAttnTile / 16; ++x)
          ptx::mma_f16_ta(d, p + 8 * x, v + x * (2048 >> 4), id_o, !first || x > 0);
      }
    };
    auto wait_k = [&](int i) {
      ok = ok && wait_bar(k_full + 8 * (i % NS), static_cast<uint32_t>(i / NS) & 1u, wc,
                          DCNV2_DEVERR_TIMEOUT_MMA);
      ptx::tc_fence_after();
      return ok = __all_sync(0xffffffffu, ok);
    };
    auto wait_pv = [&](int i, int wg, uint32_t turn) {
      ok = ok && wait_bar(v_ready + 8 * (i % NS), static_cast<uint32_t>(i / NS) & 1u, wc,
                          DCNV2_DEVERR_TIMEOUT_MMA) &&
           wait_bar(p_ready + 8 * wg, turn & 1u, wc, DCNV2_DEVERR_TIMEOUT_MMA);
      ptx::tc_fence_after();
      return ok = __all_sync(0xffffffffu, ok);
    };
    // A warpgroup's next scores are issued right behind its product, whose probabilities they
    // overwrite: the tensor core runs MMAs in the order of issue.
    if (PAIRED) {
      for (int i = 0; i < 2; ++i)
        if (exists(i) && wait_k(i)) {
          scores(i, i);
          commit(k_empty + 8 * (i % NS));
        }
      for (int i = 0; ok && exists(i); ++i) {
        const int wg = i & 1;
        if (!wait_pv(i, wg, static_cast<uint32_t>(i >> 1))) break;
        product(i, wg, i < 2);
        commit(v_empty + 8 * (i % NS));
        // the second end mark stands at most two behind the last tile
        if (exists(i + 1) && exists(i + 2) && wait_k(i + 2)) {
          scores(i + 2, wg);
          commit(k_empty + 8 * ((i + 2) % NS));
        }
      }
    } else if (exists(0) && wait_k(0)) {
      scores(0, 0);
      scores(0, 1);
      commit(k_empty);
      for (int i = 0;; ++i) {
        const bool more = exists(i + 1);
        for (int wg = 0; wg < 2 && ok; ++wg) {
          if (!wait_pv(i, wg, static_cast<uint32_t>(i))) break;
          product(i, wg, i == 0);
          if (wg) commit(v_empty + 8 * (i % NS));
          if (more && wait_k(i + 1)) scores(i + 1, wg);
        }
        if (!more || !ok) break;
        commit(k_empty + 8 * ((i + 1) % NS));
      }
    }
    commit(o_final);
    drain_bar(o_final, 0, wc);
  } else if (warp == kAttnFixWarp) {
    // ------------------------------------------------------------ V rows of unkept states
    for (int i = 0;; ++i) {
      const int s = i % NS, at = i % NI;
      bool ok = wait_bar<kSuspend>(info_full + 8 * at, static_cast<uint32_t>(i / NI) & 1u, wc,
                                   DCNV2_DEVERR_TIMEOUT_PRODUCER);
      if (!__all_sync(0xffffffffu, ok)) break;
      const volatile uint32_t* f = infos + at * 8;
      if (f[4]) break;
      const uint32_t word[4] = {f[0], f[1], f[2], f[3]};
      ok = wait_bar<kSuspend>(v_full + 8 * s, static_cast<uint32_t>(i / NS) & 1u, wc,
                              DCNV2_DEVERR_TIMEOUT_PRODUCER);
      if (!__all_sync(0xffffffffu, ok)) break;
      if ((word[0] & word[1] & word[2] & word[3]) != 0xffffffffu) {
#pragma unroll
        for (int x = 0; x < 4; ++x)
          if (!((word[x] >> lane) & 1u)) {
            const uint32_t row = base + LY::kV + s * LY::kTileBytes + (x * 32 + lane) * 128;
            for (int y = 0; y < LY::kBlocks; ++y)
              for (int z = 0; z < 8; ++z)
                ptx::st_shared_v4(row + y * kAttnBlockBytes + z * 16, make_uint4(0, 0, 0, 0));
          }
        ptx::fence_proxy_async_smem();
      }
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(v_ready + 8 * s);
    }
  } else {
    // ------------------------------------------------------------ softmax
    const int rl = (warp & 3) * 32 + lane;  // row of the tile = tensor-memory lane
    {
      // Q rows into the swizzled K-major tile: 16-byte chunks, zeros outside rows and head
      const int q_rows = PAIRED ? kAttnTile / 2 : kAttnTile;   // rows this warpgroup loads
      const int r_first = PAIRED ? w * q_rows : 0;
      uint8_t* tile = smem + LY::kQ + (PAIRED ? 0 : w) * LY::kTileBytes;
      for (int x = static_cast<int>(threadIdx.x) & 127; x < q_rows * (DP / 8); x += 128) {
        const int r = r_first + x / (DP / 8), ch = x % (DP / 8);
        const int row = row0 + (PAIRED ? 0 : w * kAttnTile) + r;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (row < args.rows && ch * 8 < args.D) {
          const int tok = row / args.group, h = g * args.group + row - tok * args.group;
          v = ptx::ld_nc_v4(static_cast<const uint16_t*>(args.q.p) + b * args.q.sb +
                            tok * args.q.st + h * args.q.sh + ch * 8);
        }
        *reinterpret_cast<uint4*>(tile + (ch >> 3) * kAttnBlockBytes + r * 128 +
                                  (((ch & 7) ^ (r & 7)) << 4)) = v;
      }
      ptx::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(q_full);
    }
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;  // this warp's 32 lanes
    const uint32_t t_s = tmem + lanes + kAttnTile * w, t_o = tmem + lanes + 2 * kAttnTile + DP * w;
    for (int turn = 0;; ++turn) {
      const int i = PAIRED ? 2 * turn + w : turn;
      bool ok = wait_bar<kSuspend>(info_full + 8 * (i % NI), static_cast<uint32_t>(i / NI) & 1u,
                                   wc, DCNV2_DEVERR_TIMEOUT_SAMPLER);
      if (!__all_sync(0xffffffffu, ok)) break;
      const volatile uint32_t* f = infos + (i % NI) * 8;
      if (f[4]) break;
      const uint32_t word[4] = {f[0], f[1], f[2], f[3]};
      ok = wait_bar<kSuspend>(s_full + 8 * w, static_cast<uint32_t>(turn) & 1u, wc,
                              DCNV2_DEVERR_TIMEOUT_SAMPLER);
      if (!__all_sync(0xffffffffu, ok)) break;
      ptx::tc_fence_after();
      uint32_t sc[4][32];
#pragma unroll
      for (int x = 0; x < 4; ++x) ptx::tmem_ld_32x32b_x32(t_s + 32 * x, sc[x]);
      ptx::tmem_wait_ld();
#pragma unroll
      for (int x = 0; x < 4; ++x) ptx::tmem_ld_use(sc[x]);
      if ((word[0] & word[1] & word[2] & word[3]) != 0xffffffffu) {
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int y = 0; y < 32; ++y)
            if (!((word[x] >> y) & 1u)) sc[x][y] = 0xff800000u;  // -inf
      }
      float top[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        top[x] = __uint_as_float(sc[x][0]);
#pragma unroll
        for (int y = 1; y < 32; ++y) top[x] = fmaxf(top[x], __uint_as_float(sc[x][y]));
      }
      const float m = fmaxf(m_ref, fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])));
      // (-inf) - (-inf) is NaN, which is not greater
      if (__any_sync(0xffffffffu, (m - m_ref) * c > kAttnLazy)) {
        const float fac = m == m_ref ? 1.f : ptx::ex2((m_ref - m) * c);
        l *= fac;
        m_ref = m;
        if (turn > 0) {
          // these scores were issued behind the last product, and have arrived: O is complete
          for (int x = 0; x < args.D; x += 16) {
            uint32_t o[16];
            ptx::tmem_ld_32x32b_x16(t_o + x, o);
            ptx::tmem_wait_ld_regs(o);
#pragma unroll
            for (int y = 0; y < 16; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * fac);
            ptx::tmem_st_32x32b_x16(t_o + x, o);
          }
        }
      }
      const float neg = (m_ref == -INFINITY ? 0.f : -m_ref * c) + shift;
      const float2 c2 = make_float2(c, c), n2 = make_float2(neg, neg);
      float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        uint32_t pk[16];
#pragma unroll
        for (int y = 0; y < 16; ++y) {
          const float2 e = ptx::fma2(make_float2(__uint_as_float(sc[x][2 * y]),
                                                 __uint_as_float(sc[x][2 * y + 1])), c2, n2);
          const float2 p = make_float2(ptx::ex2(e.x), ptx::ex2(e.y));
          sum[y & 1] = ptx::add2(sum[y & 1], p);
          pk[y] = ptx::pack16<BF16>(p.x, p.y);
        }
        ptx::tmem_st_32x32b_x16(t_s + 16 * x, pk);
      }
      l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
      ptx::tmem_wait_st();
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(p_ready + 8 * w);
    }
    // all products of both warpgroups are done: O is complete, the buffers are free
    const bool done = wait_bar<kSuspend>(o_final, 0, wc, DCNV2_DEVERR_TIMEOUT_EPILOGUE);
    if (!__all_sync(0xffffffffu, done)) l = NAN;  // shows in the result, beside the error word
    ptx::tc_fence_after();
    const int row = row0 + (PAIRED ? 0 : w * kAttnTile) + rl;
    if (!PAIRED && args.split == 1) {
      // ---------------------------------------------------------- epilogue without a join
      const int tok = row / args.group, h = g * args.group + row - tok * args.group;
      const float inv = 1.f / l;
      uint16_t* o = static_cast<uint16_t*>(const_cast<void*>(args.o.p)) + b * args.o.sb +
                    tok * args.o.st + h * args.o.sh;
      for (int x = 0; x < args.D; x += 16) {
        uint32_t r[16];
        ptx::tmem_ld_32x32b_x16(t_o + x, r);
        ptx::tmem_wait_ld_regs(r);
        if (row < args.rows) {
          uint32_t pk[8];
#pragma unroll
          for (int y = 0; y < 8; ++y)
            pk[y] = l == 0.f ? 0u
                             : ptx::pack16<BF16>(__uint_as_float(r[2 * y]) * inv,
                                                 __uint_as_float(r[2 * y + 1]) * inv);
          *reinterpret_cast<uint4*>(o + x) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
          if (x + 8 < args.D)
            *reinterpret_cast<uint4*>(o + x + 8) = make_uint4(pk[4], pk[5], pk[6], pk[7]);
        }
      }
      if (args.lse && row < args.rows)
        args.lse[(static_cast<int64_t>(b) * args.H + h) * args.L + tok] =
            l == 0.f ? -INFINITY : kLn2 * (m_ref * c - shift + log2f(l));
    } else {
      // ---------------------------------------------------------- part of this warpgroup
      if (row < args.rows) {
        *reinterpret_cast<float2*>(smem + LY::kQ + (w * kAttnTile + rl) * 8) =
            make_float2(m_ref, l);
      }
      uint8_t* part = smem + LY::kPart + w * LY::kPartBytes;
      for (int x = 0; x < args.D; x += 16) {
        uint32_t r[16];
        ptx::tmem_ld_32x32b_x16(t_o + x, r);
        ptx::tmem_wait_ld_regs(r);
        if (row < args.rows)
#pragma unroll
          for (int y = 0; y < 4; ++y)
            *reinterpret_cast<uint4*>(part + attn_part_at<DP>(rl, x / 4 + y)) =
                make_uint4(r[4 * y], r[4 * y + 1], r[4 * y + 2], r[4 * y + 3]);
      }
    }
    ptx::tc_fence_before();
  }

  if (PAIRED || args.split > 1) {
    // ------------------------------------------------------------ join of the parts
    ptx::cluster_sync();
    if (warp < 8) {
      // an item is 8 elements of a row; the CTAs of the cluster take turns
      const int chunks = args.D / 8;
      const int n_rows = min(args.rows - row0, PAIRED ? kAttnTile : 2 * kAttnTile);
      for (int x = rank * 256 + static_cast<int>(threadIdx.x); x < n_rows * chunks;
           x += args.split * 256) {
        const int r = x / chunks, ch = x - r * chunks;
        const int rt = r & (kAttnTile - 1);
        const int w0 = PAIRED ? 0 : r / kAttnTile, w1 = PAIRED ? 2 : w0 + 1;
        float top = -INFINITY;
        for (int y = 0; y < args.split; ++y)
          for (int z = w0; z < w1; ++z) {
            const float2 ml = ptx::ld_cluster_f2(
                ptx::mapa_shared(base + LY::kQ + (z * kAttnTile + rt) * 8, y));
            top = fmaxf(top, ml.x);
          }
        float total = 0.f, acc[8] = {};
        for (int y = 0; y < args.split; ++y)
          for (int z = w0; z < w1; ++z) {
            const float2 ml = ptx::ld_cluster_f2(
                ptx::mapa_shared(base + LY::kQ + (z * kAttnTile + rt) * 8, y));
            if (ml.y == 0.f) continue;  // no kept state: its O was never written
            const float f = ml.x == top ? 1.f : ptx::ex2((ml.x - top) * c);
            total = fmaf(ml.y, f, total);
            const uint32_t at = base + LY::kPart + z * LY::kPartBytes;
            const float4 lo = ptx::ld_cluster_f4(
                ptx::mapa_shared(at + attn_part_at<DP>(rt, 2 * ch), y));
            const float4 hi = ptx::ld_cluster_f4(
                ptx::mapa_shared(at + attn_part_at<DP>(rt, 2 * ch + 1), y));
            acc[0] = fmaf(lo.x, f, acc[0]); acc[1] = fmaf(lo.y, f, acc[1]);
            acc[2] = fmaf(lo.z, f, acc[2]); acc[3] = fmaf(lo.w, f, acc[3]);
            acc[4] = fmaf(hi.x, f, acc[4]); acc[5] = fmaf(hi.y, f, acc[5]);
            acc[6] = fmaf(hi.z, f, acc[6]); acc[7] = fmaf(hi.w, f, acc[7]);
          }
        const int row = row0 + r, tok = row / args.group;
        const int h = g * args.group + row - tok * args.group;
        const float inv = total == 0.f ? 0.f : 1.f / total;
        uint32_t pk[4];
#pragma unroll
        for (int y = 0; y < 4; ++y)
          pk[y] = ptx::pack16<BF16>(acc[2 * y] * inv, acc[2 * y + 1] * inv);
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(const_cast<void*>(args.o.p)) +
                                  b * args.o.sb + tok * args.o.st + h * args.o.sh + ch * 8) =
            make_uint4(pk[0], pk[1], pk[2], pk[3]);
        if (args.lse && ch == 0)
          args.lse[(static_cast<int64_t>(b) * args.H + h) * args.L + tok] =
              total == 0.f ? -INFINITY : kLn2 * (top * c - shift + log2f(total));
      }
    }
    ptx::cluster_sync();  // the parts stay until every CTA has read them
  }
  __syncthreads();
  if (warp == kAttnMmaWarp) {
    __syncwarp();
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, 512);
  }
}

}  // namespace dcnv2
