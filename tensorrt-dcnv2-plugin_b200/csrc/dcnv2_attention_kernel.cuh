// dcnv2_attention_kernel.cuh — attention of queries to the states of another sequence, on tensor
// cores, in one pass over the states.
//
// For query row i of a sequence and its kept states j: s_ij = scale q_i k_j, m = max s, p = exp(s -
// m), out_i = sum p v / sum p, lse_i = m + log sum p; without kept states out = 0, lse = -inf.
//
// Rows: the queries of one kv head, token by token, the heads of its group side by side, so
// that grouped heads fill an MMA's 128 rows together and read each state once: a tile is as
// many whole tokens as fit. (Groups of more than 128 heads are cut into equal parts that read
// the states each for itself.) Q comes and O goes as TMA boxes of such a tile; what lies behind
// the last token reads as zeros and is not written. Per tile of states: S[128 rows, states] = Q
// K^T into tensor memory; each softmax thread owns a row, reads its scores, writes the rounded
// probabilities back as the A operand; O[128, D] += P V accumulates in tensor memory. The
// running maximum is followed lazily: O and the row's sum are rescaled only when it has grown
// by more than 2^8 (probabilities up to 2^8 are as exact as those up to 1, and the sums are
// fp32), so that most tiles touch O only through the MMA. The probabilities are summed as
// computed and rounded once, to the inputs' type, for the product, beside the output's own
// rounding: an MMA takes both operands in one type, and fp32 ones (tf32) would need V converted
// and run at half the rate. Error against 64 bits (2-norm): bf16 0.0023, fp16 0.00029, where the
// output's rounding alone makes 0.0017 and 0.00021.
//
// Softmax warpgroups share the state tiles, so that the exponentials of some overlap the MMAs
// of the others:
//   PAIRED = false  two tiles of 128 rows per item and tiles of 128 states, or, for heads of up to
//                   64 elements, four and 64: S and O of all of them fill tensor memory either way
//                   (300 queries x 5456 states, heads of 32, 32 images: four warpgroups 260 us, two
//                   297 us). A CTA takes items (sequence, group, rows) in turn;
//   PAIRED = true   one tile of rows, two warpgroups take the even and the odd state tiles (few
//                   rows: some tokens, grouped heads), and their halves are joined at the end.
// A cluster of CTAs may split the states of one item; the parts (fp32 O, maximum, sum) are
// joined through distributed shared memory, every CTA finishing a share of the rows: no second
// launch, no workspace, and the order of the sums is fixed.
//
// Roles: the softmax warpgroups (which also finish the rows), then a warp each for: the
// producer (kept-state words of each tile, TMA of K and V; tiles without a kept state are left
// out altogether), zeroing the V rows of states that are not kept (their probability is 0, but
// 0 * NaN is not), and one or two issuers of MMAs (and of the loads of Q). Warps whose rows lie
// behind the last query skip their exponentials. Every wait is bounded; where one runs out, the
// CTA's rows (the cluster's item) become NaN.
//
// Bound: at heads of 128, two row tiles times 128 states take 2756 cycles of MMAs (S, both
// operands from shared memory: 102 cycles per 128 x 128 x 16; P V: 70) and 2048 of exponentials
// (16 per clock and SM), and the chain of one row tile S -> P -> O -> next S takes 3250;
// measured about 3680: 16 heads, 4096 x 16384: 541 us, 1.02 PFLOP/s (503 at best, 554-565 with
// inputs that change from call to call), tensor pipe and exponentials 56 % busy each; 256 items on
// 148 SMs are two rounds for 1.73 of work. At heads of 32 the MMAs are a quarter of that, and the
// issuing warps' instructions (about 1150 cycles per row tile and 64 states: waits, six MMAs,
// commits) and the softmax's set the time (260 us above: exponential unit 44 % busy, issue slots 46
// %).
// One tile of rows (PAIRED), 32 rows of 8 kv heads of 128, 8 x 60001 states: 311 us, 6.3 TB/s;
// 17 rows, 8 heads of 32, 32 x 5456: 85 us; 64 heads on one kv head, 8 x 60001: 81 us, 3.0 TB/s (64
// CTAs).
// Tried and slower: a polynomial on the FMA units for 1/8 to 3/8 of the exponentials (575 ->
// 622-644 us: the issue slots are scarce too), one issuer per warpgroup at heads of 128 (656
// us: they fall into step), scores a tile ahead with the probabilities beside them (heads of
// 128: 535 -> 548 us, heads of 32: 297 -> 359 us), three warpgroups with two sets of scores each
// for heads of 32 (300 queries: 251 us, but 512 queries take 1.8 times as long).
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <climits>

#include "../../include/dcnv2.h"
#include "dcnv2_wait.cuh"
#include "ptx_sm100.cuh"

namespace dcnv2 {

constexpr int kAttnTile = 128;                 // rows of a tile (MMA M, tensor-memory lanes)
constexpr uint32_t kAttnBlockBytes = kAttnTile * 128;  // 128 rows of one 128-byte swizzle block
constexpr int kAttnMaxSplit = 8;               // CTAs of a cluster (portable size)
constexpr float kAttnLazy = 8.f;               // log2 of the growth that rescales
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct AttnTensor {
  const void* p;
  int64_t sb, st, sh;                          // strides: batch, token, head (elements)
};

struct AttnArgs {
  const int* kv_lens;
  const uint8_t* key_mask;
  int64_t mask_sb;
  float* lse;                                  // [B][H][L] or null
  void* out;                                   // (joined parts are stored directly)
  int64_t out_sb, out_st, out_sh;
  int* err;                                    // one word per CTA
  int L, S, H, D;
  int heads;                                   // query heads of a tile's token
  int kv_parts;                                // parts of a kv head's group
  int groups;                                  // kv heads * kv_parts
  int tile_tokens;                             // 128 / heads
  int row_tiles;                               // items along the rows
  int items;                                   // (sequence, group, row tile)
  int split;                                   // CTAs of a cluster along the states
  int q_batch;                                 // 0: the sequences share the queries
  int k_batch, k_head, v_batch, v_head;        // 0: the tensor is shared along that axis
  float scale;
  unsigned long long timeout_ns;
};

// Shared-memory layout of an instance (bytes from a 1024-aligned base).
template <int DP, bool PAIRED>
struct AttnLayout {
  // softmax warpgroups, and states per tile: S and O of all of them fill tensor memory
  static constexpr int kWGs = !PAIRED && DP == 64 ? 4 : 2;
  static constexpr int kN = 256 / kWGs;
  static constexpr int kWords = kN / 32;                          // kept-state words of a tile
  static constexpr int kThreads = (kWGs + 1) * 128;
  static constexpr int kProducerWarp = kWGs * 4, kFixWarp = kProducerWarp + 1,
                       kMmaWarp = kProducerWarp + 2;              // and the next, of kIssuers = 2
  static constexpr int kIssuers = kWGs / 2;                       // each for two warpgroups
  static constexpr int kBlocks = DP / 64;                         // swizzle blocks of a row
  static constexpr uint32_t kTileBytes = kBlocks * kAttnBlockBytes;  // of Q or O
  static constexpr uint32_t kStateBlock = kN * 128;
  static constexpr uint32_t kStateBytes = kBlocks * kStateBlock;  // of K or V
  static constexpr int kQTiles = PAIRED ? 1 : kWGs;
  static constexpr int kStages = DP == 128 ? (PAIRED ? 3 : 2) : 6;
  static constexpr int kInfos = kStages + 2;
  // O on its way out: beside Q, or, where shared memory is short, over it
  static constexpr bool kOutBeside = !PAIRED && DP == 64;
  static constexpr uint32_t kQ = 0;
  static constexpr uint32_t kK = kQTiles * kTileBytes;
  static constexpr uint32_t kV = kK + kStages * kStateBytes;
  static constexpr uint32_t kOut = kOutBeside ? kV + kStages * kStateBytes : kQ;
  static constexpr uint32_t kInfo =                               // kInfos x 32 bytes
      kV + kStages * kStateBytes + (kOutBeside ? kWGs * kTileBytes : 0);
  static constexpr uint32_t kBars = kInfo + kInfos * 32;
  static constexpr int kNumBars = 5 * kStages + 2 * kInfos + 5 * kWGs + kIssuers;
  static constexpr uint32_t kDrain = kBars + (kNumBars - kIssuers) * 8;  // the MMA issuers' own
  static constexpr uint32_t kFlags = kBars + kNumBars * 8;        // [kStages] of the K tiles
  static constexpr uint32_t kSlot = kFlags + kStages * 4;         // TMEM address, abort flag, steps
  static constexpr uint32_t kBytes = kSlot + 16;
  // at the end, over K, V and what follows: fp32 O of the warpgroups; over Q: their (maximum, sum)
  static constexpr uint32_t kPart = kK;
  static constexpr uint32_t kPartBytes = kAttnTile * DP * 4;
  static_assert(kPart + kWGs * kPartBytes <= kInfo, "parts fit over K, V and O");
  static constexpr uint32_t kShare = kQ + kWGs * kAttnTile * 8;  // [row][part] factors, behind
  static_assert(kShare + kQTiles * kAttnTile * (PAIRED ? 2 : 1) * kAttnMaxSplit * 4 <= kK,
                "statistics and shares fit over Q");
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

// What the producer says of a tile, beside its kept-state words.
constexpr uint32_t kInfoLast = 1;   // the item's last tile
constexpr uint32_t kInfoEmpty = 2;  // no tile: the item has no kept state
// What it says of a K tile: kInfoLast, or that no tile comes any more; times kTileSkip, the items
// without a tile that were passed over.
constexpr uint32_t kTileEnd = 2, kTileSkip = 4;

template <int DP, bool PAIRED, bool BF16>
__global__ void __launch_bounds__((AttnLayout<DP, PAIRED>::kThreads), 1)
    dcnv2_cross_attention_kernel(const __grid_constant__ AttnArgs args,
                                 const __grid_constant__ CUtensorMap tmap_q,
                                 const __grid_constant__ CUtensorMap tmap_k,
                                 const __grid_constant__ CUtensorMap tmap_v,
                                 const __grid_constant__ CUtensorMap tmap_o) {
  using LY = AttnLayout<DP, PAIRED>;
  constexpr int NS = LY::kStages, NI = LY::kInfos, WG = LY::kWGs, N = LY::kN, NW = LY::kWords;
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
  const uint32_t info_full = v_empty + 8 * NS;         // [NI] words and flags of a tile
  const uint32_t info_empty = info_full + 8 * NI;      // [NI] read by everyone
  const uint32_t s_full = info_empty + 8 * NI;         // [WG] scores of warpgroup w
  const uint32_t p_ready = s_full + 8 * WG;            // [WG] its probabilities
  const uint32_t q_full = p_ready + 8 * WG;            // [WG] Q tile of warpgroup w
  const uint32_t q_empty = q_full + 8 * WG;            // [WG] its last scores done, O has left
  const uint32_t o_full = q_empty + 8 * WG;            // [WG] O of warpgroup w complete
  uint32_t* slot = reinterpret_cast<uint32_t*>(smem + LY::kSlot);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(slot + 1);
  uint32_t* infos = reinterpret_cast<uint32_t*>(smem + LY::kInfo);  // words 0-3, flags
  const WaitCtx wc{args.timeout_ns, args.err + blockIdx.x, abort_flag};
  // Waits for the producer, which may have to search one long mask after another
  volatile int* producer_steps = abort_flag + 1;
  const WaitCtx wp{args.timeout_ns, args.err + blockIdx.x, abort_flag, producer_steps};

  // A cluster of `split` CTAs takes the items cluster, cluster + clusters, ... (one item each when
  // split or PAIRED); item = (sequence * groups + group) * row_tiles + row tile.
  const int rank = static_cast<int>(blockIdx.x) % args.split;
  const int item0 = static_cast<int>(blockIdx.x) / args.split;
  const int item_step = static_cast<int>(gridDim.x) / args.split;
  struct Item {
    int tok0, g, b;  // first token, group, sequence
  };
  auto item_at = [&](int item) {
    Item it;
    it.tok0 = (item % args.row_tiles) * args.tile_tokens * LY::kQTiles;
    const int rest = item / args.row_tiles;
    it.g = rest % args.groups;
    it.b = rest / args.groups;
    return it;
  };
  // rows of warpgroup w's tile of the item (0: none)
  auto rows_of = [&](const Item& it, int w) {
    const int left = args.L - it.tok0 - (PAIRED ? 0 : w * args.tile_tokens);
    return max(0, min(args.tile_tokens, left)) * args.heads;
  };

  if (threadIdx.x == 0) {
    for (int i = 0; i < NS; ++i) {
      ptx::mbar_init(k_full + 8 * i, 1);
      ptx::mbar_init(k_empty + 8 * i, LY::kIssuers);
      ptx::mbar_init(v_full + 8 * i, 1);
      ptx::mbar_init(v_ready + 8 * i, 1);
      ptx::mbar_init(v_empty + 8 * i, LY::kIssuers);
    }
    for (int i = 0; i < NI; ++i) {
      ptx::mbar_init(info_full + 8 * i, 1);
      ptx::mbar_init(info_empty + 8 * i, WG * 4 + 1);  // softmax warps, V fixer
    }
    for (int i = 0; i < WG; ++i) {
      ptx::mbar_init(s_full + 8 * i, 1);
      ptx::mbar_init(p_ready + 8 * i, 4);
      ptx::mbar_init(q_full + 8 * i, 1);
      ptx::mbar_init(q_empty + 8 * i, 1);
      ptx::mbar_init(o_full + 8 * i, 1);
    }
    for (int i = 0; i < LY::kIssuers; ++i) ptx::mbar_init(base + LY::kDrain + 8 * i, 1);
    *abort_flag = *producer_steps = 0;
    ptx::fence_mbar_init();
  }
  if (warp == LY::kMmaWarp) {
    ptx::tmem_alloc(ptx::smem_addr(slot), 512);
    ptx::tmem_relinquish();
  }
  // (not before tensor memory is taken, which a kernel that starts behind this one may want too)
  ptx::griddep_launch_dependents();
  // the setup above overlaps the tail of the kernel ahead; memory is touched only from here
  ptx::griddep_wait();
  if (threadIdx.x == 0) *wc.err = 0;
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = *slot;
  // tensor memory: scores of warpgroup w at N w (the probabilities over their first half), its O at
  // 256 + DP w
  const int w = warp >> 2;  // softmax warpgroup
  const float c = args.scale * kLog2e;
  // fp16 probabilities are scaled by 2^7 (at most 2^15): small ones keep their bits longer
  const float shift = BF16 ? 0.f : 7.f;

  // Reads entry n of the producer's ring: words of the tile and flags. False after an abort.
  auto read_info = [&](int n, uint32_t (&word)[NW], uint32_t& flags, int code) {
    const bool ok = wait_bar<kSuspend>(info_full + 8 * (n % NI),
                                       static_cast<uint32_t>(n / NI) & 1u, wp, code);
    if (!__all_sync(0xffffffffu, ok)) return false;
    const uint4 f = ptx::ld_shared_v4(base + LY::kInfo + (n % NI) * 32);
    word[0] = f.x;
    word[1] = f.y;
    if constexpr (NW == 4) {
      word[2] = f.z;
      word[3] = f.w;
    }
    flags = ptx::ld_shared_u32_volatile(base + LY::kInfo + (n % NI) * 32 + 16);
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(info_empty + 8 * (n % NI));
    return true;
  };

  // two softmax warpgroups: 384 threads x 168 registers at launch cover 256 x 192 + 128 x 120;
  // four: 640 x 96 cover 512 x 104 + 128 x 64
  if (warp >= LY::kProducerWarp) {
  if constexpr (WG == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 120;");
  else asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
  if (warp == LY::kProducerWarp) {
    // ------------------------------------------------------------ producer
    int n = 0, i = 0;                    // ring entries, tiles
    uint32_t fetches = 0;                // of masks
    uint32_t steps = 0;                  // lane 0: what it has told the waiting ones
    uint32_t skipped = 0;                // items without a tile since the last one with tiles
    volatile uint32_t* tile_flags = reinterpret_cast<volatile uint32_t*>(smem + LY::kFlags);
    bool ok = true, k_ahead = false;     // k_ahead: K of tile i was started, V was not
    for (int item = item0; item < args.items && ok; item += item_step) {
      const Item it = item_at(item);
      int len = args.S;
      if (args.kv_lens) len = max(0, min(len, __ldg(args.kv_lens + it.b)));
      const int tiles = (len + N - 1) / N;
      const int t1 = static_cast<int>(static_cast<int64_t>(tiles) * (rank + 1) / args.split);
      int t = static_cast<int>(static_cast<int64_t>(tiles) * rank / args.split);
      const uint8_t* mask = args.key_mask ? args.key_mask + it.b * args.mask_sb : nullptr;
      // The mask is read kAhead words (256 states) at a time, the next ones on their way, so that
      // runs of tiles without a kept state pass at a few hundred cycles per load, not per tile.
      constexpr int kAhead = 8;
      constexpr uint32_t kStepFetches = (1u << 24) / (32 * kAhead);  // 2^24 states: about 25 ms
      uint8_t next[kAhead];              // the lane's bytes
      uint32_t words[kAhead] = {};
      int left_words = 0;
      auto fetch = [&](int tile) {
#pragma unroll
        for (int x = 0; x < kAhead; ++x) {
          const int64_t j = static_cast<int64_t>(tile) * N + x * 32 + lane;
          next[x] = tile < t1 && j < len ? __ldg(mask + j) : 0;
        }
      };
      // the next tile with a kept state from t on (t moves behind it), or -1
      auto find = [&](uint32_t (&word)[NW]) {
        for (; t < t1; ++t) {
          if (!mask) {
#pragma unroll
            for (int x = 0; x < NW; ++x) {
              const int left = len - t * N - x * 32;
              word[x] = left >= 32 ? 0xffffffffu : left <= 0 ? 0u : (1u << left) - 1u;
            }
            return t++;
          }
          if (left_words == 0) {
#pragma unroll
            for (int x = 0; x < kAhead; ++x)
              words[x] = __ballot_sync(0xffffffffu, next[x] != 0);
            left_words = kAhead;
            if (++fetches % kStepFetches == 0 && lane == 0) *producer_steps = ++steps & INT_MAX;
            fetch(t + kAhead / NW);
          }
#pragma unroll
          for (int x = 0; x < NW; ++x) word[x] = words[x];
#pragma unroll
          for (int x = 0; x + NW < kAhead; ++x) words[x] = words[x + NW];
          left_words -= NW;
          uint32_t some = 0;
#pragma unroll
          for (int x = 0; x < NW; ++x) some |= word[x];
          if (some) return t++;
        }
        return -1;
      };
      if (mask) fetch(t);
      uint32_t word[NW] = {}, word_next[NW];
      int tile = find(word);
      uint32_t flags = tile < 0 ? (kInfoEmpty | kInfoLast) : 0;
      do {
        const int tile_next = tile < 0 ? -1 : find(word_next);
        if (tile_next < 0) flags |= kInfoLast;
        const int s = i % NS, at = n % NI;
        const uint32_t ph = static_cast<uint32_t>(i / NS) & 1u;
        if (lane == 0) {
          ok = wait_bar<kSuspend>(info_empty + 8 * at, (static_cast<uint32_t>(n / NI) & 1u) ^ 1u,
                                  wc, DCNV2_DEVERR_TIMEOUT_PRODUCER);
          if (ok) {
            uint32_t* f = infos + at * 8;
#pragma unroll
            for (int x = 0; x < NW; ++x) f[x] = word[x];
            f[4] = flags;
            *producer_steps = ++steps & INT_MAX;
            ptx::mbar_arrive(info_full + 8 * at);
            if (tile >= 0)
              ok = wait_bar<kSuspend>(k_empty + 8 * s, ph ^ 1u, wc,
                                      DCNV2_DEVERR_TIMEOUT_PRODUCER);
          }
          if (ok && tile >= 0) {
            tile_flags[s] = (flags & kInfoLast) + skipped * kTileSkip;
            ptx::mbar_arrive_expect_tx(k_full + 8 * s, LY::kStateBytes);
            for (int x = 0; x < LY::kBlocks; ++x)
              ptx::tma_load_4d(base + LY::kK + s * LY::kStateBytes + x * LY::kStateBlock, &tmap_k,
                               x * 64, tile * N, (it.g / args.kv_parts) * args.k_head,
                               it.b * args.k_batch,
                               k_full + 8 * s);
            k_ahead = true;
            ok = wait_bar<kSuspend>(v_empty + 8 * s, ph ^ 1u, wc, DCNV2_DEVERR_TIMEOUT_PRODUCER);
            if (ok) {
              ptx::mbar_arrive_expect_tx(v_full + 8 * s, LY::kStateBytes);
              for (int x = 0; x < LY::kBlocks; ++x)
                ptx::tma_load_4d(base + LY::kV + s * LY::kStateBytes + x * LY::kStateBlock,
                                 &tmap_v, x * 64, tile * N,
                                 (it.g / args.kv_parts) * args.v_head, it.b * args.v_batch,
                                 v_full + 8 * s);
              k_ahead = false;
            }
          }
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
        if (!ok) break;
        ++n;
        skipped = tile >= 0 ? 0 : skipped + 1;
        if (tile >= 0) ++i;
        tile = tile_next;
        flags = 0;
#pragma unroll
        for (int x = 0; x < NW; ++x) word[x] = word_next[x];
      } while (tile >= 0);
    }
    if (lane == 0) {
      const int k_tiles = i + (k_ahead ? 1 : 0);
      int k_marks = k_tiles;             // K barriers' phases: the tiles, and the end's mark
      if (ok && wait_bar<kSuspend>(k_empty + 8 * (i % NS),
                                   (static_cast<uint32_t>(i / NS) & 1u) ^ 1u, wc,
                                   DCNV2_DEVERR_TIMEOUT_PRODUCER)) {
        tile_flags[i % NS] = kTileEnd;
        ptx::mbar_arrive(k_full + 8 * (i % NS));
        ++k_marks;
      }
      // Copies in flight land before the CTA ends or its buffers are used for the parts. (Only a
      // barrier's last phase can be waited for; a copy whose place another has taken has landed.)
      for (int x = k_marks > NS ? k_marks - NS : 0; x < k_tiles; ++x)
        drain_bar(k_full + 8 * (x % NS), static_cast<uint32_t>(x / NS) & 1u, wc);
      for (int x = i > NS ? i - NS : 0; x < i; ++x)
        drain_bar(v_full + 8 * (x % NS), static_cast<uint32_t>(x / NS) & 1u, wc);
    }
  } else if (warp >= LY::kMmaWarp && warp < LY::kMmaWarp + LY::kIssuers) {
    // ------------------------------------------------------------ MMA issuer
    // The warp runs this code as a whole, one elected lane issues. As little as possible stands
    // between the arrival of probabilities and the MMAs they release: what the next tile is, and
    // that its K is there, is found out while the softmax works. One issuer serves two warpgroups
    // in turn, which keeps them apart: with one each they fall into step, and MMAs and exponentials
    // wait for each other.
    const int m = warp - LY::kMmaWarp, wg0 = 2 * m;  // its first warpgroup
    constexpr uint32_t fmt = BF16 ? ptx::kFmtBf16 : 0;
    const bool leader = ptx::elect_one();
    const uint32_t id_s = ptx::make_idesc(1, fmt, N);
    const uint32_t id_o =
        ptx::make_idesc(1, fmt, static_cast<uint32_t>((args.D + 15) / 16 * 16)) | ptx::kIdescBMn;
    const int d_steps = (args.D + 15) / 16;
    const uint64_t q_desc = ptx::sw128_kmajor_desc(base + LY::kQ);
    const uint64_t k_desc = ptx::sw128_kmajor_desc(base + LY::kK);
    const uint64_t v_desc = ptx::sw128_mnmajor_desc(base + LY::kV, LY::kStateBlock);
    const uint32_t q_lo = static_cast<uint32_t>(q_desc), k_lo = static_cast<uint32_t>(k_desc);
    const uint32_t v_lo = static_cast<uint32_t>(v_desc);
    const uint32_t kd_hi = static_cast<uint32_t>(k_desc >> 32);
    const uint32_t v_hi = static_cast<uint32_t>(v_desc >> 32);
    bool ok = true;
    uint32_t q_loads[WG] = {}, p_turn[WG] = {};
    auto wait = [&](uint32_t bar, uint32_t parity, bool producer = false) {
      const bool got = wait_bar(bar, parity & 1u, producer ? wp : wc, DCNV2_DEVERR_TIMEOUT_MMA);
      return ok = __all_sync(0xffffffffu, ok && got);
    };
    auto commit = [&](uint32_t bar) {
      if (leader) ptx::tc_commit(bar);
    };
    auto load_q = [&](const Item& it, int wg) {
      if (leader) {
        const uint32_t rows = args.tile_tokens * args.heads;  // of the box
        const uint32_t to = base + LY::kQ + wg * LY::kTileBytes;
        ptx::mbar_arrive_expect_tx(q_full + 8 * wg, LY::kBlocks * rows * 128);
        for (int x = 0; x < LY::kBlocks; ++x)
          ptx::tma_load_5d(to + x * kAttnBlockBytes, &tmap_q, x * 64, 0,
                           it.tok0 + wg * args.tile_tokens, it.g, it.b * args.q_batch,
                           q_full + 8 * wg);
      }
      ++q_loads[wg];
    };
    // tile i: whether there is one (its K is there then), and of which item
    int item = item0;
    Item it = item_at(item0);
    bool begun = false, fresh = true, last = true;
    int active = 0;  // warpgroups with rows of the item
    auto next_tile = [&](int i) {
      if (!wait(k_full + 8 * (i % NS), i / NS, true)) return false;
      const uint32_t flags = ptx::ld_shared_u32_volatile(base + LY::kFlags + (i % NS) * 4);
      fresh = last;
      last = (flags & kInfoLast) != 0;
      if (flags & kTileEnd) return false;
      if (fresh) {
        item += item_step * static_cast<int>(flags / kTileSkip + (begun ? 1 : 0));
        it = item_at(item);
        begun = true;
        for (active = 0; active < LY::kQTiles && rows_of(it, active) > 0;) ++active;
      }
      return true;
    };
    auto scores = [&](int i, int wg) {  // S of warpgroup wg from K tile i
      const uint32_t q = q_lo + (PAIRED ? 0 : wg) * (LY::kTileBytes >> 4);
      const uint32_t k = k_lo + (i % NS) * (LY::kStateBytes >> 4);
      const uint32_t d = tmem + N * wg;
      ptx::tc_fence_after();
      if (leader) {
        ptx::mma_f16_run<false>(d, q, kd_hi, k, kd_hi, id_s);
#pragma unroll
        for (int x = 1; x < DP / 16; ++x) {
          const uint32_t q_off = (x >> 2) * (kAttnBlockBytes >> 4) + (x & 3) * 2;
          const uint32_t k_off = (x >> 2) * (LY::kStateBlock >> 4) + (x & 3) * 2;
          if (x < d_steps) ptx::mma_f16_run<true>(d, q + q_off, kd_hi, k + k_off, kd_hi, id_s);
        }
        ptx::tc_commit(s_full + 8 * wg);
      }
      __syncwarp();
    };
    auto product = [&](int i, int wg, bool first) {  // O of warpgroup wg += P V tile i
      if (!wait(p_ready + 8 * wg, p_turn[wg]++)) return false;
      ptx::tc_fence_after();
      const uint32_t v = v_lo + (i % NS) * (LY::kStateBytes >> 4);
      const uint32_t d = tmem + 256 + DP * wg, p = tmem + N * wg;
      if (leader) {
#pragma unroll
        for (int x = 0; x < N / 16; ++x)
          ptx::mma_f16_ta_run(d, p + 8 * x, v + x * (2048 >> 4), v_hi, id_o,
                              x > 0 ? 1u : first ? 0u : 1u);
      }
      __syncwarp();
      return true;
    };
    // A warpgroup's next scores are issued right behind its product, whose probabilities they
    // overwrite: the tensor core runs MMAs in the order of issue.
    if constexpr (PAIRED) {
      int have = 0;       // tiles found
      bool ended = false;
      auto more = [&](int upto) {
        while (ok && !ended && have < upto) {
          if (next_tile(have)) ++have;
          else ended = true;
        }
        return have >= upto;
      };
      load_q(it, 0);
      wait(q_full, 0);
      for (int i = 0; i < 2; ++i)
        if (more(i + 1)) {
          scores(i, i);
          commit(k_empty + 8 * (i % NS));
        }
      for (int i = 0; ok && i < have; ++i) {
        const bool next = more(i + 3);
        if (!wait(v_ready + 8 * (i % NS), i / NS) || !product(i, i & 1, i < 2)) break;
        if (next) scores(i + 2, i & 1);
        commit(v_empty + 8 * (i % NS));
        if (next) commit(k_empty + 8 * ((i + 2) % NS));
      }
      commit(o_full);
      commit(o_full + 8);
    } else {
      bool have = next_tile(0);
      if (have)
        for (int wg = wg0; wg < min(active, wg0 + 2); ++wg) load_q(it, wg);
      int i = 0;
      while (have && ok) {  // an item begins: its Q is on its way
        const int end = min(active, wg0 + 2);  // of its warpgroups with rows
        if (end <= wg0) {  // none: keep step with the tiles
          const bool ends = last;
          if (leader) ptx::mbar_arrive(k_empty + 8 * (i % NS));
          if (!wait(v_full + 8 * (i % NS), i / NS)) break;
          if (leader) ptx::mbar_arrive(v_empty + 8 * (i % NS));
          have = next_tile(++i);
          if (have && ends)
            for (int wg = wg0; wg < min(active, wg0 + 2); ++wg) load_q(it, wg);
          continue;
        }
        for (int wg = wg0; wg < end; ++wg)
          if (wait(q_full + 8 * wg, q_loads[wg] - 1)) scores(i, wg);
        commit(k_empty + 8 * (i % NS));
        bool first = true, ends = false;
        while (ok && !ends) {
          const int cur = i++, at = cur % NS;
          ends = last;
          // Behind an item's end the next tile is looked for after the products: the entries of
          // empty items in between are read by the softmax only when this item's O is complete.
          if (!ends) next_tile(i);
          if (!wait(v_ready + 8 * at, cur / NS)) break;
          for (int wg = wg0; wg < end; ++wg) {
            if (!product(cur, wg, first)) break;
            if (ends) commit(o_full + 8 * wg);
            else scores(i, wg);
          }
          if (!ok) break;
          commit(v_empty + 8 * at);
          if (!ends) commit(k_empty + 8 * (i % NS));
          first = false;
        }
        if (!ok) break;
        have = next_tile(i);
        // the next item's Q: this one's scores are done, and where Q is O's way out, O has left it
        if (have)
          for (int wg = wg0; wg < min(active, wg0 + 2); ++wg) {
            if (!LY::kOutBeside && q_loads[wg] && !wait(q_empty + 8 * wg, q_loads[wg] - 1)) break;
            load_q(it, wg);
          }
      }
    }
    // what is in flight ends before tensor memory and shared memory are given up
    __syncwarp();
    commit(base + LY::kDrain + 8 * m);
    drain_bar(base + LY::kDrain + 8 * m, 0, wc);
    for (int wg = 0; wg < WG; ++wg)
      if (q_loads[wg]) drain_bar(q_full + 8 * wg, (q_loads[wg] - 1) & 1u, wc);
  } else if (warp == LY::kFixWarp) {
    // ------------------------------------------------------------ V rows of unkept states
    int n = 0, i = 0;
    bool ok = true;
    for (int item = item0; item < args.items && ok; item += item_step) {
      uint32_t flags = 0;
      while (ok && !(flags & kInfoLast)) {
        uint32_t word[NW];
        ok = read_info(n, word, flags, DCNV2_DEVERR_TIMEOUT_PRODUCER);
        if (!ok) break;
        ++n;
        if (flags & kInfoEmpty) break;
        const int s = i % NS;
        ok = wait_bar<kSuspend>(v_full + 8 * s, static_cast<uint32_t>(i / NS) & 1u, wc,
                                DCNV2_DEVERR_TIMEOUT_PRODUCER);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        uint32_t whole = 0xffffffffu;
#pragma unroll
        for (int x = 0; x < NW; ++x) whole &= word[x];
        if (whole != 0xffffffffu) {
#pragma unroll
          for (int x = 0; x < NW; ++x)
            if (!((word[x] >> lane) & 1u)) {
              const uint32_t row = base + LY::kV + s * LY::kStateBytes + (x * 32 + lane) * 128;
              for (int y = 0; y < LY::kBlocks; ++y)
                for (int z = 0; z < 8; ++z)
                  ptx::st_shared_v4(row + y * LY::kStateBlock + z * 16, make_uint4(0, 0, 0, 0));
            }
          ptx::fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(v_ready + 8 * s);
        ++i;
      }
    }
  }
  if (PAIRED || args.split > 1) {  // the softmax warps join the parts between these
    __syncwarp();
    ptx::cluster_sync();
    ptx::cluster_sync();
  }
  } else {
    if constexpr (WG == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
    else asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
    // ------------------------------------------------------------ softmax
    const int rl = (warp & 3) * 32 + lane;  // row of the tile = tensor-memory lane
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;  // this warp's 32 lanes
    const uint32_t t_s = tmem + lanes + N * w, t_o = tmem + lanes + 256 + DP * w;
    int n = 0, tile = 0;         // ring entries read; tiles of the item
    uint32_t s_turn = 0, o_turn = 0;
    bool ok = true;
    for (int item = item0; item < args.items && ok; item += item_step) {
      const int n_rows = rows_of(item_at(item), w);
      const bool mine = n_rows > 0;
      const bool rows_here = (warp & 3) * 32 < n_rows;  // else the warp only keeps step
      const bool live = rl < n_rows;
      float m_ref = -INFINITY, l = 0.f;  // this thread's row: reference maximum, sum
      bool first = true, any = false;
      uint32_t flags = 0;
      for (tile = 0; !(flags & kInfoLast); ++tile) {
        uint32_t word[NW];
        ok = read_info(n, word, flags, DCNV2_DEVERR_TIMEOUT_SAMPLER);
        if (!ok) break;
        ++n;
        if (flags & kInfoEmpty) break;
        any = true;
        if (!mine || (PAIRED && (tile & 1) != w)) continue;
        ok = wait_bar<kSuspend>(s_full + 8 * w, s_turn++ & 1u, wc, DCNV2_DEVERR_TIMEOUT_SAMPLER);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        ptx::tc_fence_after();
        if (!rows_here) {
          if (lane == 0) ptx::mbar_arrive(p_ready + 8 * w);
          continue;
        }
        uint32_t sc[NW][32];
#pragma unroll
        for (int x = 0; x < NW; ++x) ptx::tmem_ld_32x32b_x32(t_s + 32 * x, sc[x]);
        ptx::tmem_wait_ld();
#pragma unroll
        for (int x = 0; x < NW; ++x) ptx::tmem_ld_use(sc[x]);
#pragma unroll
        for (int x = 0; x < NW; ++x)
          if (word[x] != 0xffffffffu) {
#pragma unroll
            for (int y = 0; y < 32; ++y)
              if (!((word[x] >> y) & 1u)) sc[x][y] = 0xff800000u;  // -inf
          }
        float top[2 * NW];
#pragma unroll
        for (int x = 0; x < 2 * NW; ++x) {
          const uint32_t* q = &sc[x >> 1][(x & 1) * 16];
          top[x] = fmaxf(__uint_as_float(q[0]), __uint_as_float(q[1]));
#pragma unroll
          for (int y = 2; y < 16; y += 2)
            top[x] = ptx::max3(top[x], __uint_as_float(q[y]), __uint_as_float(q[y + 1]));
        }
#pragma unroll
        for (int x = 2 * NW - 1; x > 1; x -= 2) top[0] = ptx::max3(top[0], top[x], top[x - 1]);
        top[0] = fmaxf(top[0], top[1]);
        const float m = fmaxf(m_ref, top[0]);
        // (-inf) - (-inf) is NaN, which is not greater. Rows behind the tile's last, whose Q is what
        // shared memory held before (boxes of whole tokens may leave some of the 128), have no say:
        // when the others are rescaled would depend on it, and with that their last bits.
        if (__any_sync(0xffffffffu, live && (m - m_ref) * c > kAttnLazy)) {
          const float fac = m == m_ref ? 1.f : ptx::ex2((m_ref - m) * c);
          l *= fac;
          m_ref = m;
          if (!first) {
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
        first = false;
        const float neg = (m_ref == -INFINITY ? 0.f : -m_ref * c) + shift;
        const float2 c2 = make_float2(c, c), n2 = make_float2(neg, neg);
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int x = 0; x < NW; ++x) {
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
        ptx::tmem_wait_st();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(p_ready + 8 * w);
        l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
      }
      if (!mine) {
        // the four warps stay on one item after an abort too: one that left alone would be missing
        // at the next item's barriers
        if (!PAIRED && args.split == 1) ok = ptx::named_barrier_and(1 + w, 128, ok);
        continue;
      }
      // all products of the item are done (both warpgroups' when their parts are joined)
      if (PAIRED || any) {
        bool done = ok && wait_bar<kSuspend>(o_full + 8 * w, o_turn & 1u, wc,
                                             DCNV2_DEVERR_TIMEOUT_EPILOGUE);
        if (PAIRED || args.split > 1)
          for (int x = 0; x < WG; ++x)
            done = done && (rows_of(item_at(item), x) == 0 ||
                            wait_bar<kSuspend>(o_full + 8 * x, o_turn & 1u, wc,
                                               DCNV2_DEVERR_TIMEOUT_EPILOGUE));
        ++o_turn;
        ok = __all_sync(0xffffffffu, done);
        ptx::tc_fence_after();
      }
      if (!PAIRED && args.split == 1) {
        // -------------------------------------------------------- epilogue without a join
        // O / sum in the output's type into the swizzled tile that the TMA store reads; the place
        // is free once the last store from it has been read (beside Q), or Q's last scores are done
        // and its last store has been read (over Q)
        const Item it = item_at(item);
        const uint32_t out = base + LY::kOut + w * LY::kTileBytes;
        const bool storer = (threadIdx.x & 127) == 0;
        if (LY::kOutBeside) {
          if (storer) ptx::bulk_wait_group_read<0>();
          ptx::named_barrier(1 + w, 128);
        }
        const int tok = it.tok0 + w * args.tile_tokens + rl / args.heads;
        const int h = it.g * args.heads + rl % args.heads;
        if (any && rows_here) {
          const float inv = l == 0.f ? 0.f : 1.f / l;
          for (int x = 0; x < args.D; x += 16) {
            uint32_t r[16];
            ptx::tmem_ld_32x32b_x16(t_o + x, r);
            ptx::tmem_wait_ld_regs(r);
            uint32_t pk[8];
#pragma unroll
            for (int y = 0; y < 8; ++y)
              pk[y] = ptx::pack16<BF16>(__uint_as_float(r[2 * y]) * inv,
                                        __uint_as_float(r[2 * y + 1]) * inv);
            const uint32_t at = out + (x >> 6) * kAttnBlockBytes + rl * 128;
            const uint32_t ch = (x & 63) >> 3;
            ptx::st_shared_v4(at + ((ch ^ (rl & 7)) << 4), make_uint4(pk[0], pk[1], pk[2], pk[3]));
            ptx::st_shared_v4(at + (((ch + 1) ^ (rl & 7)) << 4),
                              make_uint4(pk[4], pk[5], pk[6], pk[7]));
          }
        } else if (live) {
          // no kept state: zeros, past the place where the next item's Q may be arriving
          uint16_t* o = static_cast<uint16_t*>(args.out) + it.b * args.out_sb + tok * args.out_st +
                        h * args.out_sh;
          for (int x = 0; x < args.D; x += 8)
            *reinterpret_cast<uint4*>(o + x) = make_uint4(0, 0, 0, 0);
        }
        ptx::tc_fence_before();
        if (args.lse && live)
          args.lse[(static_cast<int64_t>(it.b) * args.H + h) * args.L + tok] =
              l == 0.f ? -INFINITY : kLn2 * (m_ref * c - shift + log2f(l));
        ptx::fence_proxy_async_smem();
        // (after an abort the four warps leave together, behind the same item)
        ok = ptx::named_barrier_and(1 + w, 128, ok);
        if (storer && any && ok) {
          for (int x = 0; x * 64 < args.D; ++x)
            ptx::tma_store_5d(&tmap_o, out + x * kAttnBlockBytes, x * 64, 0,
                              it.tok0 + w * args.tile_tokens, it.g, it.b);
          ptx::bulk_commit_group();
          if (!LY::kOutBeside) {
            ptx::bulk_wait_group_read<0>();
            ptx::mbar_arrive(q_empty + 8 * w);
          }
        }
      } else {
        // -------------------------------------------------------- part of this warpgroup
        if (live)
          *reinterpret_cast<float2*>(smem + LY::kQ + (w * kAttnTile + rl) * 8) =
              make_float2(m_ref, l);
        uint8_t* part = smem + LY::kPart + w * LY::kPartBytes;
        if (rows_here)
          for (int x = 0; x < args.D; x += 16) {
            uint32_t r[16];
            ptx::tmem_ld_32x32b_x16(t_o + x, r);
            ptx::tmem_wait_ld_regs(r);
            if (live)
#pragma unroll
              for (int y = 0; y < 4; ++y)
                *reinterpret_cast<uint4*>(part + attn_part_at<DP>(rl, x / 4 + y)) =
                    l == 0.f ? make_uint4(0, 0, 0, 0)  // no kept state: O was never written
                             : make_uint4(r[4 * y], r[4 * y + 1], r[4 * y + 2], r[4 * y + 3]);
          }
      }
    }
    // stores in flight are done before the CTA ends
    if (!PAIRED && (threadIdx.x & 127) == 0) ptx::bulk_wait_group<0>();
    if (PAIRED || args.split > 1) {
      // ------------------------------------------------------------ join of the parts
      ptx::tc_fence_before();
      ptx::cluster_sync();
      {
        // This CTA finishes a block of the item's rows: first every row's share of each part (part
        // y: of CTA y, or of warpgroup y % 2 of CTA y / 2), then 4 elements per thread, the loads
        // of all parts in flight at once and a warp's in one row.
        constexpr int MP = PAIRED ? 2 * kAttnMaxSplit : kAttnMaxSplit;
        const Item it = item_at(item0);
        const int parts = PAIRED ? 2 * args.split : args.split;
        const int tile_rows = args.tile_tokens * args.heads;
        int n_rows = 0;
        for (int x = 0; x < LY::kQTiles; ++x) n_rows += rows_of(it, x);
        const int block = (n_rows + args.split - 1) / args.split;
        const int r0 = rank * block, r1 = min(n_rows, r0 + block);
        auto cta = [&](int y) { return PAIRED ? y >> 1 : y; };
        auto wg = [&](int y, int r) { return PAIRED ? y & 1 : r / tile_rows; };
        auto tile_row = [&](int r) { return PAIRED ? r : r % tile_rows; };
        auto token = [&](int r) { return it.tok0 + r / args.heads; };
        // behind the statistics that the other CTAs read: [row of the block][part] factors
        float* share = reinterpret_cast<float*>(smem + LY::kShare);
        for (int r = r0 + static_cast<int>(threadIdx.x); r < r1; r += WG * 128) {
          float2 ml[MP];
          float top = -INFINITY, total = 0.f;
#pragma unroll
          for (int y = 0; y < MP; ++y)
            if (y < parts)
              ml[y] = ptx::ld_cluster_f2(ptx::mapa_shared(
                  base + LY::kQ + (wg(y, r) * kAttnTile + tile_row(r)) * 8, cta(y)));
#pragma unroll
          for (int y = 0; y < MP; ++y)
            if (y < parts) top = fmaxf(top, ml[y].x);
#pragma unroll
          for (int y = 0; y < MP; ++y)
            if (y < parts) {
              ml[y].x = ml[y].x == top ? 1.f : ptx::ex2((ml[y].x - top) * c);
              total = fmaf(ml[y].y, ml[y].x, total);
            }
          const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
          for (int y = 0; y < MP; ++y)
            if (y < parts) share[(r - r0) * MP + y] = ml[y].x * inv;
          if (args.lse) {
            const int h = it.g * args.heads + r % args.heads;
            args.lse[(static_cast<int64_t>(it.b) * args.H + h) * args.L + token(r)] =
                total == 0.f ? -INFINITY : kLn2 * (top * c - shift + log2f(total));
          }
        }
        ptx::named_barrier(1, WG * 128);
        const int quads = args.D / 4;
        for (int x = threadIdx.x; x < (r1 - r0) * quads; x += WG * 128) {
          const int rb = x / quads, r = r0 + rb, ch = x - rb * quads, tr = tile_row(r);
          float4 o[MP];
#pragma unroll
          for (int y = 0; y < MP; ++y)
            if (y < parts)
              o[y] = ptx::ld_cluster_f4(ptx::mapa_shared(
                  base + LY::kPart + wg(y, r) * LY::kPartBytes + attn_part_at<DP>(tr, ch), cta(y)));
          float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int y = 0; y < MP; ++y)
            if (y < parts) {
              const float f = share[rb * MP + y];
              acc.x = fmaf(o[y].x, f, acc.x); acc.y = fmaf(o[y].y, f, acc.y);
              acc.z = fmaf(o[y].z, f, acc.z); acc.w = fmaf(o[y].w, f, acc.w);
            }
          const int h = it.g * args.heads + r % args.heads;
          *reinterpret_cast<uint2*>(static_cast<uint16_t*>(args.out) + it.b * args.out_sb +
                                    token(r) * args.out_st + h * args.out_sh + ch * 4) =
              make_uint2(ptx::pack16<BF16>(acc.x, acc.y), ptx::pack16<BF16>(acc.z, acc.w));
        }
      }
      ptx::cluster_sync();  // the parts stay until every CTA has read them
    }
  }
  __syncthreads();
  if (warp == LY::kMmaWarp) {
    __syncwarp();
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, 512);
  }
  if (*abort_flag) {
    // A wait ran out: which rows were finished is not known, nor what this CTA's part of a split
    // item lacks. All rows of its items become NaN, behind what any warp or CTA of the cluster has
    // stored (stores of this CTA have completed, those of the others are ahead of the last
    // cluster_sync).
    for (int item = item0; item < args.items; item += item_step) {
      const Item it = item_at(item);
      int n_rows = 0;
      for (int x = 0; x < LY::kQTiles; ++x) n_rows += rows_of(it, x);
      for (int r = threadIdx.x; r < n_rows; r += LY::kThreads) {
        const int tok = it.tok0 + r / args.heads, h = it.g * args.heads + r % args.heads;
        uint16_t* o = static_cast<uint16_t*>(args.out) + it.b * args.out_sb + tok * args.out_st +
                      h * args.out_sh;
        for (int x = 0; x < args.D; x += 8)
          *reinterpret_cast<uint4*>(o + x) =
              make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);  // NaN of both types
        if (args.lse)
          args.lse[(static_cast<int64_t>(it.b) * args.H + h) * args.L + tok] = NAN;
      }
    }
  }
}

}  // namespace dcnv2
