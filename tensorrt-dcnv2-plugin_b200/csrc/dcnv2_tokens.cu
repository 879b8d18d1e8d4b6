// dcnv2_tokens.cu — host side of the token operators of include/dcnv2.h: argument checks, launch
// shapes and the C entry points of dcnv2_qk_norm_rotary and dcnv2_cross_attention.
#include <atomic>
#include <climits>
#include <cmath>
#include <cstdint>
#include <cstring>

#include "../../include/dcnv2.h"
#include "../../include/dcnv2_diag.h"
#include "dcnv2_attention_kernel.cuh"
#include "dcnv2_attention_step_kernel.cuh"
#include "dcnv2_host.cuh"
#include "dcnv2_rotary_kernel.cuh"

namespace dcnv2 {
namespace {

// The current device, or null when it cannot run this library's code.
DevInfo* current_device(int* dev) {
  if (cudaGetDevice(dev) != cudaSuccess) {
    cudaGetLastError();
    return nullptr;
  }
  DevInfo* di = device_info(*dev);
  return di && di->ok && di->major == 10 ? di : nullptr;
}

cudaLaunchConfig_t launch_config(unsigned grid, unsigned threads, size_t smem, cudaStream_t st,
                                 cudaLaunchAttribute (&attr)[2], unsigned cluster) {
  // may start while the kernel ahead of it finishes; all three kernels call griddep_wait before
  // they touch memory
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid, 1, 1);
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cfg;
}

dcnv2_status launched(cudaError_t e) {
  if (e == cudaSuccess) return DCNV2_OK;
  cudaGetLastError();  // clear the launch error
  return DCNV2_ERR_CUDA;
}

// ------------------------------------------------------------------ norm and rotation

int rotary_elem_bytes(int dtype) {
  return dtype == DCNV2_FLOAT ? 4 : dtype == DCNV2_HALF || dtype == DCNV2_BF16 ? 2 : 0;
}

// Whether `extent` steps of `stride` elements stay far inside 64 bits (and go forward).
bool stride_ok(int64_t stride, int64_t extent) {
  return stride >= 0 && (extent <= 1 || stride <= (int64_t(1) << 60) / extent);
}

// Whether no two rows of `width` elements of an output meet: each stride steps over all that the
// smaller ones reach. Rows at one place would race.
bool apart(const int64_t (&stride)[3], const int64_t (&extent)[3], int64_t width) {
  if (!extent[0] || !extent[1] || !extent[2]) return true;
  bool used[3] = {extent[0] == 1, extent[1] == 1, extent[2] == 1};
  int64_t reach = width;
  for (;;) {
    int next = -1;
    for (int j = 0; j < 3; ++j)
      if (!used[j] && (next < 0 || stride[j] < stride[next])) next = j;
    if (next < 0) return true;
    if (stride[next] < reach) return false;
    used[next] = true;
    reach += stride[next] * (extent[next] - 1);
  }
}

dcnv2_status check_rotary(const dcnv2_rotary_desc* d) {
  if (!d) return DCNV2_ERR_INVALID_ARG;
  if (!rotary_elem_bytes(d->dtype)) return DCNV2_ERR_UNSUPPORTED;
  if (d->batch < 0 || d->tokens < 0 || d->q_heads < 0 || d->k_heads < 0 ||
      int64_t(d->q_heads) + d->k_heads < 1 || int64_t(d->q_heads) + d->k_heads > 65536)
    return DCNV2_ERR_INVALID_ARG;
  if (int64_t(d->batch) * d->tokens > INT_MAX) return DCNV2_ERR_INVALID_ARG;
  if (d->head_dim < 2 || d->head_dim % 2 || d->rotary_dim < 0 || d->rotary_dim % 2 ||
      d->rotary_dim > d->head_dim)
    return DCNV2_ERR_INVALID_ARG;
  if (d->head_dim > 2 * kRotMaxPairs) return DCNV2_ERR_UNSUPPORTED;
  if (d->norm != DCNV2_NORM_NONE && d->norm != DCNV2_NORM_RMS) return DCNV2_ERR_INVALID_ARG;
  if (d->norm != DCNV2_NORM_NONE && !(d->eps >= 0.f && std::isfinite(d->eps)))
    return DCNV2_ERR_INVALID_ARG;
  if (d->interleaved != 0 && d->interleaved != 1) return DCNV2_ERR_INVALID_ARG;
  if (d->rotary_dim > 0) {
    if (d->axes < 1 || d->axes > 4) return DCNV2_ERR_INVALID_ARG;
    for (int p = 0; p < d->rotary_dim / 2; ++p)
      if (d->pair_axis[p] >= d->axes) return DCNV2_ERR_INVALID_ARG;
    if (!stride_ok(d->pos_batch_stride, d->batch)) return DCNV2_ERR_INVALID_ARG;
  }
  const int64_t* in[2] = {d->q_stride, d->k_stride};
  const int64_t* out[2] = {d->q_out_stride, d->k_out_stride};
  const int heads[2] = {d->q_heads, d->k_heads};
  for (int i = 0; i < 2; ++i) {
    if (!heads[i]) continue;
    const int64_t extent[3] = {d->batch, d->tokens, heads[i]};
    for (int j = 0; j < 3; ++j) {
      if (!stride_ok(in[i][j], extent[j]) || !stride_ok(out[i][j], extent[j]))
        return DCNV2_ERR_INVALID_ARG;
    }
    const int64_t out_stride[3] = {out[i][0], out[i][1], out[i][2]};
    if (!apart(out_stride, extent, d->head_dim)) return DCNV2_ERR_INVALID_ARG;
  }
  return DCNV2_OK;
}

// Pairs per chunk: the most of {16, 8 bytes, 1 element} that every address a lane forms allows
// (pointers, strides and the places where the rotated pairs' halves and the rest begin).
int rotary_vec(const dcnv2_rotary_desc& d, const RotaryArgs& a, int elem) {
  const int rot = a.rot_pairs, rest = a.pairs - rot;
  for (int bytes = 16; bytes >= 8; bytes >>= 1) {
    const int vec = bytes / elem;
    if (rot % vec || rest % vec) continue;
    bool ok = true;
    for (int i = 0; i < 2; ++i) {
      const RotaryTensor& t = a.t[i];
      if (!(i ? d.k_heads : d.q_heads)) continue;
      const uintptr_t ptrs = reinterpret_cast<uintptr_t>(t.in) | reinterpret_cast<uintptr_t>(t.out) |
                             reinterpret_cast<uintptr_t>(t.weight);
      const int64_t strides = t.sb | t.st | t.sh | t.ob | t.ot | t.oh;
      ok = ok && ptrs % bytes == 0 && strides % vec == 0;
    }
    if (ok) return vec;
  }
  return 1;
}

template <typename T, int VEC, int NC, bool INTER>
dcnv2_status launch_rotary(RotaryArgs a, const DevInfo& di, cudaStream_t st) {
  const int64_t most = int64_t(di.sm_count) * kRotResident;  // warps
  int64_t units = 0;
  for (int i = 0; i < 2; ++i) {
    if (!a.heads[i]) continue;
    // heads side by side: a power of two, within the warp, and enough lanes to keep the cosines
    int& sh = a.side_shift[i];
    while (sh + a.group_shift < 5 && ((kRotHeads << sh) < a.heads[i] ||
                                      2 * a.rot_pairs > (kRotLane << (sh + a.group_shift))))
      ++sh;
    const int64_t blocks = cdiv(a.rows, 32 >> (sh + a.group_shift));
    const int all_steps = static_cast<int>(cdiv(a.heads[i], int64_t(kRotHeads) << sh));
    // all heads of a token in one unit, unless that leaves warps without work
    const int64_t want = cdiv(most, blocks);
    a.steps[i] = static_cast<int>(cdiv(all_steps, want < all_steps ? want : all_steps));
    a.parts[i] = static_cast<int>(cdiv(all_steps, a.steps[i]));
    if (blocks * a.parts[i] > INT_MAX) return DCNV2_ERR_INVALID_ARG;
    a.units[i] = static_cast<int>(blocks * a.parts[i]);
    units += a.units[i];
  }
  const int64_t grid = cdiv(units < most ? units : most, kRotWarps);
  cudaLaunchAttribute at[2];
  const size_t smem = kRotMaxPairs * (sizeof(uint64_t) + sizeof(int)) +
                      size_t(kRotThreads) * kRotLane * sizeof(float);
  const cudaLaunchConfig_t cfg =
      launch_config(static_cast<unsigned>(grid), kRotThreads, smem, st, at, 1);
  return launched(cudaLaunchKernelEx(&cfg, dcnv2_qk_norm_rotary_kernel<T, VEC, NC, INTER>, a));
}

template <typename T, int VEC, int NC>
dcnv2_status launch_rotary(const RotaryArgs& a, bool interleaved, const DevInfo& di,
                           cudaStream_t st) {
  return interleaved ? launch_rotary<T, VEC, NC, true>(a, di, st)
                     : launch_rotary<T, VEC, NC, false>(a, di, st);
}

// ------------------------------------------------------------------ attention

struct AttnPlan {
  bool step = false;       // few rows: dcnv2_attention_step_kernel
  bool paired = false;     // one tile of rows, the warpgroups alternate over the states
  bool wide = false;       // heads of more than 64 elements
  int wgs = 2;             // softmax warpgroups
  int heads = 1, kv_parts = 1, tile_tokens = 1;  // rows of a tile (AttnArgs)
  int row_tiles = 0, items = 0, split = 1;
  unsigned grid = 0;
};

// Limit of each wait of the tiled kernel; shorter ones are for tests of what happens behind it.
std::atomic<unsigned long long> g_attn_wait_ns{kDefaultTimeoutNs};

// States under a key mask, tiled kernel: the search of a longer row without a kept state would hold
// an SM for more than 0.46 s per item.
constexpr int kMaskTokens = 1 << 28;
// SMs of the device that the launch shapes are made for. It is not asked: the workspace size, and the
// words that an error is read from, follow from the desc alone, whatever device is current.
constexpr int kPlanSms = 148;

// CTAs of a cluster that split the states of one item, from the time of the whole in units of a
// state tile (about 2 us: its MMAs and exponentials for both warpgroups): waves of clusters *
// (tiles of a CTA + start + join). An item that is not split costs no join, and one start for all
// items of its CTA. (18 items of 8 tiles, split 8: 15 of the clusters run at once, 26 us; split 4:
// 15 us.)
int attn_split(int64_t items, int64_t tiles) {
  // clusters of 1, 2, ... CTAs that run at once with one CTA per SM, as the GPCs of 148 SMs allow
  static constexpr int kResident[kAttnMaxSplit + 1] = {0, 148, 74, 45, 33, 26, 22, 15, 15};
  constexpr double kStart = 1.5, kJoin = 1.0;
  int best = 1;
  double least = static_cast<double>(cdiv(items, kPlanSms)) * tiles + kStart;
  for (int s = 2; s <= kAttnMaxSplit && s <= tiles; ++s) {
    const double t = static_cast<double>(cdiv(items, kResident[s])) *
                     (static_cast<double>(cdiv(tiles, s)) + kStart + kJoin);
    if (t < least) {
      least = t;
      best = s;
    }
  }
  return best;
}

dcnv2_status make_attn_plan(const dcnv2_attention_desc* d, AttnPlan* p) {
  if (!d) return DCNV2_ERR_INVALID_ARG;
  if (d->dtype != DCNV2_HALF && d->dtype != DCNV2_BF16) return DCNV2_ERR_UNSUPPORTED;
  if (d->batch < 0 || d->q_tokens < 0 || d->kv_tokens < 0 || d->q_heads < 1 || d->kv_heads < 1 ||
      d->q_heads % d->kv_heads || d->head_dim < 1 || d->kv_tokens > INT_MAX - 1024)
    return DCNV2_ERR_INVALID_ARG;
  if (d->head_dim % 8 || d->head_dim > 128) return DCNV2_ERR_UNSUPPORTED;
  if (!(d->scale > 0.f && std::isfinite(d->scale * kLog2e))) return DCNV2_ERR_INVALID_ARG;
  const int64_t qx[3] = {d->batch, d->q_tokens, d->q_heads};
  const int64_t kx[3] = {d->batch, d->kv_tokens, d->kv_heads};
  for (int j = 0; j < 3; ++j) {
    if (!stride_ok(d->q_stride[j], qx[j]) || !stride_ok(d->out_stride[j], qx[j]) ||
        !stride_ok(d->k_stride[j], kx[j]) || !stride_ok(d->v_stride[j], kx[j]))
      return DCNV2_ERR_INVALID_ARG;
    if (qx[j] > 1 && (d->q_stride[j] % 8 || d->out_stride[j] % 8)) return DCNV2_ERR_UNSUPPORTED;
    if (j > 0 && qx[j] > 1 && !d->q_stride[j]) return DCNV2_ERR_UNSUPPORTED;
    if (j == 1 && kx[j] > 1 && (!d->k_stride[j] || !d->v_stride[j])) return DCNV2_ERR_UNSUPPORTED;
    if (kx[j] > 1 && (d->k_stride[j] % 8 || d->v_stride[j] % 8)) return DCNV2_ERR_UNSUPPORTED;
  }
  if (!apart(d->out_stride, qx, d->head_dim)) return DCNV2_ERR_INVALID_ARG;
  if (!stride_ok(d->mask_batch_stride, d->batch)) return DCNV2_ERR_INVALID_ARG;
  p->wide = d->head_dim > 64;
  const int group = d->q_heads / d->kv_heads;
  const int64_t rows = int64_t(d->q_tokens) * group;
  if (rows > INT_MAX - 2 * kAttnTile) return DCNV2_ERR_INVALID_ARG;
  // The step kernel holds 16 rows. Where it can run it is the faster one (us, step / tiled): 8 x
  // 60001 states, 8 kv heads of 128, 16 rows: 288 / 309; 32 x 5456, 8 heads of 32, 1 to 16 rows: 32
  // / 88; 5456 states, 8 kv heads of 128, 4 and 16 rows: 11.2 / 15.2, 13.8 / 17.3. With one row
  // more the tiled kernel takes those times: 310 (24 rows), 85 (17), 16.5 (20).
  p->step = rows <= kStepRows;
  if (p->step) {
    if (int64_t(d->batch) * d->kv_heads * kStepMaxSplit > INT_MAX) return DCNV2_ERR_INVALID_ARG;
    p->grid = 0;  // no error words: nothing in the kernel waits for another role
    return DCNV2_OK;
  }
  for (p->heads = group < kAttnTile ? group : kAttnTile; group % p->heads;) --p->heads;
  p->kv_parts = group / p->heads;
  p->tile_tokens = kAttnTile / p->heads;
  // One tile of rows: both warpgroups take its states in turn, or they would do nothing (us, paired
  // / not): 8 x 60001 states, 8 kv heads of 128, 24 to 128 rows: 310-338 / 424-441; 32 x 5456, 8
  // heads of 32, 17 to 128 rows: 85-90 / 189-191; 8 x 4001, 8 heads of 64: 22-26 / 43-45. Many
  // items of few states are the exception (64 x 300, 8 heads of 128: 49-70 / 43-46): a paired CTA
  // starts and joins anew for each.
  p->paired = d->q_tokens <= p->tile_tokens;
  p->wgs = !p->paired && !p->wide ? AttnLayout<64, false>::kWGs : AttnLayout<128, false>::kWGs;
  p->row_tiles =
      static_cast<int>(cdiv(d->q_tokens, int64_t(p->tile_tokens) * (p->paired ? 1 : p->wgs)));
  const int64_t groups = int64_t(d->kv_heads) * p->kv_parts;
  if (groups > INT_MAX || int64_t(d->batch) * groups > INT_MAX) return DCNV2_ERR_INVALID_ARG;
  const int64_t ctas = int64_t(d->batch) * groups * p->row_tiles;
  p->split = attn_split(ctas, cdiv(d->kv_tokens, kAttnTile * (p->paired ? 2 : 1)));
  if (ctas * p->split > INT_MAX) return DCNV2_ERR_INVALID_ARG;
  p->items = static_cast<int>(ctas);
  // items that are not split or joined are taken in turn by one CTA per SM
  const int64_t most = p->paired || p->split > 1 ? ctas : kPlanSms;
  p->grid = static_cast<unsigned>((ctas < most ? ctas : most) * p->split);
  return DCNV2_OK;
}

AttnTensor attn_tensor(const void* p, const int64_t (&stride)[3], int64_t batch, int64_t tokens,
                       int64_t heads) {
  // a stride that no second element is reached by may hold anything
  return AttnTensor{p, batch > 1 ? stride[0] : 0, tokens > 1 ? stride[1] : 0,
                    heads > 1 ? stride[2] : 0};
}

bool encode_map(CUtensorMap* m, const void* p, int rank, const cuuint64_t* dims,
                const cuuint64_t* strides, const cuuint32_t* box) {
  const cuuint32_t ones[5] = {1, 1, 1, 1, 1};
  std::memset(m, 0, sizeof(*m));
  PFN_cuTensorMapEncodeTiled_v12000 encode = tensor_map_encoder();
  return encode &&
         encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT16, rank, const_cast<void*>(p), dims, strides, box,
                ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Tensor map of k or v: (element, token, head, batch), boxes of 64 elements x the 256 / wgs tokens
// of a tile in the 128-byte swizzle. Axes that no step is taken along, or that share their states,
// have extent 1. What lies outside (elements from head_dim on, tokens from kv_tokens on) reads as
// zeros.
bool states_map(CUtensorMap* m, const void* p, const int64_t (&stride)[3],
                const dcnv2_attention_desc& d, int wgs, int* batch_step, int* head_step) {
  const bool heads = d.kv_heads > 1 && stride[2] > 0, batch = d.batch > 1 && stride[0] > 0;
  *head_step = heads;
  *batch_step = batch;
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(d.head_dim),
                              static_cast<cuuint64_t>(d.kv_tokens),
                              static_cast<cuuint64_t>(heads ? d.kv_heads : 1),
                              static_cast<cuuint64_t>(batch ? d.batch : 1)};
  const cuuint64_t row = static_cast<cuuint64_t>(d.head_dim) * 2;
  const cuuint64_t strides[3] = {d.kv_tokens > 1 ? static_cast<cuuint64_t>(stride[1]) * 2 : row,
                                 heads ? static_cast<cuuint64_t>(stride[2]) * 2 : row,
                                 batch ? static_cast<cuuint64_t>(stride[0]) * 2 : row};
  const cuuint32_t box[4] = {64, 256u / static_cast<cuuint32_t>(wgs), 1, 1};
  return encode_map(m, p, 4, dims, strides, box);
}

// Tensor map of q or out: (element, head of the group, token, group, batch), boxes of 64 elements x
// the rows of a tile.
bool rows_map(CUtensorMap* m, const void* p, const int64_t (&stride)[3],
              const dcnv2_attention_desc& d, const AttnPlan& plan, int* batch_step) {
  const int64_t groups = int64_t(d.q_heads) / plan.heads;
  const bool batch = d.batch > 1 && stride[0] > 0;
  *batch_step = batch;
  const cuuint64_t dims[5] = {static_cast<cuuint64_t>(d.head_dim),
                              static_cast<cuuint64_t>(plan.heads),
                              static_cast<cuuint64_t>(d.q_tokens),
                              static_cast<cuuint64_t>(groups),
                              static_cast<cuuint64_t>(batch ? d.batch : 1)};
  const cuuint64_t row = static_cast<cuuint64_t>(d.head_dim) * 2;
  const cuuint64_t head = d.q_heads > 1 ? static_cast<cuuint64_t>(stride[2]) * 2 : row;
  const cuuint64_t strides[4] = {head,
                                 d.q_tokens > 1 ? static_cast<cuuint64_t>(stride[1]) * 2 : row,
                                 head * plan.heads,
                                 batch ? static_cast<cuuint64_t>(stride[0]) * 2 : row};
  const cuuint32_t box[5] = {64, static_cast<cuuint32_t>(plan.heads),
                             static_cast<cuuint32_t>(plan.tile_tokens), 1, 1};
  return encode_map(m, p, 5, dims, strides, box);
}

struct AttnMaps {
  CUtensorMap q, k, v, o;
};

template <int DP, bool PAIRED, bool BF16>
dcnv2_status launch_attention(const AttnArgs& a, const AttnMaps& m, const AttnPlan& p, int dev,
                              cudaStream_t st) {
  auto kernel = dcnv2_cross_attention_kernel<DP, PAIRED, BF16>;
  constexpr size_t smem = attn_smem_bytes<DP, PAIRED>();
  static_assert(smem <= kSmemLimit, "shared memory");
  static std::atomic<bool> set[kMaxDevices];  // per device; setting it twice does no harm
  if (!set[dev].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               static_cast<int>(smem));
    if (e != cudaSuccess) return launched(e);
    set[dev].store(true, std::memory_order_release);
  }
  cudaLaunchAttribute at[2];
  const cudaLaunchConfig_t cfg = launch_config(p.grid, AttnLayout<DP, PAIRED>::kThreads, smem, st,
                                               at, static_cast<unsigned>(p.split));
  return launched(cudaLaunchKernelEx(&cfg, kernel, a, m.q, m.k, m.v, m.o));
}

template <bool BF16>
dcnv2_status launch_attention(const AttnArgs& a, const AttnMaps& m, const AttnPlan& p, int dev,
                              cudaStream_t st) {
  if (p.wide)
    return p.paired ? launch_attention<128, true, BF16>(a, m, p, dev, st)
                    : launch_attention<128, false, BF16>(a, m, p, dev, st);
  return p.paired ? launch_attention<64, true, BF16>(a, m, p, dev, st)
                  : launch_attention<64, false, BF16>(a, m, p, dev, st);
}

// CTAs of a cluster that split the states of one (sequence, kv head): as few as give every SM a
// CTA, with a chunk for each of their warps. One CTA draws at most about 50 GB/s, so that fewer
// CTAs than SMs leave bandwidth unused, while more cost their start and end again (32 x 8 heads of
// 32, 5456 states: 256 CTAs 32 us, 512 36 us, 1024 44 us; 8 kv heads of 128, 5456 states: 64 CTAs
// 12.9 us, 128 10.9 us). Lengths of their own leave SMs idle behind the short sequences; four times
// the CTAs even that out (8 x 8 heads of 128, up to 60001 states: 128 CTAs 240 us, 512 208 us, 1024
// 200 us).
int step_split(int64_t units, const AttnStepArgs& a, int sm_count) {
  const int keys = a.D > 64 ? 16 : a.D > 32 ? 32 : 64;
  const int64_t want = int64_t(sm_count) * (a.kv_lens ? 4 : 1);
  int split = 1;
  while (split < kStepMaxSplit && units * split < want &&
         cdiv(a.S, keys) >= int64_t(split) * 2 * kStepWarps)
    split *= 2;
  return split;
}

template <int DP, bool BF16>
dcnv2_status launch_step(const AttnStepArgs& a, int64_t units, int dev, cudaStream_t st) {
  auto kernel = dcnv2_attention_step_kernel<DP, BF16>;
  constexpr size_t smem = StepLayout<DP>::kTotal;
  static_assert(2 * (smem + 1024) <= 228 * 1024, "two CTAs per SM");
  static std::atomic<bool> set[kMaxDevices];  // per device; setting it twice does no harm
  if (!set[dev].load(std::memory_order_acquire)) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         static_cast<int>(smem));
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return launched(e);
    set[dev].store(true, std::memory_order_release);
  }
  cudaLaunchAttribute at[2];
  const cudaLaunchConfig_t cfg =
      launch_config(static_cast<unsigned>(units * a.split), kStepThreads, smem, st, at,
                    static_cast<unsigned>(a.split));
  return launched(cudaLaunchKernelEx(&cfg, kernel, a));
}

template <bool BF16>
dcnv2_status launch_step(const AttnStepArgs& a, int64_t units, int dev, cudaStream_t st) {
  return a.D > 64   ? launch_step<128, BF16>(a, units, dev, st)
         : a.D > 32 ? launch_step<64, BF16>(a, units, dev, st)
                    : launch_step<32, BF16>(a, units, dev, st);
}

}  // namespace
}  // namespace dcnv2

using namespace dcnv2;

extern "C" {

dcnv2_status dcnv2_qk_norm_rotary(const dcnv2_rotary_desc* desc, const void* q, const void* k,
                                  const int32_t* positions, const float* freqs,
                                  const void* q_weight, const void* k_weight, void* q_out,
                                  void* k_out, dcnv2_stream_t stream) {
  const dcnv2_status s = check_rotary(desc);
  if (s != DCNV2_OK) return s;
  const dcnv2_rotary_desc& d = *desc;
  if (d.batch == 0 || d.tokens == 0) return DCNV2_OK;
  if ((d.q_heads && (!q || !q_out)) || (d.k_heads && (!k || !k_out)) ||
      (d.rotary_dim && (!positions || !freqs)))
    return DCNV2_ERR_INVALID_ARG;
  const int elem = rotary_elem_bytes(d.dtype);
  RotaryArgs a = {};
  const bool norm = d.norm != DCNV2_NORM_NONE;
  const void* in[2] = {q, k};
  void* out[2] = {q_out, k_out};
  const void* weight[2] = {norm ? q_weight : nullptr, norm ? k_weight : nullptr};
  const int64_t* is[2] = {d.q_stride, d.k_stride};
  const int64_t* os[2] = {d.q_out_stride, d.k_out_stride};
  const int heads[2] = {d.q_heads, d.k_heads};
  for (int i = 0; i < 2; ++i) {
    if (!heads[i]) continue;
    // a stride that no second element is reached by may hold anything
    const bool many[3] = {d.batch > 1, d.tokens > 1, heads[i] > 1};
    a.t[i] = RotaryTensor{in[i], out[i], weight[i],
                          many[0] ? is[i][0] : 0, many[1] ? is[i][1] : 0, many[2] ? is[i][2] : 0,
                          many[0] ? os[i][0] : 0, many[1] ? os[i][1] : 0, many[2] ? os[i][2] : 0};
    if ((reinterpret_cast<uintptr_t>(in[i]) | reinterpret_cast<uintptr_t>(out[i]) |
         reinterpret_cast<uintptr_t>(weight[i])) % elem)
      return DCNV2_ERR_INVALID_ARG;
  }
  if ((reinterpret_cast<uintptr_t>(positions) | reinterpret_cast<uintptr_t>(freqs)) % 4)
    return DCNV2_ERR_INVALID_ARG;
  a.pos = positions;
  a.freqs = freqs;
  a.pos_sb = d.batch > 1 ? d.pos_batch_stride : 0;
  a.rows = d.batch * d.tokens;
  a.tokens = d.tokens;
  a.heads[0] = d.q_heads;
  a.heads[1] = d.k_heads;
  a.pairs = d.head_dim / 2;
  a.rot_pairs = d.rotary_dim / 2;
  a.axes = d.axes;
  a.norm = norm;
  a.eps = d.eps;
  a.inv_d = 1.0f / static_cast<float>(d.head_dim);
  for (int p = 0; p < a.rot_pairs; ++p)
    a.pair_axis[p >> 4] |= static_cast<uint32_t>(d.pair_axis[p]) << (2 * (p & 15));
  const int vec = rotary_vec(d, a, elem);
  a.chunks = a.pairs / vec;
  while ((1 << a.group_shift) < a.chunks && a.group_shift < 5) ++a.group_shift;
  int dev = 0;
  const DevInfo* di = current_device(&dev);
  if (!di) return DCNV2_ERR_NO_DEVICE;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool inter = d.interleaved != 0;
  if (d.dtype == DCNV2_FLOAT)
    return vec == 4   ? launch_rotary<float, 4, 1>(a, inter, *di, st)
           : vec == 2 ? launch_rotary<float, 2, 2>(a, inter, *di, st)
                      : launch_rotary<float, 1, 4>(a, inter, *di, st);
  if (d.dtype == DCNV2_HALF)
    return vec == 8   ? launch_rotary<__half, 8, 1>(a, inter, *di, st)
           : vec == 4 ? launch_rotary<__half, 4, 1>(a, inter, *di, st)
                      : launch_rotary<__half, 1, 4>(a, inter, *di, st);
  return vec == 8   ? launch_rotary<__nv_bfloat16, 8, 1>(a, inter, *di, st)
         : vec == 4 ? launch_rotary<__nv_bfloat16, 4, 1>(a, inter, *di, st)
                    : launch_rotary<__nv_bfloat16, 1, 4>(a, inter, *di, st);
}

size_t dcnv2_cross_attention_workspace_size(const dcnv2_attention_desc* desc) {
  AttnPlan p;
  if (make_attn_plan(desc, &p) != DCNV2_OK) return 0;
  return align_up(size_t(p.grid) * sizeof(int), 256);
}

dcnv2_status dcnv2_cross_attention(const dcnv2_attention_desc* desc, const void* q, const void* k,
                                   const void* v, const int32_t* kv_lens, const uint8_t* key_mask,
                                   void* out, float* lse, void* workspace, size_t workspace_bytes,
                                   dcnv2_stream_t stream) {
  AttnPlan p;
  const dcnv2_status s = make_attn_plan(desc, &p);
  if (s != DCNV2_OK) return s;
  const dcnv2_attention_desc& d = *desc;
  if (d.batch == 0 || d.q_tokens == 0) return DCNV2_OK;
  if (!q || !out || (d.kv_tokens && (!k || !v))) return DCNV2_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) |
       reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(out)) % 16)
    return DCNV2_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(kv_lens) | reinterpret_cast<uintptr_t>(lse)) % 4)
    return DCNV2_ERR_INVALID_ARG;
  if (p.grid && key_mask && d.kv_tokens > kMaskTokens) return DCNV2_ERR_UNSUPPORTED;
  if (p.grid && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 4 ||
                 workspace_bytes < size_t(p.grid) * sizeof(int)))
    return DCNV2_ERR_WORKSPACE;
  int dev = 0;
  DevInfo* di = current_device(&dev);
  if (!di) return DCNV2_ERR_NO_DEVICE;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int group = d.q_heads / d.kv_heads;
  const AttnTensor tq = attn_tensor(q, d.q_stride, d.batch, d.q_tokens, d.q_heads);
  const AttnTensor to = attn_tensor(out, d.out_stride, d.batch, d.q_tokens, d.q_heads);
  const int64_t mask_sb = d.batch > 1 ? d.mask_batch_stride : 0;
  if (p.step) {
    AttnStepArgs a = {tq,
                      attn_tensor(k, d.k_stride, d.batch, d.kv_tokens, d.kv_heads),
                      attn_tensor(v, d.v_stride, d.batch, d.kv_tokens, d.kv_heads),
                      to, kv_lens, key_mask, mask_sb, lse, d.q_tokens, d.kv_tokens, d.q_heads,
                      d.kv_heads, d.head_dim, group, d.q_tokens * group, 1, d.scale};
    const int64_t units = int64_t(d.batch) * d.kv_heads;
    a.split = step_split(units, a, di->sm_count);
    return d.dtype == DCNV2_BF16 ? launch_step<true>(a, units, dev, st)
                                 : launch_step<false>(a, units, dev, st);
  }
  AttnArgs a = {};
  a.kv_lens = kv_lens;
  a.key_mask = key_mask;
  a.mask_sb = mask_sb;
  a.lse = lse;
  a.out = out;
  a.out_sb = to.sb; a.out_st = to.st; a.out_sh = to.sh;
  a.err = static_cast<int*>(workspace);
  a.L = d.q_tokens; a.S = d.kv_tokens; a.H = d.q_heads; a.D = d.head_dim;
  a.heads = p.heads;
  a.kv_parts = p.kv_parts;
  a.groups = d.kv_heads * p.kv_parts;
  a.tile_tokens = p.tile_tokens;
  a.row_tiles = p.row_tiles;
  a.items = p.items;
  a.split = p.split;
  a.scale = d.scale;
  a.timeout_ns = g_attn_wait_ns.load(std::memory_order_relaxed);
  AttnMaps m;
  int out_batch = 0;
  if (!rows_map(&m.q, q, d.q_stride, d, p, &a.q_batch) ||
      !rows_map(&m.o, out, d.out_stride, d, p, &out_batch))
    return DCNV2_ERR_UNSUPPORTED;  // strides of 2^40 bytes and more
  if (d.kv_tokens == 0) {  // nothing is loaded
    m.k = m.v = m.q;
  } else if (!states_map(&m.k, k, d.k_stride, d, p.wgs, &a.k_batch, &a.k_head) ||
             !states_map(&m.v, v, d.v_stride, d, p.wgs, &a.v_batch, &a.v_head)) {
    return DCNV2_ERR_UNSUPPORTED;
  }
  return d.dtype == DCNV2_BF16 ? launch_attention<true>(a, m, p, dev, st)
                               : launch_attention<false>(a, m, p, dev, st);
}

dcnv2_status dcnv2_cross_attention_read_error(const dcnv2_attention_desc* desc,
                                              const void* workspace, dcnv2_stream_t stream,
                                              int32_t* code) {
  AttnPlan p;
  const dcnv2_status s = make_attn_plan(desc, &p);
  if (s != DCNV2_OK) return s;
  if (!code || (p.grid && !workspace)) return DCNV2_ERR_INVALID_ARG;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  int32_t bits = 0;
  const int* words = static_cast<const int*>(workspace);
  for (unsigned at = 0; at < p.grid;) {  // (none for a few rows)
    int32_t part[1024];
    const unsigned n = p.grid - at < 1024u ? p.grid - at : 1024u;
    if (cudaMemcpyAsync(part, words + at, n * sizeof(int), cudaMemcpyDeviceToHost, st) !=
            cudaSuccess ||
        cudaStreamSynchronize(st) != cudaSuccess) {
      cudaGetLastError();
      return DCNV2_ERR_CUDA;
    }
    for (unsigned i = 0; i < n; ++i) bits |= part[i];
    at += n;
  }
  *code = bits;
  return bits ? DCNV2_ERR_DEVICE_TIMEOUT : DCNV2_OK;
}

dcnv2_status dcnv2_diag_set_attention_wait_limit(int32_t limit_us) {
  if (limit_us < -1 || limit_us > static_cast<int32_t>(kDefaultTimeoutNs / 1000))
    return DCNV2_ERR_INVALID_ARG;
  g_attn_wait_ns.store(limit_us < 0 ? kDefaultTimeoutNs : 1000ull * limit_us);
  return DCNV2_OK;
}

}  // extern "C"
