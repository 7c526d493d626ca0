// pad_decode_fp4.cu -- host side of the decode over the 4-bit paged cache
// (pad_decode_fp4_kernel.cuh): argument checks, the plan and the launches.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>
#include <cstdint>

#include "pad_b200.h"
#include "pad_decode_fp4_kernel.cuh"
#include "pad_decode_instance.cuh"
#include "pad_error.cuh"

namespace {

using namespace pad;

constexpr int kMaxG = 16;
constexpr int kFp4Devices = 64;
constexpr int kTile = 32;  // tokens of a tile, Fp4Traits::TT

bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
size_t align_up(size_t x, size_t a) { return (x + a - 1) / a * a; }

struct Fp4Instance {
  const void* kernel;
  int smem_bytes, threads, key;
};

template <int D, int NT, bool WT>
Fp4Instance instance(int key) {
  using TR = Fp4Traits<D, NT, WT>;
  static_assert(TR::TT == kTile, "tile");
  return {reinterpret_cast<const void*>(&decode_fp4_kernel<TR>), TR::SMEM_BYTES, TR::THREADS, key};
}

// Query heads per KV head up to 8 fill one n8 tile of the tensor cores, more
// take two (and half the warps, for their registers).
template <int D>
Fp4Instance pick(int64_t gqa, bool weights, int key) {
  if (gqa <= 8) return weights ? instance<D, 1, true>(key) : instance<D, 1, false>(key + 1);
  return weights ? instance<D, 2, true>(key + 2) : instance<D, 2, false>(key + 3);
}

constexpr int kInstances = 12;

int prepare(int device, const Fp4Instance& in) {
  static std::atomic<bool> done[kFp4Devices][kInstances];  // set twice by racing threads at worst
  if (device < 0 || device >= kFp4Devices) return fail(PAD_ERR_INVALID_ARGUMENT, "device %d out of range", device);
  if (!done[device][in.key].load()) {
    const cudaError_t e = cudaFuncSetAttribute(in.kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, in.smem_bytes);
    if (e != cudaSuccess) return cuda_fail(e, "configuring the decode_fp4 kernel");
    done[device][in.key].store(true);
  }
  return PAD_OK;
}

struct Fp4Plan {
  int hg = 1;
  int64_t partitions = 1, slots = 0, raw_tiles = 0;
  size_t off_ml = 0, off_o = 0, off_total = 0, off_norm = 0, off_tiles = 0, off_raw = 0, bytes = 0;
};

int make_plan(int device, int64_t batch, int64_t hkv, int64_t gqa, int64_t head_dim, int64_t num_pages,
              int64_t page_size, int64_t max_pages, int64_t num_splits, bool weights, Fp4Plan* plan) {
  const char* what = "decode_fp4";
  if (batch < 0 || hkv <= 0 || gqa <= 0 || num_pages < 0 || page_size <= 0 || max_pages < 0)
    return fail(PAD_ERR_INVALID_ARGUMENT, "%s: negative or zero size", what);
  if (head_dim != 32 && head_dim != 64 && head_dim != 128)
    return fail(PAD_ERR_UNSUPPORTED, "%s: head_dim %lld not supported (32, 64 or 128)", what, (long long)head_dim);
  if (gqa > kMaxG) return fail(PAD_ERR_UNSUPPORTED, "%s: gqa_ratio %lld > 16 not supported", what, (long long)gqa);
  if (num_pages > INT32_MAX || max_pages > INT32_MAX || page_size > INT32_MAX || hkv > INT32_MAX ||
      max_pages * page_size > INT32_MAX / 2)
    return fail(PAD_ERR_UNSUPPORTED, "%s: problem too large for 32-bit indexing", what);
  // KV heads per tile: what divides the kernel's 12 or 8 warps
  plan->hg = std::min(4, head_group_for(hkv, gqa));
  const int64_t groups = hkv / plan->hg, tiles = (max_pages * page_size + kTile - 1) / kTile;
  if (batch > INT32_MAX / 4 / groups || batch * groups > INT32_MAX / 4 / std::max<int64_t>(tiles, 1))
    return fail(PAD_ERR_UNSUPPORTED, "%s: problem too large for 32-bit indexing", what);
  const int64_t tiles_ub = batch * groups * tiles, pairs = batch * groups;
  int64_t parts;
  if (num_splits <= 0) {
    int sms = 0;
    const int st = sm_count(device, &sms);
    if (st != PAD_OK) return st;
    parts = std::min<int64_t>(sms, tiles_ub);
  } else {
    if (num_splits > ((int64_t)1 << 30) / std::max<int64_t>(pairs, 1))
      return fail(PAD_ERR_UNSUPPORTED, "%s: num_splits %lld too large", what, (long long)num_splits);
    parts = num_splits * pairs;
  }
  plan->partitions = std::max<int64_t>(parts, 1);
  plan->slots = plan->partitions + pairs;
  const int64_t rows = plan->hg * gqa;
  plan->off_ml = align_up((size_t)std::max(plan->partitions, pairs) * sizeof(int4), 256);
  plan->off_o = align_up(plan->off_ml + (size_t)(plan->slots * rows) * sizeof(float2), 256);
  plan->bytes = align_up(plan->off_o + (size_t)(plan->slots * rows * head_dim) * sizeof(float), 256);
  if (weights) {
    // as for the fp16 decode: no more tiles than the table names or the pool holds
    plan->raw_tiles = std::min(tiles_ub, groups * (num_pages * page_size / kTile + batch));
    plan->off_total = plan->bytes;
    plan->off_norm = plan->off_total + 256;
    plan->off_tiles = align_up(plan->off_norm + (size_t)(pairs * rows) * sizeof(float2), 256);
    plan->off_raw = align_up(plan->off_tiles + (size_t)plan->raw_tiles * sizeof(int4), 256);
    plan->bytes = align_up(plan->off_raw + (size_t)(plan->raw_tiles * rows * kTile) * sizeof(float), 256);
  }
  return PAD_OK;
}

// Whether every offset of a tensor of these strides stays below 2^32 units.
bool offsets_fit(const int64_t* s, int64_t pages, int64_t ps, int64_t hkv, int unit) {
  if (s[0] < 0 || s[1] < 0 || s[2] < 0) return false;
  const double last = (double)(pages - 1) * (double)s[0] + (double)(ps - 1) * (double)s[1] + (double)(hkv - 1) * (double)s[2];
  return pages == 0 || last / unit < 4294967296.0;
}

// num_new_of: new tokens of each sequence, or null: num_new of every one.
int decode_fp4(
    const void* q, const void* k_cache, const void* k_scales, const void* v_cache, const void* v_scales,
    const int32_t* block_table, const int32_t* seq_lens, void* out, float* weights, int32_t* slot_positions,
    const int32_t* total_lens, int64_t num_new, const int32_t* num_new_of, int64_t batch, int64_t num_q_heads, int64_t num_kv_heads,
    int64_t head_dim, int64_t num_pages, int64_t page_size, int64_t max_pages_per_seq, const int64_t* q_strides,
    const int64_t* k_strides, const int64_t* ks_strides, const int64_t* v_strides, const int64_t* vs_strides,
    int64_t block_table_stride, const int64_t* out_strides, const int64_t* weight_strides,
    const int64_t* position_strides, float scale, int64_t num_splits, void* workspace, size_t workspace_bytes,
    void* stream, int32_t* error_flags) {
  const char* what = "decode_fp4";
  if (batch < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_pages < 0 || page_size <= 0 || max_pages_per_seq < 0)
    return fail(PAD_ERR_INVALID_ARGUMENT, "%s: negative or zero size", what);
  if (head_dim != 32 && head_dim != 64 && head_dim != 128)
    return fail(PAD_ERR_UNSUPPORTED, "%s: head_dim %lld not supported (32, 64 or 128)", what, (long long)head_dim);
  if (num_q_heads % num_kv_heads != 0)
    return fail(PAD_ERR_INVALID_ARGUMENT, "%s: num_q_heads (%lld) must be divisible by num_kv_heads (%lld)", what,
                (long long)num_q_heads, (long long)num_kv_heads);
  const int64_t gqa = num_q_heads / num_kv_heads;
  if (gqa > kMaxG) return fail(PAD_ERR_UNSUPPORTED, "%s: gqa_ratio %lld > 16 not supported", what, (long long)gqa);
  if (!std::isfinite(scale)) return fail(PAD_ERR_INVALID_ARGUMENT, "%s: scale must be finite", what);
  if (num_new < 0) return fail(PAD_ERR_INVALID_ARGUMENT, "%s: num_new must not be negative", what);
  if (batch == 0) return PAD_OK;
  // a pool or a table of nothing has no address: every sequence is then empty
  if (q == nullptr || seq_lens == nullptr || (max_pages_per_seq > 0 && block_table == nullptr) ||
      (num_pages > 0 && (k_cache == nullptr || k_scales == nullptr || v_cache == nullptr || v_scales == nullptr)) ||
      out == nullptr || q_strides == nullptr ||
      k_strides == nullptr || ks_strides == nullptr || v_strides == nullptr || vs_strides == nullptr ||
      out_strides == nullptr || (weights != nullptr && weight_strides == nullptr) ||
      (slot_positions != nullptr && (weights == nullptr || position_strides == nullptr || total_lens == nullptr)))
    return fail(PAD_ERR_INVALID_ARGUMENT, "%s: null pointer argument", what);
  if (q_strides[2] != 1 || k_strides[3] != 1 || ks_strides[3] != 1 || v_strides[3] != 1 || vs_strides[3] != 1 ||
      out_strides[2] != 1)
    return fail(PAD_ERR_UNSUPPORTED, "%s: the last axis of every tensor must be contiguous", what);
  for (int i = 0; i < 3; ++i)
    if (k_strides[i] % 16 || v_strides[i] % 16 || ks_strides[i] % kFp4ScaleRow || vs_strides[i] % kFp4ScaleRow)
      return fail(PAD_ERR_UNSUPPORTED, "%s: code strides must be multiples of 16 bytes, scale strides of 4", what);
  if (q_strides[0] % 8 || q_strides[1] % 8 || !aligned(q, 16))
    return fail(PAD_ERR_UNSUPPORTED, "%s: q must be 16-byte aligned with strides that are multiples of 8", what);
  if (out_strides[0] % 2 || out_strides[1] % 2 || !aligned(out, 4))
    return fail(PAD_ERR_UNSUPPORTED, "%s: out must be 4-byte aligned with even strides", what);
  if (!aligned(k_cache, 16) || !aligned(v_cache, 16) || !aligned(k_scales, 4) || !aligned(v_scales, 4))
    return fail(PAD_ERR_UNSUPPORTED, "%s: codes must be 16-byte aligned, scales 4-byte aligned", what);
  if (block_table_stride < max_pages_per_seq)
    return fail(PAD_ERR_INVALID_ARGUMENT, "%s: block_table row stride smaller than its width", what);
  int device = 0;
  cudaError_t e = cudaSuccess;
  // the sizes are checked before the device is asked for
  Fp4Plan plan;
  int st = make_plan(0, batch, num_kv_heads, gqa, head_dim, num_pages, page_size, max_pages_per_seq,
                     std::max<int64_t>(num_splits, 1), weights != nullptr, &plan);
  if (st != PAD_OK) return st;
  // Offsets are kept in 32 bits, those of codes in units of the largest power of
  // two (16 to 64 bytes) that divides every stride.
  uint64_t all = 0;
  for (int i = 0; i < 3; ++i) all |= (uint64_t)k_strides[i] | (uint64_t)v_strides[i];
  int unit = 16;
  while (unit < 64 && all % (2 * unit) == 0) unit *= 2;
  if (!offsets_fit(k_strides, num_pages, page_size, num_kv_heads, unit) ||
      !offsets_fit(v_strides, num_pages, page_size, num_kv_heads, unit) ||
      !offsets_fit(ks_strides, num_pages, page_size, num_kv_heads, kFp4ScaleRow) ||
      !offsets_fit(vs_strides, num_pages, page_size, num_kv_heads, kFp4ScaleRow))
    return fail(PAD_ERR_UNSUPPORTED,
                "%s: cache strides are negative or reach past 2^32 units (codes: %d bytes, scales: 4)", what, unit);
  if (block_table_stride > INT32_MAX)
    return fail(PAD_ERR_UNSUPPORTED, "%s: block_table row stride exceeds int32", what);
  if ((e = cudaGetDevice(&device)) != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  if (num_splits <= 0 && (st = make_plan(device, batch, num_kv_heads, gqa, head_dim, num_pages, page_size,
                                         max_pages_per_seq, num_splits, weights != nullptr, &plan)) != PAD_OK)
    return st;
  if (workspace == nullptr || workspace_bytes < plan.bytes)
    return fail(PAD_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, %zu given", what, plan.bytes,
                workspace == nullptr ? (size_t)0 : workspace_bytes);
  if (!aligned(workspace, 16)) return fail(PAD_ERR_WORKSPACE, "%s: workspace must be 16-byte aligned", what);
  const Fp4Instance in = head_dim == 32   ? pick<32>(gqa, weights != nullptr, 0)
                         : head_dim == 64 ? pick<64>(gqa, weights != nullptr, 4)
                                          : pick<128>(gqa, weights != nullptr, 8);
  if ((st = prepare(device, in)) != PAD_OK) return st;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  Fp4DecodeParams p = {};
  p.q = static_cast<const __half*>(q);
  p.k = static_cast<const uint8_t*>(k_cache);
  p.ks = static_cast<const uint8_t*>(k_scales);
  p.v = static_cast<const uint8_t*>(v_cache);
  p.vs = static_cast<const uint8_t*>(v_scales);
  p.block_table = block_table;
  p.seq_lens = seq_lens;
  p.out = static_cast<__half*>(out);
  p.ws_meta = reinterpret_cast<int4*>(ws);
  p.ws_ml = reinterpret_cast<float2*>(ws + plan.off_ml);
  p.ws_o = reinterpret_cast<float*>(ws + plan.off_o);
  p.error_flags = error_flags;
  p.q0 = q_strides[0];
  p.q1 = q_strides[1];
  p.bt_stride = (int)block_table_stride;
  p.out_sb = out_strides[0];
  p.out_sh = out_strides[1];
  p.unit = (uint32_t)unit;
  p.k0 = (uint32_t)(k_strides[0] / unit);
  p.k1 = (uint32_t)(k_strides[1] / unit);
  p.k2 = (uint32_t)(k_strides[2] / unit);
  p.v0 = (uint32_t)(v_strides[0] / unit);
  p.v1 = (uint32_t)(v_strides[1] / unit);
  p.v2 = (uint32_t)(v_strides[2] / unit);
  p.ks0 = (uint32_t)(ks_strides[0] / kFp4ScaleRow);
  p.ks1 = (uint32_t)(ks_strides[1] / kFp4ScaleRow);
  p.ks2 = (uint32_t)(ks_strides[2] / kFp4ScaleRow);
  p.vs0 = (uint32_t)(vs_strides[0] / kFp4ScaleRow);
  p.vs1 = (uint32_t)(vs_strides[1] / kFp4ScaleRow);
  p.vs2 = (uint32_t)(vs_strides[2] / kFp4ScaleRow);
  p.batch = (int)batch;
  p.hkv = (int)num_kv_heads;
  p.gqa = (int)gqa;
  p.hg_log2 = __builtin_ctz((unsigned)plan.hg);
  p.page_size = (int)page_size;
  // division by page_size: with 2^(L - 1) < page_size <= 2^L, the multiplier
  // floor(2^(31 + L) / page_size) + 1 is exact for every dividend below 2^31
  int log2_up = 0;
  while (((int64_t)1 << log2_up) < page_size) ++log2_up;
  p.page_mul = (uint32_t)((((uint64_t)1 << (31 + log2_up)) / (uint64_t)page_size) + 1);
  p.page_shr = log2_up;  // umulhi(2 t, mul) >> log2_up = (t * mul) >> (31 + log2_up)
  p.num_pages = (int)num_pages;
  p.max_pages = (int)max_pages_per_seq;
  p.same_strides = p.k0 == p.v0 && p.k1 == p.v1 && p.k2 == p.v2 && p.ks0 == p.vs0 && p.ks1 == p.vs1 && p.ks2 == p.vs2;
  const int64_t pairs = batch * (num_kv_heads / plan.hg);
  p.meta_by_pair = pairs < plan.partitions ? 1 : 0;
  p.scale_log2 = scale * kLog2e;
  if (weights != nullptr) {
    p.track.raw = reinterpret_cast<float*>(ws + plan.off_raw);
    p.track.tiles = reinterpret_cast<int4*>(ws + plan.off_tiles);
    p.track.norm = reinterpret_cast<float2*>(ws + plan.off_norm);
    p.track.total = reinterpret_cast<int*>(ws + plan.off_total);
    p.track.raw_tiles = (int)plan.raw_tiles;
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  {
    void* args[] = {&p};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)plan.partitions);
    cfg.blockDim = dim3((unsigned)in.threads);
    cfg.dynamicSmemBytes = (size_t)in.smem_bytes;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if ((e = cudaLaunchKernelExC(&cfg, in.kernel, args)) != cudaSuccess)
      return cuda_fail(e, "launching the decode_fp4 kernel");
  }
  if (plan.partitions > 1) {
    MergeLaunch m = {};
    m.ws_o = p.ws_o;
    m.ws_ml = p.ws_ml;
    m.ws_meta = p.ws_meta;
    m.out = p.out;
    m.out_sb = p.out_sb;
    m.out_sh = p.out_sh;
    m.ngroups = (int)(num_kv_heads / plan.hg);
    m.rows = (int)(gqa * plan.hg);
    m.guess_ncap = p.meta_by_pair ? (int)((max_pages_per_seq * page_size + kTile - 1) / kTile) : 0;
    m.guess_parts = (int)plan.partitions;
    m.batch = batch;
    m.partitions = plan.partitions;
    m.head_dim = head_dim;
    m.meta_by_pair = p.meta_by_pair;
    m.norm = p.track.norm;
    if ((st = launch_merge(m, s)) != PAD_OK) return st;
  }
  if (weights != nullptr) {
    WeightParams wp = {};
    wp.track = p.track;
    wp.block_table = block_table;
    wp.total_lens = total_lens;
    wp.num_new_of = num_new_of;
    wp.weights = weights;
    wp.slot_positions = slot_positions;
    wp.w0 = weight_strides[0];
    wp.w1 = weight_strides[1];
    wp.w2 = weight_strides[2];
    if (slot_positions != nullptr) {
      wp.p0 = position_strides[0];
      wp.p1 = position_strides[1];
      wp.p2 = position_strides[2];
    }
    wp.bt_stride = block_table_stride;
    wp.batch = (int)batch;
    wp.cap = (int)(max_pages_per_seq * page_size);
    wp.hg_log2 = p.hg_log2;
    wp.gqa = (int)gqa;
    wp.tt_log2 = __builtin_ctz((unsigned)kTile);
    wp.ngroups = (int)(num_kv_heads / plan.hg);
    wp.page_size = (int)page_size;
    wp.page_shift = (page_size & (page_size - 1)) == 0 ? __builtin_ctzll((unsigned long long)page_size) : -1;
    wp.num_pages = (int)num_pages;
    wp.num_new = (int)std::min<int64_t>(num_new, wp.cap);
    if ((st = launch_weights(wp, s)) != PAD_OK) return st;
  }
  return PAD_OK;
}

}  // namespace

extern "C" int pad_decode_fp4_workspace_bytes(int device, int64_t batch, int64_t num_kv_heads, int64_t gqa_ratio,
                                              int64_t head_dim, int64_t num_pages, int64_t page_size,
                                              int64_t max_pages_per_seq, int64_t num_splits, int with_weights,
                                              size_t* bytes) {
  if (bytes == nullptr) return fail(PAD_ERR_INVALID_ARGUMENT, "decode_fp4: null output pointer");
  Fp4Plan plan;
  const int st = make_plan(device, batch, num_kv_heads, gqa_ratio, head_dim, num_pages, page_size, max_pages_per_seq,
                           num_splits, with_weights != 0, &plan);
  if (st == PAD_OK) *bytes = plan.bytes;
  return st;
}

extern "C" int pad_paged_attention_decode_fp4(
    const void* q, const void* k_cache, const void* k_scales, const void* v_cache, const void* v_scales,
    const int32_t* block_table, const int32_t* seq_lens, void* out, float* weights, int32_t* slot_positions,
    const int32_t* total_lens, int64_t num_new, int64_t batch, int64_t num_q_heads, int64_t num_kv_heads,
    int64_t head_dim, int64_t num_pages, int64_t page_size, int64_t max_pages_per_seq, const int64_t* q_strides,
    const int64_t* k_strides, const int64_t* ks_strides, const int64_t* v_strides, const int64_t* vs_strides,
    int64_t block_table_stride, const int64_t* out_strides, const int64_t* weight_strides,
    const int64_t* position_strides, float scale, int64_t num_splits, void* workspace, size_t workspace_bytes,
    void* stream, int32_t* error_flags) {
  return decode_fp4(q, k_cache, k_scales, v_cache, v_scales, block_table, seq_lens, out, weights, slot_positions,
                    total_lens, num_new, nullptr, batch, num_q_heads, num_kv_heads, head_dim, num_pages, page_size,
                    max_pages_per_seq, q_strides, k_strides, ks_strides, v_strides, vs_strides, block_table_stride,
                    out_strides, weight_strides, position_strides, scale, num_splits, workspace, workspace_bytes,
                    stream, error_flags);
}

extern "C" int pad_paged_attention_decode_fp4_by_seq(
    const void* q, const void* k_cache, const void* k_scales, const void* v_cache, const void* v_scales,
    const int32_t* block_table, const int32_t* seq_lens, void* out, float* weights, int32_t* slot_positions,
    const int32_t* total_lens, const int32_t* num_new, int64_t batch, int64_t num_q_heads, int64_t num_kv_heads,
    int64_t head_dim, int64_t num_pages, int64_t page_size, int64_t max_pages_per_seq, const int64_t* q_strides,
    const int64_t* k_strides, const int64_t* ks_strides, const int64_t* v_strides, const int64_t* vs_strides,
    int64_t block_table_stride, const int64_t* out_strides, const int64_t* weight_strides,
    const int64_t* position_strides, float scale, int64_t num_splits, void* workspace, size_t workspace_bytes,
    void* stream, int32_t* error_flags) {
  if (batch > 0 && num_new == nullptr) return fail(PAD_ERR_INVALID_ARGUMENT, "decode_fp4: null num_new");
  return decode_fp4(q, k_cache, k_scales, v_cache, v_scales, block_table, seq_lens, out, weights, slot_positions,
                    total_lens, 0, num_new, batch, num_q_heads, num_kv_heads, head_dim, num_pages, page_size,
                    max_pages_per_seq, q_strides, k_strides, ks_strides, v_strides, vs_strides, block_table_stride,
                    out_strides, weight_strides, position_strides, scale, num_splits, workspace, workspace_bytes,
                    stream, error_flags);
}
