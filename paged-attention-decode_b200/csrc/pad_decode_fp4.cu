// pad_decode_fp4.cu -- decode attention over the 4-bit paged cache (format:
// pad_fp4.cuh). One CTA per (sequence, KV head): a warp takes every fourth
// token, a lane D/32 of its dims, for all G query heads, with an online softmax
// in base 2; the four warps' states are joined through shared memory. Attention
// weights take a second pass over K, when (M, L) is known.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdint>

#include "pad_b200.h"
#include "pad_error.cuh"
#include "pad_fp4.cuh"
#include "pad_ptx.cuh"

namespace {

using namespace pad;

constexpr int kWarps = 4;
constexpr int kMaxG = 16;

struct Params {
  const __half* q;
  const uint8_t *k, *ks, *v, *vs;
  const int32_t *block_table, *seq_lens, *total_lens;
  __half* out;
  float* weights;
  int32_t* slot_positions;
  int32_t* error_flags;
  int64_t q0, q1, k0, k1, k2, ks0, ks1, ks2, v0, v1, v2, vs0, vs1, vs2, o0, o1, w0, w1, w2, p0, p1, p2, bt_stride;
  int hkv, gqa, num_pages, page_size, max_pages, num_new;
  float scale_log2;
};

__device__ __forceinline__ float code_value(uint32_t n) {
  const float m = (float)(n & 7u);
  const float v = m <= 4.f ? 0.5f * m : (m == 7.f ? 6.f : m - 2.f);
  return (n & 8u) ? -v : v;
}

// This lane's D/32 dims of a row (at least one byte: D = 32 shares it).
template <int D>
__device__ __forceinline__ void row_values(const uint8_t* codes, const uint8_t* scales, int lane, float (&x)[D / 32]) {
  constexpr int E = D / 32;
  const int d0 = lane * E;
  const float f = fp4_scale_f32(scales[d0 / 32]);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const uint32_t b = codes[(d0 + e) / 2];
    x[e] = code_value(((d0 + e) & 1) ? b >> 4 : b & 15u) * f;
  }
}

template <int D>
__global__ void __launch_bounds__(32 * kWarps) decode_fp4_kernel(const __grid_constant__ Params p) {
  constexpr int E = D / 32;
  __shared__ float so[kWarps][D];
  __shared__ float sm[kWarps][kMaxG], sl[kWarps][kMaxG];
  const int b = blockIdx.x / p.hkv, h = blockIdx.x % p.hkv;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t cap = (int64_t)p.max_pages * p.page_size;
  const int raw = p.seq_lens[b];
  const int n = (int)min((int64_t)max(raw, 0), cap);
  if (raw != n && threadIdx.x == 0 && p.error_flags != nullptr) atomicOr(p.error_flags, PAD_FLAG_SEQ_LEN_RANGE);
  for (int g = 0; g < p.gqa; ++g) {
    const __half* qr = p.q + b * p.q0 + (int64_t)(h * p.gqa + g) * p.q1 + lane * E;
    float q[E], acc[E], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      q[e] = __half2float(qr[e]);
      acc[e] = 0.f;
    }
    auto page_of = [&](int t) {
      const int page = p.block_table[b * p.bt_stride + t / p.page_size];
      if ((unsigned)page < (unsigned)p.num_pages) return (int64_t)page;
      if (lane == 0 && p.error_flags != nullptr) atomicOr(p.error_flags, PAD_FLAG_BAD_PAGE_ID);
      return (int64_t)-1;
    };
    auto score = [&](int64_t page, int64_t row) {
      float x[E], s = 0.f;
      row_values<D>(p.k + page * p.k0 + row * p.k1 + h * p.k2, p.ks + page * p.ks0 + row * p.ks1 + h * p.ks2, lane, x);
#pragma unroll
      for (int e = 0; e < E; ++e) s += q[e] * x[e];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      return s * p.scale_log2;
    };
    for (int t = warp; t < n; t += kWarps) {
      const int64_t page = page_of(t), row = t % p.page_size;
      const float s = page < 0 ? 0.f : score(page, row);
      const float mn = fmaxf(m, s), mu = mn == -INFINITY ? 0.f : mn;
      const float al = ex2(m - mu), w = ex2(s - mu);
      float x[E] = {};
      if (page >= 0)
        row_values<D>(p.v + page * p.v0 + row * p.v1 + h * p.v2, p.vs + page * p.vs0 + row * p.vs1 + h * p.vs2, lane, x);
      l = l * al + w;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = acc[e] * al + w * x[e];
      m = mn;
    }
    if (lane == 0) {
      sm[warp][g] = m;
      sl[warp][g] = l;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) so[warp][lane * E + e] = acc[e];
    __syncthreads();
    float M = -INFINITY, L = 0.f;
    for (int x = 0; x < kWarps; ++x) M = fmaxf(M, sm[x][g]);
    const float Mu = M == -INFINITY ? 0.f : M;
    for (int x = 0; x < kWarps; ++x) L += sl[x][g] * ex2(sm[x][g] - Mu);
    const float inv = L == 0.f ? 0.f : 1.f / L;
    for (int d = threadIdx.x; d < D; d += 32 * kWarps) {
      float o = 0.f;
      for (int x = 0; x < kWarps; ++x) o += so[x][d] * ex2(sm[x][g] - Mu);
      p.out[b * p.o0 + (int64_t)(h * p.gqa + g) * p.o1 + d] = __float2half_rn(o * inv);
    }
    if (p.weights != nullptr) {
      for (int t = warp; t < n; t += kWarps) {
        const int64_t page = page_of(t), row = t % p.page_size;
        if (page < 0) continue;
        const float w = ex2(score(page, row) - Mu) * inv;
        if (lane != 0) continue;
        const bool fresh = t >= n - p.num_new;
        float* at = p.weights + page * p.w0 + h * p.w1 + row * p.w2;
        *at = fresh && g == 0 ? w : *at + w;
        if (fresh && p.slot_positions != nullptr)
          p.slot_positions[page * p.p0 + h * p.p1 + row * p.p2] = p.total_lens[b] - n + t;
      }
    }
    __syncthreads();
  }
}

bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

}  // namespace

extern "C" int pad_decode_fp4_workspace_bytes(int device, int64_t batch, int64_t num_kv_heads, int64_t gqa_ratio,
                                              int64_t head_dim, int64_t num_pages, int64_t page_size,
                                              int64_t max_pages_per_seq, int64_t num_splits, int with_weights,
                                              size_t* bytes) {
  if (bytes == nullptr) return fail(PAD_ERR_INVALID_ARGUMENT, "decode_fp4: null output pointer");
  *bytes = 256;
  return PAD_OK;
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
  if (num_pages > INT32_MAX || max_pages_per_seq > INT32_MAX || page_size > INT32_MAX ||
      max_pages_per_seq * page_size > INT32_MAX / 2 || batch > INT32_MAX / num_q_heads / 4)
    return fail(PAD_ERR_UNSUPPORTED, "%s: problem too large for 32-bit indexing", what);
  Params p = {};
  p.q = static_cast<const __half*>(q);
  p.k = static_cast<const uint8_t*>(k_cache);
  p.ks = static_cast<const uint8_t*>(k_scales);
  p.v = static_cast<const uint8_t*>(v_cache);
  p.vs = static_cast<const uint8_t*>(v_scales);
  p.block_table = block_table;
  p.seq_lens = seq_lens;
  p.total_lens = total_lens;
  p.out = static_cast<__half*>(out);
  p.weights = weights;
  p.slot_positions = slot_positions;
  p.error_flags = error_flags;
  p.q0 = q_strides[0], p.q1 = q_strides[1];
  p.k0 = k_strides[0], p.k1 = k_strides[1], p.k2 = k_strides[2];
  p.ks0 = ks_strides[0], p.ks1 = ks_strides[1], p.ks2 = ks_strides[2];
  p.v0 = v_strides[0], p.v1 = v_strides[1], p.v2 = v_strides[2];
  p.vs0 = vs_strides[0], p.vs1 = vs_strides[1], p.vs2 = vs_strides[2];
  p.o0 = out_strides[0], p.o1 = out_strides[1];
  if (weights != nullptr) p.w0 = weight_strides[0], p.w1 = weight_strides[1], p.w2 = weight_strides[2];
  if (slot_positions != nullptr) p.p0 = position_strides[0], p.p1 = position_strides[1], p.p2 = position_strides[2];
  p.bt_stride = block_table_stride;
  p.hkv = (int)num_kv_heads;
  p.gqa = (int)gqa;
  p.num_pages = (int)num_pages;
  p.page_size = (int)page_size;
  p.max_pages = (int)max_pages_per_seq;
  p.num_new = (int)std::min<int64_t>(num_new, INT32_MAX);
  p.scale_log2 = scale * 1.4426950408889634f;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const unsigned grid = (unsigned)(batch * num_kv_heads);
  if (head_dim == 32) decode_fp4_kernel<32><<<grid, 32 * kWarps, 0, s>>>(p);
  else if (head_dim == 64) decode_fp4_kernel<64><<<grid, 32 * kWarps, 0, s>>>(p);
  else decode_fp4_kernel<128><<<grid, 32 * kWarps, 0, s>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? PAD_OK : cuda_fail(e, "launching the decode_fp4 kernel");
}
