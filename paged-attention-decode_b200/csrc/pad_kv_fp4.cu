// pad_kv_fp4.cu -- writing tokens into the 4-bit paged cache and reading them
// back (format: pad_fp4.cuh). Tokens are given as (sequence, position) pairs,
// so one call covers a decoding step (one token of each sequence) as well as
// whole prompts.
//
// Per block of 32 values x along the head dim, with a = max |x|:
//   E = max(floor(log2 a) - 2, -24),  scale byte = E + 127,
//   code = e2m1(x / 2^E), rounded to nearest even, saturated at 6
// (floor(log2 a) - 2 puts a into [4, 8), e2m1's top binade). x / 2^E is exact
// in fp32, so the one rounding is the conversion's. A block with an Inf or NaN
// gets scale 255 (NaN) and zero codes. Every value that quantised fp16 stands
// for is an fp16 value again: E >= -24 keeps the half steps of a tiny block on
// fp16's own grid (such a block has integer multiples of 2^-24 below 4, which
// e2m1 holds exactly).
//
// Bound: the latency of three dependent loads (position, page id, row), alone for
// a step; for prompts (fp16 rows in, 4.25 bits a value out, or the other way round)
// it leaves HBM two thirds used, with instructions issued in 60% of the cycles. A thread owns 8 dims of the K and V rows of HU heads of one
// token (HU = 4, 2 or 1, what divides the heads): 16-byte loads, the block
// maximum by two shuffles among the four threads of a block, 4-byte stores. The
// heads share the look-up of the token's place, and their loads are in flight
// together. Measured on prompts of 8 sequences (20 thousand tokens, 8 heads,
// head_dim 128), written and read back: 46 us, 67% of the copy rate over both
// directions' bytes (67.6 us with one head a thread and fp32 arithmetic).
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdint>

#include "pad_b200.h"
#include "pad_error.cuh"
#include "pad_fp4.cuh"

namespace {

using namespace pad;

constexpr int kThreadsFp4 = 256;

struct Fp4Rows {  // strides in bytes for the cache, in elements for the fp16 rows
  int64_t s0, s1, s2;
};

struct Fp4Params {
  const __half *k_in, *v_in;    // append: new rows
  __half *k_out, *v_out;        // read: rows given back
  uint8_t *k, *ks, *v, *vs;
  const int32_t *block_table, *positions, *seq_ids;
  Fp4Rows k_st, ks_st, v_st, vs_st;
  int64_t kr_t, kr_h, vr_t, vr_h;  // token and head strides of the fp16 rows
  int64_t bt_stride;
  uint32_t rows;  // tokens x runs of HU heads
  int batch, hkv, num_pages, page_size, max_pages;
  int vec;                         // fp16 rows may be moved 16 bytes at a time
  int32_t* error_flags;
};

// Page and row of token t, or false (flagged, except for a negative position).
__device__ __forceinline__ bool locate(const Fp4Params& p, int64_t t, int64_t& page, int64_t& row, bool report) {
  const int pos = __ldg(p.positions + t);
  if (pos < 0) return false;
  const int64_t seq = p.seq_ids != nullptr ? (int64_t)__ldg(p.seq_ids + t) : t;
  const int lp = pos / p.page_size;
  int bad = 0;
  if (seq < 0 || seq >= p.batch) bad = PAD_FLAG_BAD_SEQ_ID;
  else if (lp >= p.max_pages) bad = PAD_FLAG_SEQ_LEN_RANGE;
  if (bad == 0) {
    page = __ldg(p.block_table + seq * p.bt_stride + lp);
    row = pos - lp * p.page_size;
    if (page < 0 || page >= p.num_pages) bad = PAD_FLAG_BAD_PAGE_ID;
  }
  if (bad != 0 && report && p.error_flags != nullptr) atomicOr(p.error_flags, bad);
  return bad == 0;
}

__device__ __forceinline__ uint4 load_row8(const __half* x, int vec) {
  if (vec) return __ldg(reinterpret_cast<const uint4*>(x));
  uint4 r;
  uint32_t* w = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = (uint32_t)__half_as_ushort(x[2 * i]) | ((uint32_t)__half_as_ushort(x[2 * i + 1]) << 16);
  return r;
}

// Quantises this thread's 8 values of a block whose other values the three
// threads beside it hold; every thread of the block gets the scale byte.
__device__ __forceinline__ uint32_t quantise8(const uint4& r, uint32_t& scale) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
  __half2 m[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) m[i] = __habs2(*reinterpret_cast<const __half2*>(&w[i]));
  // maxima that keep a NaN
  __half2 a2 = __hmax2_nan(__hmax2_nan(m[0], m[1]), __hmax2_nan(m[2], m[3]));
  a2 = __hmax2_nan(a2, __shfl_xor_sync(0xffffffffu, a2, 1));
  a2 = __hmax2_nan(a2, __shfl_xor_sync(0xffffffffu, a2, 2));
  const float top = __half2float(__hmax_nan(__low2half(a2), __high2half(a2)));
  const bool fine = top <= 65504.f;  // neither Inf nor NaN
  const int e = max((int)(__float_as_uint(top) >> 23) - 127 - 2, kFp4MinExp);
  scale = fine ? (uint32_t)(e + 127) : kFp4NanScale;
  const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
  float x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    x[2 * i] = f.x * inv;
    x[2 * i + 1] = f.y * inv;
  }
  return fine ? fp4_pack8(x) : 0u;
}

// A row's scale bytes, by the first thread of each block; the row's unused
// bytes become 0.
template <int D>
__device__ __forceinline__ void store_scale(uint8_t* row, int c, uint32_t scale) {
  if (c % 4 != 0) return;
  if constexpr (D == 32) {
    *reinterpret_cast<uint32_t*>(row) = scale;
  } else {
    row[c / 4] = (uint8_t)scale;
    if constexpr (D == 64) row[c / 4 + 2] = 0;
  }
}

template <int D, int HU>
__global__ void __launch_bounds__(kThreadsFp4) fp4_append_kernel(const __grid_constant__ Fp4Params p) {
  constexpr int LPR = D / 8;  // threads per row
  const uint32_t r = blockIdx.x * (kThreadsFp4 / LPR) + threadIdx.x / LPR;  // (token, run of HU heads)
  const int c = (int)(threadIdx.x % LPR);
  const uint32_t groups = p.hkv / HU;
  const bool on = r < p.rows;
  const int64_t t = on ? r / groups : 0;
  const int h0 = on ? (int)(r % groups) * HU : 0;
  const __half* kn = p.k_in + t * p.kr_t + h0 * p.kr_h + c * 8;
  const __half* vn = p.v_in + t * p.vr_t + h0 * p.vr_h + c * 8;
  uint4 kx[HU], vx[HU];
#pragma unroll
  for (int u = 0; u < HU; ++u) {
    kx[u] = vx[u] = make_uint4(0, 0, 0, 0);
    if (on) {
      kx[u] = load_row8(kn, p.vec);
      vx[u] = load_row8(vn, p.vec);
    }
    kn += p.kr_h;
    vn += p.vr_h;
  }
  int64_t page = 0, row = 0;
  const bool ok = on && locate(p, t, page, row, c == 0);
  uint8_t* ko = p.k + page * p.k_st.s0 + row * p.k_st.s1 + h0 * p.k_st.s2 + c * 4;
  uint8_t* vo = p.v + page * p.v_st.s0 + row * p.v_st.s1 + h0 * p.v_st.s2 + c * 4;
  uint8_t* kso = p.ks + page * p.ks_st.s0 + row * p.ks_st.s1 + h0 * p.ks_st.s2;
  uint8_t* vso = p.vs + page * p.vs_st.s0 + row * p.vs_st.s1 + h0 * p.vs_st.s2;
#pragma unroll
  for (int u = 0; u < HU; ++u) {
    uint32_t ksc, vsc;
    const uint32_t kc = quantise8(kx[u], ksc), vc = quantise8(vx[u], vsc);
    if (ok) {
      *reinterpret_cast<uint32_t*>(ko) = kc;
      *reinterpret_cast<uint32_t*>(vo) = vc;
      store_scale<D>(kso, c, ksc);
      store_scale<D>(vso, c, vsc);
    }
    ko += p.k_st.s2;
    vo += p.v_st.s2;
    kso += p.ks_st.s2;
    vso += p.vs_st.s2;
  }
}

// Four code bytes and their scale -> 8 fp16 values, rounded once (exact for
// every row that fp4_append_kernel wrote). A scale that fp16 holds, which is all
// the append writes, multiplies as fp16; any other goes through fp32.
__device__ __forceinline__ uint4 dequantise8(uint32_t codes, uint32_t scale) {
  uint32_t h[4];
  fp4_unpack4(codes, h[0], h[1], h[2], h[3]);
  const float f = fp4_scale_f32(scale);
  uint4 r;
  uint32_t* w = reinterpret_cast<uint32_t*>(&r);
  if (scale - 103u <= 39u) {  // 2^-24 .. 2^15
    const __half2 f2 = __float2half2_rn(f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 o = __hmul2(*reinterpret_cast<const __half2*>(&h[i]), f2);
      w[i] = *reinterpret_cast<const uint32_t*>(&o);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
      const __half2 o = __floats2half2_rn(v.x * f, v.y * f);
      w[i] = *reinterpret_cast<const uint32_t*>(&o);
    }
  }
  return r;
}

__device__ __forceinline__ void store_row8(__half* x, const uint4& r, int vec) {
  if (vec) {
    *reinterpret_cast<uint4*>(x) = r;
    return;
  }
  const uint32_t* w = reinterpret_cast<const uint32_t*>(&r);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __ushort_as_half((unsigned short)(w[i] & 0xffffu));
    x[2 * i + 1] = __ushort_as_half((unsigned short)(w[i] >> 16));
  }
}

template <int D, int HU>
__global__ void __launch_bounds__(kThreadsFp4) fp4_read_kernel(const __grid_constant__ Fp4Params p) {
  constexpr int LPR = D / 8;
  const uint32_t r = blockIdx.x * (kThreadsFp4 / LPR) + threadIdx.x / LPR;
  const int c = (int)(threadIdx.x % LPR);
  if (r >= p.rows) return;
  const uint32_t groups = p.hkv / HU;
  const int64_t t = r / groups;
  const int h0 = (int)(r % groups) * HU;
  int64_t page = 0, row = 0;
  uint32_t kc[HU], vc[HU], ks[HU], vs[HU];
  const bool ok = locate(p, t, page, row, c == 0);
  const uint8_t* ki = p.k + page * p.k_st.s0 + row * p.k_st.s1 + h0 * p.k_st.s2 + c * 4;
  const uint8_t* vi = p.v + page * p.v_st.s0 + row * p.v_st.s1 + h0 * p.v_st.s2 + c * 4;
  const uint8_t* ksi = p.ks + page * p.ks_st.s0 + row * p.ks_st.s1 + h0 * p.ks_st.s2 + c / 4;
  const uint8_t* vsi = p.vs + page * p.vs_st.s0 + row * p.vs_st.s1 + h0 * p.vs_st.s2 + c / 4;
#pragma unroll
  for (int u = 0; u < HU; ++u) {
    kc[u] = vc[u] = 0;  // a token without a place reads as zero
    ks[u] = vs[u] = 127;
    if (ok) {
      kc[u] = *reinterpret_cast<const uint32_t*>(ki);
      vc[u] = *reinterpret_cast<const uint32_t*>(vi);
      ks[u] = *ksi;
      vs[u] = *vsi;
    }
    ki += p.k_st.s2;
    vi += p.v_st.s2;
    ksi += p.ks_st.s2;
    vsi += p.vs_st.s2;
  }
  __half* kr = p.k_out + t * p.kr_t + h0 * p.kr_h + c * 8;
  __half* vr = p.v_out + t * p.vr_t + h0 * p.vr_h + c * 8;
#pragma unroll
  for (int u = 0; u < HU; ++u) {
    store_row8(kr, dequantise8(kc[u], ks[u]), p.vec);
    store_row8(vr, dequantise8(vc[u], vs[u]), p.vec);
    kr += p.kr_h;
    vr += p.vr_h;
  }
}

bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// The arguments that both entry points share, checked and put into `p`.
int fill(Fp4Params* p, const char* what, const void* k_rows, const void* v_rows, void* k_cache, void* k_scales,
         void* v_cache, void* v_scales, const int32_t* block_table, const int32_t* positions, const int32_t* seq_ids,
         int64_t tokens, int64_t batch, int64_t num_kv_heads, int64_t head_dim, int64_t num_pages, int64_t page_size,
         int64_t max_pages, const int64_t* kr, const int64_t* vr, const int64_t* k, const int64_t* ks,
         const int64_t* v, const int64_t* vs, int64_t bt_stride, int32_t* error_flags) {
  // a pool or a table of nothing has no address: its tokens are flagged before one is needed
  if (k_rows == nullptr || v_rows == nullptr || positions == nullptr ||
      (num_pages > 0 && (k_cache == nullptr || k_scales == nullptr || v_cache == nullptr || v_scales == nullptr)) ||
      (batch > 0 && max_pages > 0 && block_table == nullptr) || kr == nullptr || vr == nullptr || k == nullptr ||
      ks == nullptr || v == nullptr || vs == nullptr)
    return fail(PAD_ERR_INVALID_ARGUMENT, "%s: null pointer argument", what);
  if (seq_ids == nullptr && tokens > batch)
    return fail(PAD_ERR_INVALID_ARGUMENT, "%s: %lld tokens for %lld sequences need seq_ids", what, (long long)tokens,
                (long long)batch);
  if (bt_stride < max_pages)
    return fail(PAD_ERR_INVALID_ARGUMENT, "%s: block_table row stride smaller than its width", what);
  if (kr[2] != 1 || vr[2] != 1 || k[3] != 1 || ks[3] != 1 || v[3] != 1 || vs[3] != 1)
    return fail(PAD_ERR_UNSUPPORTED, "%s: the last axis of every tensor must be contiguous", what);
  for (int i = 0; i < 3; ++i)
    if (k[i] % 16 || v[i] % 16 || ks[i] % kFp4ScaleRow || vs[i] % kFp4ScaleRow)
      return fail(PAD_ERR_UNSUPPORTED, "%s: code strides must be multiples of 16 bytes, scale strides of 4", what);
  if (!aligned(k_cache, 16) || !aligned(v_cache, 16) || !aligned(k_scales, 4) || !aligned(v_scales, 4))
    return fail(PAD_ERR_UNSUPPORTED, "%s: codes must be 16-byte aligned, scales 4-byte aligned", what);
  if (num_pages > INT32_MAX || batch > INT32_MAX || num_kv_heads > INT32_MAX || page_size > INT32_MAX ||
      max_pages > INT32_MAX || tokens > INT32_MAX / num_kv_heads)
    return fail(PAD_ERR_UNSUPPORTED, "%s: sizes exceed the kernels' indexing", what);
  p->k = static_cast<uint8_t*>(k_cache);
  p->ks = static_cast<uint8_t*>(k_scales);
  p->v = static_cast<uint8_t*>(v_cache);
  p->vs = static_cast<uint8_t*>(v_scales);
  p->block_table = block_table;
  p->positions = positions;
  p->seq_ids = seq_ids;
  p->k_st = {k[0], k[1], k[2]};
  p->ks_st = {ks[0], ks[1], ks[2]};
  p->v_st = {v[0], v[1], v[2]};
  p->vs_st = {vs[0], vs[1], vs[2]};
  p->kr_t = kr[0];
  p->kr_h = kr[1];
  p->vr_t = vr[0];
  p->vr_h = vr[1];
  p->bt_stride = bt_stride;
  p->batch = (int)batch;
  p->hkv = (int)num_kv_heads;
  p->num_pages = (int)num_pages;
  p->page_size = (int)page_size;
  p->max_pages = (int)max_pages;
  p->vec = aligned(k_rows, 16) && aligned(v_rows, 16) && kr[0] % 8 == 0 && kr[1] % 8 == 0 && vr[0] % 8 == 0 &&
           vr[1] % 8 == 0;
  p->error_flags = error_flags;
  return PAD_OK;
}

int check_sizes(const char* what, int64_t tokens, int64_t batch, int64_t num_kv_heads, int64_t head_dim,
                int64_t num_pages, int64_t page_size, int64_t max_pages) {
  if (tokens < 0 || batch < 0 || num_kv_heads <= 0 || num_pages < 0 || page_size <= 0 || max_pages < 0)
    return fail(PAD_ERR_INVALID_ARGUMENT, "%s: negative or zero size", what);
  if (head_dim != 32 && head_dim != 64 && head_dim != 128)
    return fail(PAD_ERR_UNSUPPORTED, "%s: head_dim %lld not supported (32, 64 or 128)", what, (long long)head_dim);
  return PAD_OK;
}

using Fp4Kernel = void (*)(const Fp4Params);

// [head_dim 32, 64, 128][heads a thread 1, 2, 4]
constexpr Fp4Kernel kAppend[3][3] = {
    {fp4_append_kernel<32, 1>, fp4_append_kernel<32, 2>, fp4_append_kernel<32, 4>},
    {fp4_append_kernel<64, 1>, fp4_append_kernel<64, 2>, fp4_append_kernel<64, 4>},
    {fp4_append_kernel<128, 1>, fp4_append_kernel<128, 2>, fp4_append_kernel<128, 4>}};
constexpr Fp4Kernel kRead[3][3] = {{fp4_read_kernel<32, 1>, fp4_read_kernel<32, 2>, fp4_read_kernel<32, 4>},
                                   {fp4_read_kernel<64, 1>, fp4_read_kernel<64, 2>, fp4_read_kernel<64, 4>},
                                   {fp4_read_kernel<128, 1>, fp4_read_kernel<128, 2>, fp4_read_kernel<128, 4>}};

int launch(Fp4Params& p, int64_t tokens, int64_t head_dim, const Fp4Kernel (&kernels)[3][3], void* stream,
           const char* what) {
  const int heads = p.hkv % 4 == 0 ? 2 : p.hkv % 2 == 0 ? 1 : 0;  // log2 of HU
  p.rows = (uint32_t)(tokens * (p.hkv >> heads));
  const int64_t threads = (int64_t)p.rows * (head_dim / 8);
  const unsigned blocks = (unsigned)((threads + kThreadsFp4 - 1) / kThreadsFp4);
  kernels[head_dim == 32 ? 0 : head_dim == 64 ? 1 : 2][heads]<<<blocks, kThreadsFp4, 0,
                                                               static_cast<cudaStream_t>(stream)>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? PAD_OK : cuda_fail(e, what);
}

}  // namespace

extern "C" int pad_paged_kv_append_fp4(const void* k_new, const void* v_new, void* k_cache, void* k_scales,
                                       void* v_cache, void* v_scales, const int32_t* block_table,
                                       const int32_t* positions, const int32_t* seq_ids, int64_t tokens, int64_t batch,
                                       int64_t num_kv_heads, int64_t head_dim, int64_t num_pages, int64_t page_size,
                                       int64_t max_pages_per_seq, const int64_t* k_new_strides,
                                       const int64_t* v_new_strides, const int64_t* k_strides,
                                       const int64_t* ks_strides, const int64_t* v_strides, const int64_t* vs_strides,
                                       int64_t block_table_stride, void* stream, int32_t* error_flags) {
  int st = check_sizes("kv_append_fp4", tokens, batch, num_kv_heads, head_dim, num_pages, page_size, max_pages_per_seq);
  if (st != PAD_OK || tokens == 0) return st;
  Fp4Params p = {};
  st = fill(&p, "kv_append_fp4", k_new, v_new, k_cache, k_scales, v_cache, v_scales, block_table, positions, seq_ids,
            tokens, batch, num_kv_heads, head_dim, num_pages, page_size, max_pages_per_seq, k_new_strides,
            v_new_strides, k_strides, ks_strides, v_strides, vs_strides, block_table_stride, error_flags);
  if (st != PAD_OK) return st;
  p.k_in = static_cast<const __half*>(k_new);
  p.v_in = static_cast<const __half*>(v_new);
  return launch(p, tokens, head_dim, kAppend, stream, "launching the kv_append_fp4 kernel");
}

extern "C" int pad_paged_kv_read_fp4(const void* k_cache, const void* k_scales, const void* v_cache,
                                     const void* v_scales, const int32_t* block_table, const int32_t* positions,
                                     const int32_t* seq_ids, void* k_out, void* v_out, int64_t tokens, int64_t batch,
                                     int64_t num_kv_heads, int64_t head_dim, int64_t num_pages, int64_t page_size,
                                     int64_t max_pages_per_seq, const int64_t* k_strides, const int64_t* ks_strides,
                                     const int64_t* v_strides, const int64_t* vs_strides,
                                     const int64_t* k_out_strides, const int64_t* v_out_strides,
                                     int64_t block_table_stride, void* stream, int32_t* error_flags) {
  int st = check_sizes("kv_read_fp4", tokens, batch, num_kv_heads, head_dim, num_pages, page_size, max_pages_per_seq);
  if (st != PAD_OK || tokens == 0) return st;
  Fp4Params p = {};
  st = fill(&p, "kv_read_fp4", k_out, v_out, const_cast<void*>(k_cache), const_cast<void*>(k_scales),
            const_cast<void*>(v_cache), const_cast<void*>(v_scales), block_table, positions, seq_ids, tokens, batch,
            num_kv_heads, head_dim, num_pages, page_size, max_pages_per_seq, k_out_strides, v_out_strides, k_strides,
            ks_strides, v_strides, vs_strides, block_table_stride, error_flags);
  if (st != PAD_OK) return st;
  p.k_out = static_cast<__half*>(k_out);
  p.v_out = static_cast<__half*>(v_out);
  return launch(p, tokens, head_dim, kRead, stream, "launching the kv_read_fp4 kernel");
}
