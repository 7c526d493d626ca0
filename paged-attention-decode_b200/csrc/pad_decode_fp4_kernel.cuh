// pad_decode_fp4_kernel.cuh -- decode attention over the 4-bit paged cache
// (format: pad_fp4.cuh), the split-K phase; merge_kernel joins its partials.
//
// Work unit: a tile of 32 tokens of a head group of HG KV heads. The batch is
// one list of tiles ordered (sequence, head group, tile) and every CTA takes an
// equal contiguous range of it, as the fp16 decode does.
//
// At 4.25 bits a value the arithmetic is as close to the limit as the copy (an
// SM is sent about 43 values a clock at full bandwidth, and every one has to
// become fp16), so the kernel is built around the fewest instructions a value:
//   - A warp owns whole (tile, head) pieces: WPH = warps / HG warps share a
//     head and take turns at its tiles. It copies its own pieces into its own
//     ring with cp.async and waits for nobody: no producer, and barriers between
//     the warps of a head only where a (sequence, head group) ends.
//   - Codes go from shared memory to registers by ldmatrix on 16-bit units of
//     four codes. For K a lane gets 8 consecutive dims of its row, for V
//     (transposed) four dims of two neighbouring tokens. The order in which a
//     contraction runs through its index is free, so Q is loaded in the order
//     K's bytes come out in and no code is ever moved to another lane.
//   - One conversion instruction makes two fp16 values of a code byte, exactly.
//   - K's scales are powers of two of 32 dims and leave the sum: the tensor
//     cores add up each block by itself, and the block's sum is scaled in fp32
//     (with the softmax scale folded in). V's scales differ along the
//     contraction and go onto the values, one packed multiplication for two.
//     Both are unpacked once per token through shared memory.
//   - P is split into two fp16 terms as in the fp16 decode.
// Rows of tokens past the sequence, and of pages that are none, are copied as
// zeros (cp.async with no source bytes): zero codes with a finite scale, so
// nothing that a page holds behind its sequence reaches the sums.
// V's scales go onto codes in fp16, exactly for 2^-24 .. 2^13, all that the append
// writes. Smaller ones become 0; a larger one would make codes infinite and is flagged.
//
// Measured (12/2 heads, head_dim 128, page 16): 64 x 4096 tokens 25.1 us a call
// (10.9 at the measured copy rate), each further 4096 tokens of the 64 sequences
// 14.4 us (75% of the copy rate); one sequence of 131072 tokens 16.4 us (5.4).
// About 630 instructions a piece of 32 tokens; the schedulers issue in 59% of the
// cycles and the integer pipe, which also converts, is busy in 52%. No unit is
// full: with three warps a scheduler it is latency, and some 10 us of a call do not
// depend on its length.
#pragma once

#include <cfloat>
#include <climits>

#include "pad_b200.h"
#include "pad_decode_kernel.cuh"
#include "pad_fp4.cuh"

namespace pad {

constexpr int kFp4SeqCache = 512;  // seq_lens kept in shared memory

struct Fp4DecodeParams {
  const __half* q;
  const uint8_t *k, *ks, *v, *vs;
  const int32_t *block_table, *seq_lens;
  __half* out;
  float* ws_o;      // as in DecodeParams
  float2* ws_ml;
  int4* ws_meta;
  int32_t* error_flags;
  int64_t q0, q1, out_sb, out_sh;
  // Offsets fit 32 bits: code strides in units of `unit` bytes, scale strides in
  // words of 4.
  uint32_t k0, k1, k2, v0, v1, v2, ks0, ks1, ks2, vs0, vs1, vs2, unit;
  // token / page_size = umulhi(2 * token, page_mul) >> page_shr, for tokens below 2^31
  uint32_t page_mul, page_shr;
  int batch, hkv, gqa, hg_log2, page_size, num_pages, max_pages, bt_stride;
  int same_strides;  // K and V have the same ones
  int meta_by_pair;
  float scale_log2;
  TrackParams track;
};

// Where a running maximum starts: at or below every score, and finite, so that a
// difference to it is never NaN.
constexpr float kLeastScore = -FLT_MAX;
// How far (in log2 units) a score may pass the reference point before it moves.
constexpr float kSlack = 8.f;

template <int D_, int NT_, bool WT_>
struct Fp4Traits {
  static constexpr int D = D_, NT = NT_;
  static constexpr bool WT = WT_;
  // Warps: 12 of 168 registers, 8 of 255 for two query tiles. When this was chosen
  // (64 x 4096, 12/2 heads) 12 took 28.5 us; 16 of 128 registers 29.4, with 70 more
  // instructions a tile to recompute addresses; 8, two a scheduler, 30.8.
  static constexpr int NW = NT == 1 ? 12 : 8;
  static constexpr int THREADS = 32 * NW;
  static constexpr int TT = 32;                    // tokens per tile
  static constexpr int NB = D / kFp4Block;         // blocks of 32 dims
  static constexpr int ROW = D / 2;                // code bytes of a row
  static constexpr int CPR = ROW / 16;             // 16-byte chunks of a row
  static constexpr int CODES = TT * ROW;
  static constexpr int STAGE = 2 * CODES + 2 * TT * kFp4ScaleRow;
  // about 150 KB of ring: two or three pieces in flight per warp at D = 128
  static constexpr int FIT = (NT == 1 ? 156672 : 139264) / NW / STAGE;
  static constexpr int STAGES = FIT > 6 ? 6 : FIT;
  static_assert(STAGES >= 2, "the ring needs two stages");
  static constexpr int SCRATCH = TT * 16 + TT / 2 * 16;  // unpacked scales of K (fp32) and V (fp16 pairs)
  static constexpr int LD = D + 4;                 // padded row of the epilogue
  static constexpr int ROWS = 8 * NT;              // query rows a head holds
  static constexpr int OFF_SCRATCH = NW * STAGES * STAGE;
  static constexpr int OFF_EPI = OFF_SCRATCH + NW * SCRATCH;
  static constexpr int OFF_ML = OFF_EPI + NW * ROWS * LD * 4;
  static constexpr int OFF_MISC = OFF_ML + NW * ROWS * 8;
  static constexpr int SMEM_BYTES = OFF_MISC + 256 + kFp4SeqCache * 4 + 128 /*align slack*/;
  static_assert(SMEM_BYTES <= kSmemBudget, "shared memory");
  // XOR on a row's chunk index that spreads ldmatrix's 8 rows over all banks
  __device__ static __forceinline__ uint32_t swz(uint32_t row) {
    if constexpr (CPR == 4) return (row >> 1) & 3u;
    else if constexpr (CPR == 2) return (row >> 2) & 1u;
    else return 0u;
  }
};

__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, uint32_t bytes, uint64_t policy) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(dst), "l"(src), "r"(bytes),
               "l"(policy)
               : "memory");
}
__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, uint64_t policy) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "l"(policy)
               : "memory");
}
__device__ __forceinline__ void cp_async_4(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// Position in the flattened (sequence, head group, tile) list.
struct Fp4Cursor {
  int b, hg, i, n, seq;  // tile i of n of the pair
  int start;             // global index of the pair's tile 0
};

template <class TR>
struct Fp4Walk {
  const Fp4DecodeParams& p;
  const int* sseq;
  int cap, ngroups;
  __device__ __forceinline__ int seq_at(int b) const {
    return b < kFp4SeqCache ? sseq[b] : clamp_seq(__ldg(p.seq_lens + b), cap);
  }
  __device__ __forceinline__ void next_pair(Fp4Cursor& c) const {
    c.start += c.n;
    if (++c.hg < ngroups) return;
    c.hg = 0;
    do {
      if (++c.b >= p.batch) {
        c.n = 0;
        return;
      }
      c.seq = seq_at(c.b);
      c.n = (c.seq + TR::TT - 1) / TR::TT;
    } while (c.n == 0);
  }
  // Steps on by `step` tiles; past the end n = 0.
  __device__ __forceinline__ void advance(Fp4Cursor& c, int step) const {
    c.i += step;
    while (c.n > 0 && c.i >= c.n) {
      c.i -= c.n;
      next_pair(c);
    }
  }
};

// Flags scales of V above 2^13 among the NB of the scale row at shared address `row`
// (NaN is none). Out of line: 64 x 16384 68.3 us so, 68.5 inside the loop, 67.8 unchecked.
template <int NB>
__device__ __noinline__ void flag_high_scales(const Fp4DecodeParams& p, uint32_t row) {
  uint32_t vw;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(vw) : "r"(row));
#pragma unroll
  for (int blk = 0; blk < NB; ++blk) {
    const uint32_t byte = (vw >> (8 * blk)) & 255u;
    if (byte > 140u && byte != kFp4NanScale && p.error_flags != nullptr) atomicOr(p.error_flags, PAD_FLAG_SCALE_RANGE);
  }
}

template <class TR>
__global__ void __launch_bounds__(TR::THREADS, 1) decode_fp4_kernel(const __grid_constant__ Fp4DecodeParams p) {
  constexpr int D = TR::D, NT = TR::NT, NB = TR::NB, S = TR::STAGES, TT = TR::TT, NW = TR::NW;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~uintptr_t(127));
  float* epi = reinterpret_cast<float*>(smem + TR::OFF_EPI);      // [warp][ROWS][LD]
  float2* sml = reinterpret_cast<float2*>(smem + TR::OFF_ML);     // [warp][ROWS]
  int* scan = reinterpret_cast<int*>(smem + TR::OFF_MISC);        // [16]
  int* cur = scan + 16;                                           // the first cursor
  int* sseq = scan + 64;                                          // [kFp4SeqCache]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cap = p.max_pages * p.page_size;
  const int64_t W = gridDim.x;
  const int w = blockIdx.x, G = p.gqa, HG = 1 << p.hg_log2, ngroups = p.hkv >> p.hg_log2;
  const int WPH = NW >> p.hg_log2;          // warps that share a head
  const int hl = warp / WPH, turn = warp - hl * WPH;
  const Fp4Walk<TR> walk{p, sseq, cap, ngroups};

  if (tid == 0) cur[0] = -1;
  pdl_wait_primary();

  // ---- tiles per sequence, scanned: this CTA's range and its first cursor
  int t0, t1, total = 0;
  {
    const int per = (p.batch + TR::THREADS - 1) / TR::THREADS;
    const int lo = min(p.batch, tid * per), hi = min(p.batch, lo + per);
    int local = 0, bad = 0, none = 0;
    for (int b = lo; b < hi; ++b) {
      const int raw = __ldg(p.seq_lens + b), sq = clamp_seq(raw, cap);
      bad |= raw != sq;
      none |= sq == 0;
      if (b < kFp4SeqCache) sseq[b] = sq;
      local += (sq + TT - 1) / TT;
    }
    local *= ngroups;
    int incl = local;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    if (lane == 31) scan[warp] = incl;
    none = __syncthreads_or(none);
    int excl = incl - local;
#pragma unroll
    for (int x = 0; x < NW; ++x) {
      const int v = scan[x];
      if (x < warp) excl += v;
      total += v;
    }
    if (bad && w == 0 && p.error_flags != nullptr) atomicOr(p.error_flags, PAD_FLAG_SEQ_LEN_RANGE);
    t0 = total > 0 ? part_begin(w, total, W) : 0;
    t1 = total > 0 ? part_begin(w + 1, total, W) : 0;
    if (t0 < total && excl <= t0 && t0 < excl + local) {
      int acc = excl;
      for (int b = lo; b < hi; ++b) {
        const int seq = walk.seq_at(b), n = (seq + TT - 1) / TT;
        if (t0 < acc + n * ngroups) {
          const int o = t0 - acc;
          cur[0] = b;
          cur[1] = o / n;
          cur[2] = o % n;
          cur[3] = n;
          cur[4] = seq;
          cur[5] = acc + (o / n) * n;
          break;
        }
        acc += n * ngroups;
      }
    }
    __syncthreads();
    pdl_launch_dependents();
    if (tid == 0) {
      if (!p.meta_by_pair) p.ws_meta[w] = make_int4(-1, 0, 0, 0);
      if constexpr (TR::WT) {
        if (w == 0) *p.track.total = total;
      }
    }
    // empty sequences: zero output rows, no merge
    for (int b = w; none && b < p.batch; b += (int)W) {
      if (walk.seq_at(b) != 0) continue;
      if (p.meta_by_pair)
        for (int x = tid; x < ngroups; x += TR::THREADS) p.ws_meta[b * ngroups + x] = make_int4(-1, 0, 0, 0);
      for (int x = tid; x < p.hkv * G * (D / 2); x += TR::THREADS)
        *reinterpret_cast<__half2*>(p.out + b * p.out_sb + (x / (D / 2)) * p.out_sh + (x % (D / 2)) * 2) =
            __floats2half2_rn(0.f, 0.f);
    }
  }
  Fp4Cursor seg{cur[0], cur[1], cur[2], cur[3], cur[4], cur[5]};
  if (t1 <= t0) {
    // an empty partition may still lie between those of a split pair: its
    // partial there is empty
    if (seg.b >= 0 && seg.start < t0)
      for (int x = tid; x < HG * G; x += TR::THREADS)
        p.ws_ml[(int64_t)(seg.b * ngroups + seg.hg + w) * HG * G + x] = make_float2(-INFINITY, 0.f);
    return;
  }

  // ---- this warp's ring and its copies
  const uint32_t ring = smem_u32(smem) + warp * (S * TR::STAGE);
  const uint32_t scratch = smem_u32(smem + TR::OFF_SCRATCH) + warp * TR::SCRATCH;
  const uint64_t policy = l2_evict_first_policy();
  const uint32_t chunk = lane % TR::CPR, row_of_lane = lane / TR::CPR;
  const uint32_t copy_dst = row_of_lane * TR::ROW + ((chunk ^ TR::swz(row_of_lane)) << 4);
  // Where this lane's token of a tile lies: its page (-1: it has no token) and
  // row, and the tile. Page ids are loaded a turn before the copy that needs them.
  struct Place {
    int page, row, left;  // left: tokens of the sequence from the tile's first on (0: no tile)
    uint32_t head;
  };
  Fp4Cursor ld = seg;                  // the pair of the tile looked up last
  int ld_t = t0 + turn - WPH;          // that tile (before the first: a turn ahead of it)
  int ld_tok = (seg.i + turn - WPH) * TT + lane;  // this lane's token in it
  const int32_t* ids = p.block_table + (int64_t)ld.b * p.bt_stride;  // page ids of its sequence
  // From the place of one tile of this warp to that of its next.
  auto place = [&](Place& o) {
    ld_t += WPH;
    ld_tok += WPH * TT;
    o.left = 0;
    if (ld_t >= t1) return;
    if (ld_tok - lane >= ld.seq) {  // another pair
      ld.i = (ld_tok - lane) / TT;
      walk.advance(ld, 0);
      ld_tok = ld.i * TT + lane;
      ids = p.block_table + (int64_t)ld.b * p.bt_stride;
    }
    const int lp = __umulhi(2u * (uint32_t)ld_tok, p.page_mul) >> p.page_shr;
    o.row = ld_tok - lp * p.page_size;
    o.left = ld.seq - (ld_tok - lane);
    o.head = ld.hg * HG + hl;
    o.page = ld_tok < ld.seq ? ld_nc_early(ids + lp) : -1;
  };
  bool bad_page = false;
  const uint8_t *k_chunk = p.k + chunk * 16, *v_chunk = p.v + chunk * 16;
  auto copy = [&](const Place& at, int stage) {
    if (at.left > 0) {
      const bool ok = (unsigned)at.page < (unsigned)p.num_pages;
      const uint32_t pg = ok ? at.page : 0, rw = ok ? at.row : 0;
      const uint32_t ko = pg * p.k0 + rw * p.k1 + at.head * p.k2;
      const uint32_t kso = pg * p.ks0 + rw * p.ks1 + at.head * p.ks2;
      const uint32_t dst = ring + stage * TR::STAGE + copy_dst;
      const uint32_t sdst = ring + stage * TR::STAGE + 2 * TR::CODES + lane * kFp4ScaleRow;
      constexpr int STEP = 32 / TR::CPR;  // rows between a lane's chunks
      const uint32_t good = __ballot_sync(0xffffffffu, ok);
      if (good == 0xffffffffu && p.same_strides) {
        // a whole tile, offsets of K and V alike: nearly always
#pragma unroll
        for (int x = 0; x < TR::CPR; ++x) {
          const uint32_t o = __shfl_sync(0xffffffffu, ko, row_of_lane + x * STEP);
          cp_async_16(dst + x * STEP * TR::ROW, k_chunk + (uint64_t)o * p.unit, policy);
          cp_async_16(dst + TR::CODES + x * STEP * TR::ROW, v_chunk + (uint64_t)o * p.unit, policy);
        }
        cp_async_4(sdst, p.ks + (uint64_t)kso * 4u, 4u);
        cp_async_4(sdst + TT * kFp4ScaleRow, p.vs + (uint64_t)kso * 4u, 4u);
      } else {
        bad_page |= !ok && lane < at.left;
        const uint32_t vo = pg * p.v0 + rw * p.v1 + at.head * p.v2;
        const uint32_t vso = pg * p.vs0 + rw * p.vs1 + at.head * p.vs2;
#pragma unroll 1
        for (int x = 0; x < TR::CPR; ++x) {
          const int r = row_of_lane + x * STEP;
          const uint32_t kr = __shfl_sync(0xffffffffu, ko, r), vr = __shfl_sync(0xffffffffu, vo, r);
          const uint32_t bytes = ((good >> r) & 1u) << 4;
          cp_async_16(dst + x * STEP * TR::ROW, k_chunk + (uint64_t)kr * p.unit, bytes, policy);
          cp_async_16(dst + TR::CODES + x * STEP * TR::ROW, v_chunk + (uint64_t)vr * p.unit, bytes, policy);
        }
        cp_async_4(sdst, p.ks + (uint64_t)kso * 4u, ok ? 4u : 0u);
        cp_async_4(sdst + TT * kFp4ScaleRow, p.vs + (uint64_t)vso * 4u, ok ? 4u : 0u);
      }
    }
    cp_async_commit();
  };
  Place next;
  {
    Place at[S];
#pragma unroll
    for (int s = 0; s < S - 1; ++s) place(at[s]);
    place(next);
#pragma unroll
    for (int s = 0; s < S - 1; ++s) copy(at[s], s);
  }

  // ldmatrix addresses of this lane within a tile's codes: rows 0-7 and 8-15 of
  // one chunk, then of the next (a row of one chunk: rows 0-31)
  uint32_t mat[NB >= 2 ? NB / 2 : 1];
  if constexpr (NB >= 2) {
    const uint32_t r = (lane & 7) + ((lane >> 3) & 1) * 8;
#pragma unroll
    for (int jj = 0; jj < NB / 2; ++jj) mat[jj] = r * TR::ROW + (((2 * jj + (lane >> 4)) ^ TR::swz(r)) << 4);
  } else {
    mat[0] = lane * TR::ROW;
  }
  // codes of blocks 2jj and 2jj + 1 (or the one) of the 16 tokens m: lower and upper 8 rows of each
  const int gl = lane >> 2, tl = lane & 3;

  uint32_t qf[NT][NB][4];
  auto load_q = [&](const Fp4Cursor& c) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int g = nt * 8 + gl;
      const __half* qr = p.q + c.b * p.q0 + (int64_t)((c.hg * HG + hl) * G + g) * p.q1 + 8 * tl;
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        uint4 x = make_uint4(0, 0, 0, 0);
        if (g < G) x = __ldg(reinterpret_cast<const uint4*>(qr + j * 32));
        qf[nt][j][0] = x.x;
        qf[nt][j][1] = x.y;
        qf[nt][j][2] = x.z;
        qf[nt][j][3] = x.w;
      }
    }
  };
  load_q(seg);

  float acc[NB][2][NT][4];
  float m_run[NT][2], l_run[NT][2];
  int k = t0 + turn, stage = 0;  // this warp's next tile and its ring slot
  int seg_t = t0;                // first tile of the segment in this CTA
  for (;;) {
    const int seg_end = min(t1, seg.start + seg.n);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m_run[nt][0] = m_run[nt][1] = kLeastScore;
      l_run[nt][0] = l_run[nt][1] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) acc[j][x][nt][0] = acc[j][x][nt][1] = acc[j][x][nt][2] = acc[j][x][nt][3] = 0.f;

    for (; k < seg_end; k += WPH) {
      cp_async_wait_group<S - 2>();
      __syncwarp();
      const uint32_t kb = ring + stage * TR::STAGE, vb = kb + TR::CODES, sb = vb + TR::CODES;
      const int tok0 = (k - seg.start) * TT, nv = seg.seq - tok0;
      // ---- scales, a lane per token: K's blocks in fp32 with the softmax scale
      // and log2 e folded in, V's as fp16, laid out as the fragments want them:
      // pairs of neighbouring tokens
      bool high;  // a scale of V is above 2^13 or NaN
      {
        uint32_t kw, vw;
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(kw) : "r"(sb + lane * 4));
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(vw) : "r"(sb + TT * 4 + lane * 4));
        const uint32_t k01 = fp4_scale2_bf16(kw), k23 = fp4_scale2_bf16(kw >> 16);
        const uint32_t w01 = fp4_scale2_bf16(vw), w23 = fp4_scale2_bf16(vw >> 16);
        const float kf[4] = {__uint_as_float(k01 << 16) * p.scale_log2, __uint_as_float(k01 & 0xffff0000u) * p.scale_log2,
                             __uint_as_float(k23 << 16) * p.scale_log2, __uint_as_float(k23 & 0xffff0000u) * p.scale_log2};
        asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(scratch + lane * 16), "f"(kf[0]), "f"(kf[1]),
                     "f"(kf[2]), "f"(kf[3])
                     : "memory");
        const uint32_t v01 = pack_half2(__uint_as_float(w01 << 16), __uint_as_float(w01 & 0xffff0000u));
        const uint32_t v23 = pack_half2(__uint_as_float(w23 << 16), __uint_as_float(w23 & 0xffff0000u));
        // (a byte above 140: its top bit is set and the others are at least 13)
        high = (((vw & 0x7f7f7f7fu) + 0x73737373u) & vw & (NB == 4 ? 0x80808080u : NB == 2 ? 0x8080u : 0x80u)) != 0u;
        const bool odd = lane & 1;
        // an even lane makes the pairs of blocks 0 and 1, its neighbour of 2 and 3
        const uint32_t mine = odd ? v23 : v01, theirs = __shfl_xor_sync(0xffffffffu, odd ? v01 : v23, 1);
        const uint32_t first = odd ? theirs : mine, second = odd ? mine : theirs;
        asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(scratch + TT * 16 + (lane >> 1) * 16 + (lane & 1) * 8),
                     "r"(__byte_perm(first, second, 0x5410)), "r"(__byte_perm(first, second, 0x7632))
                     : "memory");
        __syncwarp();
      }
      // ---- S^T = K . Q^T, block by block
      float sc[2][NT][4];
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        float4 f[2];  // scales of rows gl and gl + 8
#pragma unroll
        for (int x = 0; x < 2; ++x)
          asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                       : "=f"(f[x].x), "=f"(f[x].y), "=f"(f[x].z), "=f"(f[x].w)
                       : "r"(scratch + (m * 16 + x * 8 + gl) * 16));
        const float f0[4] = {f[0].x, f[0].y, f[0].z, f[0].w}, f1[4] = {f[1].x, f[1].y, f[1].z, f[1].w};
        uint32_t r[2 * NB];  // [block][rows gl / gl + 8]
        if constexpr (NB >= 2) {
#pragma unroll
          for (int jj = 0; jj < NB / 2; ++jj)
            ldsm_x4(kb + m * 16 * TR::ROW + mat[jj], r[4 * jj], r[4 * jj + 1], r[4 * jj + 2], r[4 * jj + 3]);
        } else {
          uint32_t a, b;
          if (m == 0) ldsm_x4(kb + mat[0], r[0], r[1], a, b);
          else ldsm_x4(kb + mat[0], a, b, r[0], r[1]);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) sc[m][nt][0] = sc[m][nt][1] = sc[m][nt][2] = sc[m][nt][3] = 0.f;
        // the first products of all blocks, then the second, so that none waits for
        // its neighbour
        uint32_t a[NB][4], b[NB][4];
        float d[NB][NT][4];
#pragma unroll
        for (int j = 0; j < NB; ++j) {
          fp4_unpack4(r[2 * j], a[j][0], a[j][1], a[j][2], a[j][3]);
          fp4_unpack4(r[2 * j + 1], b[j][0], b[j][1], b[j][2], b[j][3]);
        }
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            mma_16816_zero(d[j][nt], a[j][0], b[j][0], a[j][1], b[j][1], qf[nt][j][0], qf[nt][j][1]);
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            mma_16816(d[j][nt], a[j][2], b[j][2], a[j][3], b[j][3], qf[nt][j][2], qf[nt][j][3]);
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            sc[m][nt][0] += d[j][nt][0] * f0[j];
            sc[m][nt][1] += d[j][nt][1] * f0[j];
            sc[m][nt][2] += d[j][nt][2] * f1[j];
            sc[m][nt][3] += d[j][nt][3] * f1[j];
          }
      }
      if (nv < TT) {
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (m * 16 + gl + (e >> 1) * 8 >= nv) sc[m][nt][e] = -INFINITY;
      }
      if constexpr (TR::WT) {
        if (k < p.track.raw_tiles) {
          float* raw = p.track.raw + (int64_t)k * (HG * G * TT) + hl * G * TT + gl;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const int g = nt * 8 + 2 * tl + j;
              if (g >= G) continue;
#pragma unroll
              for (int m = 0; m < 2; ++m) {
                raw[g * TT + m * 16] = sc[m][nt][j];
                raw[g * TT + m * 16 + 8] = sc[m][nt][j + 2];
              }
            }
          if (hl == 0 && lane == 0) p.track.tiles[k] = make_int4(seg.b, seg.hg, k - seg.start, seg.seq);
        } else if (lane == 0 && p.error_flags != nullptr) {
          atomicOr(p.error_flags, PAD_FLAG_SHARED_PAGE);
        }
      }
      // ---- copy a later tile into the slot of the one before this. Here its
      // instructions fill the gaps between scores and softmax: 26.4 us at 64 x 4096
      // against 28.6 with the copy at the end of a turn, when it was moved.
      copy(next, stage == 0 ? S - 1 : stage - 1);
      place(next);
      // ---- online softmax over the 32 tokens. The reference point m_run need not be
      // the maximum, only near it: it moves when a score passes it by more than
      // kSlack, so p <= 2^kSlack, which fp16's range takes and which cancels in
      // O / l. Nearly every tile then needs no exchange between lanes and no
      // rescaling (64 x 16384: 71.9 -> 68.7 us).
      bool beyond = high;
      float top[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          top[nt][j] = fmaxf(fmaxf(sc[0][nt][j], sc[0][nt][j + 2]), fmaxf(sc[1][nt][j], sc[1][nt][j + 2]));
          beyond |= top[nt][j] > m_run[nt][j] + kSlack;
        }
      if (__any_sync(0xffffffffu, beyond)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float mx = top[nt][j];
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            const float mu = fmaxf(m_run[nt][j], mx), alpha = ex2(m_run[nt][j] - mu);
            m_run[nt][j] = mu;
            l_run[nt][j] *= alpha;
#pragma unroll
            for (int blk = 0; blk < NB; ++blk)
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                acc[blk][x][nt][j] *= alpha;
                acc[blk][x][nt][j + 2] *= alpha;
              }
          }
        // Up to 2^13, the largest the append writes, every code of V is an fp16 value.
        if (high) flag_high_scales<NB>(p, sb + TT * kFp4ScaleRow + lane * kFp4ScaleRow);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float sum = 0.f;
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            sc[m][nt][j] = ex2(sc[m][nt][j] - m_run[nt][j]);
            sc[m][nt][j + 2] = ex2(sc[m][nt][j + 2] - m_run[nt][j]);
            sum += sc[m][nt][j] + sc[m][nt][j + 2];
          }
          l_run[nt][j] += sum;
        }
      // ---- O^T += V^T . (P_hi + P_lo)^T
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const float y0 = sc[m][nt][2 * x], y1 = sc[m][nt][2 * x + 1];
            const __half2 hi = __floats2half2_rn(y0, y1);
            const float2 hf = __half22float2(hi);
            ph[nt][x] = movmatrix_trans(*reinterpret_cast<const uint32_t*>(&hi));
            pl[nt][x] = movmatrix_trans(pack_half2(y0 - hf.x, y1 - hf.y));
          }
        uint4 s[2];  // scale pairs of tokens 2 tl, 2 tl + 1 and of those 8 on, per block
#pragma unroll
        for (int x = 0; x < 2; ++x)
          asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(s[x].x), "=r"(s[x].y), "=r"(s[x].z), "=r"(s[x].w)
                       : "r"(scratch + TT * 16 + (m * 8 + x * 4 + tl) * 16));
        const uint32_t s0[4] = {s[0].x, s[0].y, s[0].z, s[0].w}, s1[4] = {s[1].x, s[1].y, s[1].z, s[1].w};
        uint32_t r[2 * NB];
        if constexpr (NB >= 2) {
#pragma unroll
          for (int jj = 0; jj < NB / 2; ++jj)
            ldsm_x4_trans(vb + m * 16 * TR::ROW + mat[jj], r[4 * jj], r[4 * jj + 1], r[4 * jj + 2], r[4 * jj + 3]);
        } else {
          uint32_t a, b;
          if (m == 0) ldsm_x4_trans(vb + mat[0], r[0], r[1], a, b);
          else ldsm_x4_trans(vb + mat[0], a, b, r[0], r[1]);
        }
#pragma unroll
        for (int j = 0; j < NB; ++j) {
          // A register holds four codes (dims 4 gl ..) of token 2 tl in its low
          // half, of the next token in its high half; r[2j] of the lower, r[2j+1]
          // of the upper 8 tokens. Nibbles are paired across the two tokens before
          // the conversion, so that it yields (token, next token) of one dim:
          // bytes of `even` are dims 0 and 2 of the lower, then of the upper
          // tokens, of `odd` dims 1 and 3.
          const uint32_t own = __byte_perm(r[2 * j], r[2 * j + 1], 0x5410);
          const uint32_t nxt = __byte_perm(r[2 * j], r[2 * j + 1], 0x7632);
          const uint32_t even = (own & 0x0f0f0f0fu) | ((nxt << 4) & 0xf0f0f0f0u);
          const uint32_t odd = ((own >> 4) & 0x0f0f0f0fu) | (nxt & 0xf0f0f0f0u);
          uint32_t e[4], o[4];
          fp4_unpack4(even, e[0], e[1], e[2], e[3]);
          fp4_unpack4(odd, o[0], o[1], o[2], o[3]);
          const __half2 lower = *reinterpret_cast<const __half2*>(&s0[j]), upper = *reinterpret_cast<const __half2*>(&s1[j]);
          auto scaled = [](uint32_t y, __half2 f) {
            const __half2 z = __hmul2(*reinterpret_cast<const __half2*>(&y), f);
            return *reinterpret_cast<const uint32_t*>(&z);
          };
          uint32_t va[2][4];
#pragma unroll
          for (int x = 0; x < 2; ++x) {  // dims 4 gl + 2 x and the next
            va[x][0] = scaled(e[x], lower);
            va[x][1] = scaled(o[x], lower);
            va[x][2] = scaled(e[x + 2], upper);
            va[x][3] = scaled(o[x + 2], upper);
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 2; ++x)
              mma_16816(acc[j][x][nt], va[x][0], va[x][1], va[x][2], va[x][3], ph[nt][0], ph[nt][1]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 2; ++x)
              mma_16816(acc[j][x][nt], va[x][0], va[x][1], va[x][2], va[x][3], pl[nt][0], pl[nt][1]);
        }
      }
      if (++stage == S) stage = 0;
    }

    // ---- end of the segment: join the warps of each head
    const bool split = !(seg.start >= t0 && seg.start + seg.n <= t1);
    const Fp4Cursor done = seg;
    const int pair = seg.b * ngroups + seg.hg, slot = pair + w;
    if (tid == 0 && seg_t == seg.start) {
      if (split || p.meta_by_pair) {
        const int owner = part_owner((int64_t)seg.start + seg.n - 1, total, W);
        p.ws_meta[p.meta_by_pair ? pair : w] =
            split ? make_int4(pair, slot, owner - w + 1, 1) : make_int4(-1, 0, 0, 0);
      }
    }
    const bool more = seg_end < t1;
    if (more) {  // the next segment's queries arrive while this one is joined
      seg_t = seg_end;
      walk.next_pair(seg);
      load_q(seg);
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float l = l_run[nt][j];
        l += __shfl_xor_sync(0xffffffffu, l, 4);
        l += __shfl_xor_sync(0xffffffffu, l, 8);
        l += __shfl_xor_sync(0xffffffffu, l, 16);
        const int g = nt * 8 + 2 * tl + j;
        if (gl == 0) sml[warp * TR::ROWS + g] = make_float2(m_run[nt][j], l);
        if (g < G) {
          float* row = epi + (warp * TR::ROWS + g) * TR::LD + 4 * gl;
#pragma unroll
          for (int blk = 0; blk < NB; ++blk)
            *reinterpret_cast<float4*>(row + blk * 32) =
                make_float4(acc[blk][0][nt][j], acc[blk][0][nt][j + 2], acc[blk][1][nt][j], acc[blk][1][nt][j + 2]);
        }
      }
    // (the warps of a head wait for one another, not for the other heads)
    named_barrier(1 + hl, 32 * WPH);
    for (int x = turn * 32 + lane; x < G * (D / 4); x += 32 * WPH) {
      const int g = x / (D / 4), d = (x % (D / 4)) * 4, row = hl * G + g;
      const float2* ml = sml + hl * WPH * TR::ROWS + g;
      const float* src = epi + (hl * WPH * TR::ROWS + g) * TR::LD + d;
      float Mu = kLeastScore, L = 0.f;
      for (int x2 = 0; x2 < WPH; ++x2) Mu = fmaxf(Mu, ml[x2 * TR::ROWS].x);
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int x2 = 0; x2 < WPH; ++x2) {
        const float2 y = ml[x2 * TR::ROWS];
        const float f = ex2(y.x - Mu);
        const float4 z = *reinterpret_cast<const float4*>(src + x2 * TR::ROWS * TR::LD);
        L += y.y * f;
        o.x += z.x * f;
        o.y += z.y * f;
        o.z += z.z * f;
        o.w += z.w * f;
      }
      if (split) {
        *reinterpret_cast<float4*>(p.ws_o + ((int64_t)slot * HG * G + row) * D + d) = o;
      } else {
        const float inv = L == 0.f ? 0.f : 1.f / L;
        __half2* out = reinterpret_cast<__half2*>(p.out + done.b * p.out_sb +
                                                  (int64_t)(done.hg * HG * G + row) * p.out_sh + d);
        out[0] = __floats2half2_rn(o.x * inv, o.y * inv);
        out[1] = __floats2half2_rn(o.z * inv, o.w * inv);
      }
      if (split && d == 0) p.ws_ml[(int64_t)slot * HG * G + row] = make_float2(Mu, L);
      if constexpr (TR::WT) {
        if (!split && d == 0)
          p.track.norm[(int64_t)pair * HG * G + row] = make_float2(Mu, L == 0.f ? 0.f : 1.f / L);
      }
    }
    if (!more) break;
    named_barrier(1 + hl, 32 * WPH);  // the buffers are read before the next segment writes them
  }
  cp_async_wait_all();
  if (bad_page && p.error_flags != nullptr) atomicOr(p.error_flags, PAD_FLAG_BAD_PAGE_ID);
}

}  // namespace pad
