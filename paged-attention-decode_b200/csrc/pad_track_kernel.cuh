// pad_track_kernel.cuh -- the kernel that turns a decode's scores into
// accumulated attention weights (the design is in pad_track.cuh).
#pragma once

#include "pad_b200.h"
#include "pad_ptx.cuh"
#include "pad_track.cuh"

namespace pad {

constexpr int kWeightThreads = 128;
constexpr int kWeightGrid = 148 * 16;  // every SM full; more tiles loop
constexpr int kMaxTrackRows = 128;  // query rows of a head group: 8 heads x 8, 4 x 16

// One tile at a time: fold the (m, l) of its rows (a warp per row, its lanes
// over the slots), then a thread per (head, token) adds up the heads.
__global__ void __launch_bounds__(kWeightThreads) weights_kernel(const __grid_constant__ WeightParams p) {
  __shared__ float sM[kMaxTrackRows], sI[kMaxTrackRows];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rows = p.hg * p.gqa;
  pdl_launch_dependents();
  pdl_wait_primary();
  const int total = min(*p.track.total, p.track.raw_tiles);
  for (int t = blockIdx.x; t < total; t += gridDim.x) {
    const int4 d = p.track.tiles[t];
    const int2 pr = p.track.pairs[d.x * p.ngroups + d.y];
    for (int r = warp; r < rows; r += kWeightThreads / 32) {
      float m = -INFINITY, l = 0.f;
      for (int s = lane; s < pr.y; s += 32) {
        const float2 x = p.ml[(int64_t)(pr.x + s) * rows + r];
        const float mn = fmaxf(m, x.x), mu = mn == -INFINITY ? 0.f : mn;
        l = l * ex2(m - mu) + x.y * ex2(x.x - mu);
        m = mn;
      }
      float M = m;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
      if (M == -INFINITY) M = 0.f;
      l *= ex2(m - M);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
      if (lane == 0) {
        sM[r] = M;
        sI[r] = l == 0.f ? 0.f : 1.f / l;
      }
    }
    __syncthreads();
    const float* raw = p.track.raw + (int64_t)t * rows * p.tt;
    for (int x = tid; x < p.hg * p.tt; x += kWeightThreads) {
      const int hl = x / p.tt, tok = x - hl * p.tt, slot = d.z * p.tt + tok;
      if (slot >= d.w) continue;
      float sum = 0.f;
      for (int g = 0; g < p.gqa; ++g) {
        const int r = hl * p.gqa + g;
        sum += ex2(raw[r * p.tt + tok] - sM[r]) * sI[r];
      }
      const int lp = p.page_shift >= 0 ? slot >> p.page_shift : slot / p.page_size;
      const int64_t row = slot - (int64_t)lp * p.page_size;
      const int page = __ldg(p.block_table + d.x * p.bt_stride + lp);
      if ((unsigned)page >= (unsigned)p.num_pages) continue;  // flagged by the decode kernel
      const int h = d.y * p.hg + hl;
      float* w = p.weights + page * p.w0 + h * p.w1 + row * p.w2;
      const bool fresh = slot >= d.w - p.num_new;
      *w = fresh ? sum : *w + sum;
      if (fresh && p.slot_positions != nullptr)
        p.slot_positions[page * p.p0 + h * p.p1 + row * p.p2] = __ldg(p.total_lens + d.x) - d.w + slot;
    }
    __syncthreads();
  }
}

}  // namespace pad
