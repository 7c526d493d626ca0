// pad_track_kernel.cuh -- the kernel that turns a decode's scores into
// accumulated attention weights (the design is in pad_track.cuh).
#pragma once

#include "pad_b200.h"
#include "pad_ptx.cuh"
#include "pad_track.cuh"

namespace pad {

constexpr int kWeightThreads = 256;
constexpr int kWeightGrid = 148 * 8;  // every SM full; more tiles loop

// A thread per (head, token) of a tile. What it needs is three loads deep: the
// scores (their place follows from the tile's number) with the tile's record,
// then the norms with the page id, then the weight itself. Each weight has one
// writer, so results do not depend on any order.
__global__ void __launch_bounds__(kWeightThreads) weights_kernel(const __grid_constant__ WeightParams p) {
  pdl_launch_dependents();
  pdl_wait_primary();
  const int per_log2 = p.hg_log2 + p.tt_log2, tt = 1 << p.tt_log2, G = p.gqa;
  const int64_t total = (int64_t)min(*p.track.total, p.track.raw_tiles) << per_log2;
  for (int64_t e = (int64_t)blockIdx.x * kWeightThreads + threadIdx.x; e < total; e += (int64_t)gridDim.x * kWeightThreads) {
    const int64_t t = e >> per_log2, ht = e >> p.tt_log2;  // tile; (tile, head)
    const int hl = (int)ht & ((1 << p.hg_log2) - 1), tok = (int)e & (tt - 1);
    const float* raw = p.track.raw + ((ht * G) << p.tt_log2) + tok;
    float s[4];
    const int4 d = __ldg(p.track.tiles + t);
#pragma unroll
    for (int g = 0; g < 4; ++g)
      if (g < G) s[g] = __ldg(raw + (g << p.tt_log2));
    const int slot = (d.z << p.tt_log2) + tok;
    if (slot >= d.w) continue;
    const int lp = p.page_shift >= 0 ? slot >> p.page_shift : slot / p.page_size;
    const int page = __ldg(p.block_table + d.x * p.bt_stride + lp);
    const float2* norm = p.track.norm + ((int64_t)(d.x * p.ngroups + d.y) << p.hg_log2) * G + hl * G;
    const int64_t row = slot - (int64_t)lp * p.page_size;
    if ((unsigned)page >= (unsigned)p.num_pages) continue;  // flagged by the decode kernel
    const int h = (d.y << p.hg_log2) + hl;
    float* w = p.weights + page * p.w0 + h * p.w1 + row * p.w2;
    const bool fresh = slot >= d.w - p.num_new;
    const float was = fresh ? 0.f : *w;
    float sum = 0.f;
#pragma unroll
    for (int g = 0; g < 4; ++g)
      if (g < G) {
        const float2 n = __ldg(norm + g);
        sum += ex2(s[g] - n.x) * n.y;
      }
#pragma unroll 4
    for (int g = 4; g < G; ++g) {
      const float2 n = __ldg(norm + g);
      sum += ex2(__ldg(raw + (g << p.tt_log2)) - n.x) * n.y;
    }
    *w = was + sum;
    if (fresh && p.slot_positions != nullptr)
      p.slot_positions[page * p.p0 + h * p.p1 + row * p.p2] = __ldg(p.total_lens + d.x) - d.w + slot;
  }
}

}  // namespace pad
