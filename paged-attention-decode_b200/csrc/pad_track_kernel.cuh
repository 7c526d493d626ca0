// pad_track_kernel.cuh -- the kernel that turns a decode's scores into
// accumulated attention weights (the design is in pad_track.cuh).
#pragma once

#include "pad_b200.h"
#include "pad_ptx.cuh"
#include "pad_track.cuh"

namespace pad {

constexpr int kWeightThreads = 256;
constexpr int kWeightGrid = 148 * 8;  // every SM full; more tiles loop

// A thread per head and 4 neighbouring tokens of a tile. What it needs is three
// loads deep: the scores (their place follows from the tile's number) with the
// tile's record, then the norms with the page id, then the weights themselves.
// Each weight has one writer, so results do not depend on any order. GM >= G
// score loads of 16 bytes are in flight together.
template <int GM>
__global__ void __launch_bounds__(kWeightThreads) weights_kernel(const __grid_constant__ WeightParams p) {
  pdl_launch_dependents();
  pdl_wait_primary();
  const int per_log2 = p.hg_log2 + p.tt_log2 - 2, quads_log2 = p.tt_log2 - 2, G = p.gqa;
  const int64_t total = (int64_t)min(*p.track.total, p.track.raw_tiles) << per_log2;
  for (int64_t e = (int64_t)blockIdx.x * kWeightThreads + threadIdx.x; e < total; e += (int64_t)gridDim.x * kWeightThreads) {
    const int64_t t = e >> per_log2, ht = e >> quads_log2;  // tile; (tile, head)
    const int hl = (int)ht & ((1 << p.hg_log2) - 1), tok = ((int)e & ((1 << quads_log2) - 1)) * 4;
    const float* raw = p.track.raw + ((ht * G) << p.tt_log2) + tok;
    const int4 d = __ldg(p.track.tiles + t);
    float4 s[GM];
#pragma unroll
    for (int g = 0; g < GM; ++g)
      if (g < G) s[g] = __ldg(reinterpret_cast<const float4*>(raw + (g << p.tt_log2)));
    const int slot = (d.z << p.tt_log2) + tok, left = d.w - slot;
    // a record is trusted only within the batch and its table (a decode that gave
    // up on a wait leaves records unwritten)
    if (left <= 0 || (unsigned)d.x >= (unsigned)p.batch || (unsigned)d.y >= (unsigned)p.ngroups || slot < 0 || d.w > p.cap)
      continue;
    const int32_t* ids = p.block_table + d.x * p.bt_stride;
    const int lp0 = p.page_shift >= 0 ? slot >> p.page_shift : slot / p.page_size;
    int page[4], row[4];
    page[0] = __ldg(ids + lp0);
    row[0] = slot - lp0 * p.page_size;
#pragma unroll
    for (int j = 1; j < 4; ++j) {
      page[j] = page[0];
      row[j] = row[0] + j;
      if (row[j] >= p.page_size && j < left) {  // (never where 4 divides the page)
        const int lp = (slot + j) / p.page_size;
        page[j] = __ldg(ids + lp);
        row[j] = slot + j - lp * p.page_size;
      }
    }
    const int num_new = p.num_new_of != nullptr ? min(max(__ldg(p.num_new_of + d.x), 0), d.w) : p.num_new;
    const int h = (d.y << p.hg_log2) + hl, fresh = d.w - num_new - slot;  // tokens from `fresh` on are new
    float* w[4];
    float was[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // (a page that is none was flagged by the decode kernel)
      const bool on = j < left && (unsigned)page[j] < (unsigned)p.num_pages;
      w[j] = on ? p.weights + page[j] * p.w0 + h * p.w1 + row[j] * p.w2 : nullptr;
      was[j] = on && j < fresh ? *w[j] : 0.f;
    }
    const float2* norm = p.track.norm + ((int64_t)(d.x * p.ngroups + d.y) << p.hg_log2) * G + hl * G;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int g = 0; g < GM; ++g)
      if (g < G) {
        const float2 n = __ldg(norm + g);
        sum[0] += ex2(s[g].x - n.x) * n.y;
        sum[1] += ex2(s[g].y - n.x) * n.y;
        sum[2] += ex2(s[g].z - n.x) * n.y;
        sum[3] += ex2(s[g].w - n.x) * n.y;
      }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (w[j] == nullptr) continue;
      *w[j] = was[j] + sum[j];
      if (j >= fresh && p.slot_positions != nullptr)
        p.slot_positions[page[j] * p.p0 + h * p.p1 + row[j] * p.p2] = __ldg(p.total_lens + d.x) - d.w + slot + j;
    }
  }
}

}  // namespace pad
