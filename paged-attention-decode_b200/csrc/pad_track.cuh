// pad_track.cuh -- attention weights beside a decode: what the decode kernels
// leave behind for them, and the kernel that adds them up
// (pad_track_kernel.cuh).
//
//   w[page, h, row] (+)= sum over the G query heads g of KV head h of
//                        2^(s_g - M_g) / L_g
//
// with s_g the token's score in log2 units and (M_g, L_g) the softmax maximum
// and sum of the whole row. The decode kernel holds a token's score long before
// (M_g, L_g) are known, so it stores the scores in fp32 (4 G bytes a token and
// KV head beside the 4 D bytes of K and V it reads) and this kernel reads them
// back, usually from L2, when every row's (M, 1 / L) is there. Recomputing them
// would read K again, 2 D bytes. 2^(s - M) / L instead of 2^(s - M - log2 L):
// s - M is exact where it matters, so no rounding of a large exponent enters.
//
// Measured beside the fp16 decode: 64 x 4096 tokens, 12/2 heads, 53.2 us a call
// (45.4 without weights, 41.6 for all bytes at the copy rate); 256 ragged sequences,
// 32/8 heads, 349 us (297.5; 308).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace pad {

// Written by the decode kernel (all in the call's workspace).
struct TrackParams {
  float* raw;     // [raw_tiles][HG * G][TT] scores in log2 units
  int4* tiles;    // [raw_tiles] {sequence, head group, tile of the pair, seq_len}
  float2* norm;   // [batch * head groups][HG * G] {M, 1 / L}: by the decode kernel for
                  // pairs that one CTA finished, by the merge kernel for split ones
  int* total;     // tiles of the batch
  int raw_tiles;  // tiles there is room for: what the pool's pages can hold, each in one sequence
};

struct WeightParams {
  TrackParams track;
  const int32_t *block_table, *total_lens;
  const int32_t* num_new_of;  // new tokens of each sequence, or null: num_new of every one
  float* weights;
  int32_t* slot_positions;
  int64_t w0, w1, w2, p0, p1, p2, bt_stride;
  int batch, cap;  // sequences; slots a table row names
  int hg_log2, gqa, tt_log2, ngroups, page_size, page_shift, num_pages, num_new;
};

// Adds the weights of the decode whose kernels precede it in the stream.
int launch_weights(const WeightParams& p, cudaStream_t stream);

}  // namespace pad
