// pad_decode_instance.cuh -- the instances of the decode kernel and their choice.
#pragma once

#include "pad_decode_kernels.cuh"

namespace pad {

struct Instance {
  const void* kernel;          // decode_stream_kernel<TR>
  int smem_bytes;
  int segw;                    // bytes per row segment (TMA box inner extent)
  bool swz;
  int hg;                      // KV heads per tile
  int tt;                      // tokens per tile
};

template <int D, int NT, int HG, bool SWZ, bool WT>
Instance make_instance() {
  using TR = Traits<D, NT, HG, SWZ, WT>;
  Instance in = {};
  in.kernel = reinterpret_cast<const void*>(&decode_stream_kernel<TR>);
  in.smem_bytes = TR::SMEM_BYTES;
  in.segw = TR::SEGW;
  in.swz = SWZ;
  in.hg = HG;
  in.tt = TR::TT;
  return in;
}

template <int D, int NT, int HG, bool WT>
Instance pick_swz(bool swz) {
  return swz ? make_instance<D, NT, HG, true, WT>() : make_instance<D, NT, HG, false, WT>();
}

template <int D, int NT, bool WT>
Instance pick_hg(int hg, bool swz) {
  switch (hg) {
    case 8:
      if constexpr (NT == 1) return pick_swz<D, NT, 8, WT>(swz);
      else return pick_swz<D, NT, 4, WT>(swz);  // not reached: G > 8 caps the head group at 4
    case 4: return pick_swz<D, NT, 4, WT>(swz);
    case 2: return pick_swz<D, NT, 2, WT>(swz);
    default: return pick_swz<D, NT, 1, WT>(swz);
  }
}

template <bool WT>
bool pick_decode(int64_t head_dim, int64_t gqa, int hg, bool swz, Instance* out) {
  const bool nt1 = gqa <= 8;
  switch (head_dim) {
    case 16: *out = nt1 ? pick_hg<16, 1, WT>(hg, swz) : pick_hg<16, 2, WT>(hg, swz); return true;
    case 32: *out = nt1 ? pick_hg<32, 1, WT>(hg, swz) : pick_hg<32, 2, WT>(hg, swz); return true;
    case 64: *out = nt1 ? pick_hg<64, 1, WT>(hg, swz) : pick_hg<64, 2, WT>(hg, swz); return true;
    case 128: *out = nt1 ? pick_hg<128, 1, WT>(hg, swz) : pick_hg<128, 2, WT>(hg, swz); return true;
    default: return false;
  }
}

// Phase 2 of a decode, launched as a programmatic dependent of phase 1
// (pad_decode.cu): joins the partials of the split pairs.
struct MergeLaunch {
  const float* ws_o;
  const float2* ws_ml;
  const int4* ws_meta;
  __half* out;
  int64_t out_sb, out_sh;
  int ngroups, rows;            // head groups; query rows of one
  int guess_ncap, guess_parts;  // closed-form descriptors (guess_ncap 0: none)
  int64_t batch, partitions, head_dim;
  int meta_by_pair;
  float2* norm;                 // where the rows' (M, 1 / L) go, or null
};
int launch_merge(const MergeLaunch& m, cudaStream_t stream);

// KV heads per tile, and the SM count of a device (pad_decode.cu).
int head_group_for(int64_t hkv, int64_t gqa);
int sm_count(int device, int* num_sms);

// The instances that keep their scores (pad_decode_weights.cu).
bool pick_decode_weights(int64_t head_dim, int64_t gqa, int hg, bool swz, Instance* out);

}  // namespace pad
