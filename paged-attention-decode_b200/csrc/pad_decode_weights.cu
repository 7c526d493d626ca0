// pad_decode_weights.cu -- the decode kernel instances that keep their scores
// for the attention weights (pad_track.cuh), in a translation unit of their own
// so that they compile beside the others.
#include "pad_decode_instance.cuh"

namespace pad {

bool pick_decode_weights(int64_t head_dim, int64_t gqa, int hg, bool swz, Instance* out) {
  return pick_decode<true>(head_dim, gqa, hg, swz, out);
}

}  // namespace pad
