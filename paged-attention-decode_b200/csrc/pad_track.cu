// pad_track.cu -- the launch of the attention-weight kernel (pad_track.cuh).
#include <algorithm>

#include "pad_error.cuh"
#include "pad_track.cuh"
#include "pad_track_kernel.cuh"

namespace pad {

int launch_weights(const WeightParams& p, cudaStream_t stream) {
  if (p.track.raw_tiles == 0) return PAD_OK;
  WeightParams prm = p;
  void* args[] = {&prm};
  cudaLaunchConfig_t cfg = {};
  const int64_t elements = (int64_t)p.track.raw_tiles << (p.hg_log2 + p.tt_log2 - 2);
  cfg.gridDim = dim3((unsigned)std::min<int64_t>((elements + kWeightThreads - 1) / kWeightThreads, kWeightGrid));
  cfg.blockDim = dim3(kWeightThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // overlap its launch with the kernel before
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const void* kernel = p.gqa <= 4   ? reinterpret_cast<const void*>(&weights_kernel<4>)
                       : p.gqa <= 8 ? reinterpret_cast<const void*>(&weights_kernel<8>)
                                    : reinterpret_cast<const void*>(&weights_kernel<16>);
  const cudaError_t e = cudaLaunchKernelExC(&cfg, kernel, args);
  return e == cudaSuccess ? PAD_OK : cuda_fail(e, "launching the attention-weight kernel");
}

}  // namespace pad
