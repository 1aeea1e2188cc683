// The tcgen05 forward's kSink instantiations (sliding window whose first keys stay visible), in a
// translation unit of their own so that the library's units compile side by side.
#include <cuda.h>
#include <cuda_runtime.h>

#include "sm100_launch.cuh"

namespace mfa {

int launch_sm100_sink(const Sm100Args& args, int dev, bool wide, bool bf16, int gen,
                      bool short_rows, bool one, int64_t grid, cudaStream_t st) {
  return launch_sm100_rt<true>(args, dev, wide, bf16, gen, short_rows, one, grid, st);
}

}  // namespace mfa
