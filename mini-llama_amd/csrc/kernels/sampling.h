// Launchers of the sampling operator (C++ linkage, library-private). The C ABI
// in sampling.cpp validates arguments; these configure and launch.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mlq {

struct SampleArgs {
  int rows, vocab;
  const float* logits;
  int64_t stride;
  const float* uniform;
  const float* temperature;  // each of the four may be null
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  int32_t* tokens;
};
size_t sample_workspace(int rows, int vocab);
hipError_t launch_sample(const SampleArgs& a, void* ws, hipStream_t stream);

}  // namespace mlq
