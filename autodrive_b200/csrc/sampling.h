// The sampling kernels (sampling.cu) as the entry point (sampling_ops.cpp) calls them.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace sampling {

// A number for all rows, or one for each.
struct Real {
  double all;
  const float* each;
};
struct Whole {
  int64_t all;
  const void* each;
  int bytes;        // 4 or 8, of each
};

struct Args {
  const void* logits;
  int type;                     // 0 fp32, 1 bf16, 2 fp16
  int64_t rows, v, ld;          // ld: elements between rows
  const void* uniforms;
  int u_double;
  const uint8_t* mask;          // or null
  int64_t mask_row, mask_col;   // its strides
  Real temperature, top_p, min_p;
  Whole top_k;
  int64_t* token;
  float* log_prob;
};

cudaError_t launch(const Args& a, int sms, cudaStream_t st);

}  // namespace sampling
