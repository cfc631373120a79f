// The weights of differential attention.
#pragma once

#include <cuda_fp16.h>
#include <math.h>

#include "common.h"

namespace fa {

inline int check_weights(const FaDiffWeights& w, int h, float softmax_scale, const char* who) {
  FA_CHECK_ARG(w.lam != nullptr, std::string(who) + ": lam must be non-NULL");
  FA_CHECK_ARG(w.count == 1 || w.count == h, std::string(who) + ": weights.count must be 1 or h");
  FA_CHECK_ARG(w.is_half == 0 || w.is_half == 1, std::string(who) + ": weights.is_half must be 0 or 1");
  // the row maximum is that of the unscaled scores, and the backward divides by the scale
  FA_CHECK_ARG(softmax_scale >= 1e-6f && softmax_scale < INFINITY, std::string(who) + ": softmax_scale must be at least 1e-6");
  return FA_OK;
}

#ifdef __CUDACC__
__device__ __forceinline__ float weight_of(const FaDiffWeights& w, int head) {
  const int64_t at = w.count == 1 ? 0 : head * w.stride;
  return w.is_half ? __half2float(static_cast<const __half*>(w.lam)[at]) : static_cast<const float*>(w.lam)[at];
}
#endif

}  // namespace fa
