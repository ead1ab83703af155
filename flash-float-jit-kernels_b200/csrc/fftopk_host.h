// Host-side helpers shared by the translation units of libfftopk.so.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/fftopk.h"

namespace fftopk {

// cudaError_t of the last failing runtime call on this thread (fftopk_last_cuda_error()).
inline thread_local int g_last_cuda_error = 0;

inline int cuda_fail(cudaError_t e) {
  g_last_cuda_error = (int)e;
  return FFTOPK_ECUDA;
}

// no row of `width` elements lies on another one of its sequence or of its head, as in a broadcast view (the stride of a lone one says nothing)
inline bool rows_apart(int64_t seqs, int64_t seq, int64_t heads, int64_t head, int64_t width) {
  return (seqs <= 1 || seq >= width || -seq >= width) && (heads <= 1 || head >= width || -head >= width);
}

}  // namespace fftopk
