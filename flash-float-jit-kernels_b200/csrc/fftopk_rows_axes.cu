// Head rows of tokens with a position on each of several axes: the kernel of fftopk_head_rows.cuh, compiled beside the one of a single
// position (together they take a compiler twice as long).
#include "fftopk_head_rows.cuh"

namespace fftopk {

cudaError_t launch_rows_axes(AxesParams& p, int32_t dtype, bool vec, int heads, cudaStream_t stream) {
  return launch_rows<true>(p, dtype, vec, heads, stream);
}

}  // namespace fftopk
