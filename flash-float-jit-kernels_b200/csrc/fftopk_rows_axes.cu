// Head rows of tokens with a position on each of several axes. Few rows: the kernel of fftopk_head_rows.cuh, whose blocks make a row of cosines and sines for each of
// their tokens in shared memory first. Many: those rows are made for all tokens by a kernel in front, and the kernel of a single position reads
// them (16,384 tokens of 72 heads: 124 us so, 126 with a single position, 146 with the rows made by every block, 144 with every lane looking its own
// pairs up; one token in one kernel: 2.9 us).
#include "fftopk_head_rows.cuh"

namespace fftopk {
namespace {

constexpr int kMergeTokens = 4;  // of a block

__global__ void __launch_bounds__(256) merge_rows_kernel(const __grid_constant__ AxesParams p, float* merged, uint32_t tokens) {
  const uint32_t token0 = blockIdx.x * kMergeTokens;
  merge_rows(p, merged + (uint64_t)token0 * (uint32_t)p.R, token0, min((uint32_t)kMergeTokens, tokens - token0), threadIdx.x, 256u);
}

}  // namespace

cudaError_t launch_rows_axes(AxesParams& p, int32_t dtype, bool vec, cudaStream_t stream) { return launch_rows<true>(p, dtype, vec, 1, stream); }

cudaError_t launch_merge_rows(const AxesParams& p, float* merged, uint32_t tokens, cudaStream_t stream) {
  merge_rows_kernel<<<(tokens + kMergeTokens - 1) / kMergeTokens, 256, 0, stream>>>(p, merged, tokens);
  return cudaGetLastError();
}

}  // namespace fftopk
