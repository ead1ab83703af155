// What the two attention kernels over selected rows share.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "fftopk_host.h"

namespace fftopk {

struct AttendParams {
  const void* q;
  int64_t q_token, q_head;  // strides, elements
  const void* k;
  const void* v;
  int64_t k_slot, k_head, v_slot, v_head;
  const float* k_scale;
  const float* v_scale;
  int64_t ks_slot, ks_head, vs_slot, vs_head;
  const int32_t* indices;
  int64_t idx_row;
  const int32_t* offsets;
  void* out;
  int64_t out_token, out_head;
  float* lse;  // [T, q heads]
  int64_t slots;
  int32_t tokens, kv_heads, group, picks;
  int32_t head_blocks;  // blocks of query heads per key head: of 16 (narrow) or 128 (wide)
  float scale_log2;     // softmax scale * log2(e)
  int32_t out_vec;      // rows of out start on 16 bytes
  uint32_t* status;
  uint64_t wait_ns;     // wide: longest wait for the scout
  uint32_t stop_after;  // wide, for tests: tiles after which the scout hands out no more
};

constexpr unsigned kAll = 0xffffffffu;
constexpr int kAttendMaxCluster = 8;  // CTAs that share a token's keys: the portable cluster size

// fftopk_attend_wide.cu; fp8: e4m3 caches; `units` pieces of work (token, key head, 128 query heads), `ctas` CTAs each
int attend_wide_setup(int& eights);  // clusters of eight CTAs the device holds at once
cudaError_t attend_wide(const AttendParams& p, bool bf16, bool fp8, int D, int ctas, int64_t units, int sms, cudaStream_t stream);

#ifdef __CUDACC__
// clusters of kAttendMaxCluster CTAs that the device holds at once
template <typename F>
int clusters_of(int& clusters, F kernel, int threads, size_t smem) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(kAttendMaxCluster, 1, 1);
  cfg.blockDim = dim3((unsigned)threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = kAttendMaxCluster;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg);
  return e == cudaSuccess ? 0 : cuda_fail(e);
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// exponent of a v scale of either sign, within +-100 (sums of weights that are held against it have the room)
__device__ __forceinline__ int scale_exponent(float scale) { return max(-100, min((int)(__float_as_uint(scale) >> 23 & 255u) - 127, 100)); }
// A sum of weights held against 2^from, against 2^to, with v scales in the references: scales of 2^-100 and 2^100 in a list make the
// sum as far from 1 as the factor is, the other way, so it comes in halves.
__device__ __forceinline__ float brought(float sum, float from, float to) {
  if (from == to) return sum;  // (-inf both: nothing seen yet)
  const float half = ex2(0.5f * (from - to));
  return sum * half * half;
}
__device__ __forceinline__ uint4 ldg16(const void* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}
// shared memory of another CTA of the cluster, by its 32-bit address there
__device__ __forceinline__ uint32_t shared_of(uint32_t addr, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float2 lds_cluster2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 lds_cluster4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
#endif  // __CUDACC__

}  // namespace fftopk
