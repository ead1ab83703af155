// Channels of a head row in a lane's registers, four at a time: loads, stores, conversions and sums over a row's lanes.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>

namespace fftopk {

// n / d for 0 <= n < 2^31 by a multiplication (Granlund and Montgomery, 1994): with s = ceil(log2 d) and
// m = floor(2^32 (2^s - d) / d) + 1, floor(n / d) = (mulhi(n, m) + n) >> s
struct FastDiv {
  uint32_t d = 1, m = 1, s = 0;
  FastDiv() = default;
  __host__ explicit FastDiv(uint32_t div) : d(div) {
    while (((uint64_t)1 << s) < d) ++s;
    m = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << s) - d)) / d + 1);
  }
#ifdef __CUDACC__
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(n, m) + n) >> s; }
#endif
};

#ifdef __CUDACC__

__device__ __forceinline__ float2 widen2(uint32_t v, __nv_bfloat16) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
__device__ __forceinline__ float2 widen2(uint32_t v, __half) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
__device__ __forceinline__ uint32_t narrow2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t narrow2(float a, float b, __half) {
  const __half2 r = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&r);
}

// Two fp32 values in one 64-bit register: sm_100 multiplies and adds them with one instruction
using Pair = unsigned long long;
__device__ __forceinline__ Pair pair(float a, float b) {
  Pair r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 apart(Pair p) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p));
  return r;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ Pair turned(Pair a) {  // the two the other way around
  const float2 f = apart(a);
  return pair(f.y, f.x);
}

// Four neighbouring channels: 8 bytes of a 16-bit type, 16 of fp32
template <typename T>
struct Four {
  uint32_t v[2];
  __device__ __forceinline__ void zero() { v[0] = v[1] = 0u; }
  template <bool kVec>
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (kVec) {
      const uint2 r = *reinterpret_cast<const uint2*>(p);
      v[0] = r.x, v[1] = r.y;
    } else {
      const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
      v[0] = (uint32_t)q[0] | (uint32_t)q[1] << 16, v[1] = (uint32_t)q[2] | (uint32_t)q[3] << 16;
    }
  }
  template <bool kVec>
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (kVec) {
      *reinterpret_cast<uint2*>(p) = make_uint2(v[0], v[1]);
    } else {
      uint16_t* q = reinterpret_cast<uint16_t*>(p);
      q[0] = (uint16_t)v[0], q[1] = (uint16_t)(v[0] >> 16), q[2] = (uint16_t)v[1], q[3] = (uint16_t)(v[1] >> 16);
    }
  }
  __device__ __forceinline__ void widen(float* y) const {
    const float2 a = widen2(v[0], T()), b = widen2(v[1], T());
    y[0] = a.x, y[1] = a.y, y[2] = b.x, y[3] = b.y;
  }
  __device__ __forceinline__ void narrow(const float* y) { v[0] = narrow2(y[0], y[1], T()), v[1] = narrow2(y[2], y[3], T()); }
  __device__ __forceinline__ void widen(Pair* y) const {
    const float2 a = widen2(v[0], T()), b = widen2(v[1], T());
    y[0] = pair(a.x, a.y), y[1] = pair(b.x, b.y);
  }
  __device__ __forceinline__ void narrow(const Pair* y) {
    const float2 a = apart(y[0]), b = apart(y[1]);
    v[0] = narrow2(a.x, a.y, T()), v[1] = narrow2(b.x, b.y, T());
  }
};

template <>
struct Four<float> {
  float v[4];
  __device__ __forceinline__ void zero() { v[0] = v[1] = v[2] = v[3] = 0.f; }
  template <bool kVec>
  __device__ __forceinline__ void load(const float* p) {
    if constexpr (kVec) {
      const float4 a = *reinterpret_cast<const float4*>(p);
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = p[i];
    }
  }
  template <bool kVec>
  __device__ __forceinline__ void store(float* p) const {
    if constexpr (kVec) {
      *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) p[i] = v[i];
    }
  }
  __device__ __forceinline__ void widen(float* y) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = v[i];
  }
  __device__ __forceinline__ void narrow(const float* y) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = y[i];
  }
  __device__ __forceinline__ void widen(Pair* y) const { y[0] = pair(v[0], v[1]), y[1] = pair(v[2], v[3]); }
  __device__ __forceinline__ void narrow(const Pair* y) {
    const float2 a = apart(y[0]), b = apart(y[1]);
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
  }
};

template <typename T>
__device__ __forceinline__ void load4(float* y, const T* p, bool aligned) {
  Four<T> r;
  if (aligned)
    r.template load<true>(p);
  else
    r.template load<false>(p);
  r.widen(y);
}

// The lanes of the calling group, as a mask of its warp: one group of a warp may look for the largest finite value of a row with
// infinities while the others do not, so a group's shuffles name its own lanes alone.
template <int kLanes>
__device__ __forceinline__ uint32_t group_mask() {
  if constexpr (kLanes == 32) return 0xffffffffu;
  return ((1u << (kLanes & 31)) - 1u) << (threadIdx.x & 31u & ~(uint32_t)(kLanes - 1));
}
template <int kLanes>
__device__ __forceinline__ float group_sum(float x, uint32_t mask) {
#pragma unroll
  for (int i = kLanes / 2; i > 0; i >>= 1) x += __shfl_xor_sync(mask, x, i);
  return x;
}
template <int kLanes>
__device__ __forceinline__ float group_max(float x, uint32_t mask) {
#pragma unroll
  for (int i = kLanes / 2; i > 0; i >>= 1) x = fmaxf(x, __shfl_xor_sync(mask, x, i));
  return x;
}

// e4m3 of four, to nearest even; beyond 448 and infinities become 448, NaN stays NaN
__device__ __forceinline__ uint32_t to_e4m3(Pair a, Pair b) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(apart(a), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(apart(b), __NV_SATFINITE, __NV_E4M3);
  return lo | hi << 16;
}
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint16_t v) {
  const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2(v, __NV_E4M3);
  return (uint32_t)r.x | (uint32_t)r.y << 16;
}
__device__ __forceinline__ void from_e4m3(float* y, uint32_t codes) {
  const float2 a = widen2(e4m3x2_to_half2((uint16_t)codes), __half()), b = widen2(e4m3x2_to_half2((uint16_t)(codes >> 16)), __half());
  y[0] = a.x, y[1] = a.y, y[2] = b.x, y[3] = b.y;
}

#endif  // __CUDACC__

}  // namespace fftopk
