// Head rows: what lies in front of the indexer and of the attention behind the selector. One pass over the heads of q, k and v
// that normalises each head, rotates it by its token's position, and writes it as it came, quantised, or quantised into a cache
// row; and the way back, rows of a quantised cache gathered and widened.
//
// A head row of D channels x:
//   norm    rms:   y = x * rsqrt(mean(x^2) + eps) * w          layer: y = (x - mean(x)) * rsqrt(var(x) + eps) * w + b
//   rotate  the first R channels in pairs (i, i + R/2), or (2i, 2i + 1), by the angle whose cosine and sine the table holds for
//           the token's position: a' = a c - b s, b' = b c + a s. With several axes (time, height, width) a token has a position on each,
//           and every pair turns by the one of its axis
//   quantise  amax = largest finite |y|, at least 2^-96 (a row of zeros gets a positive scale); codes = e4m3(y * (448 / amax)),
//           to nearest even, infinities to 448, NaN kept; scale = amax / 448
// in 32 bits throughout, rounded once, where it is written. The reference has no counterpart: it starts from finished logits.
//
// What bounds it is memory. A lane has two pieces of four neighbouring channels (8 bytes each of a 16-bit type): where the
// rotation pairs channel i with i + R/2, the piece at i and the piece at its partners, so that it needs no exchange between lanes
// and a piece of the table serves both; elsewhere one piece in each half of what is left. 8 to 32 lanes make a row, its sums are three to
// five shuffles. A group of lanes takes several heads of ONE token where there are rows enough: it loads the token's cosines and
// sines and the norm's weights once, and has that many loads in flight. A block works on one part alone.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

#include "../../include/fftopk.h"
#include "fftopk_head_rows.cuh"
#include "fftopk_host.h"
#include "fftopk_internal.h"
#include "fftopk_rows.cuh"

namespace fftopk {
namespace {

// ---- rows of a quantised cache, gathered and widened -----------------------------------------------
struct ReadParams {
  const uint8_t* cache;
  int64_t slot_stride, head_stride, n_slots;
  const float* scale;
  int64_t scale_slot_stride, scale_head_stride;
  const int32_t* slots;
  const int32_t* offsets;
  void* out;
  FastDiv per_slot, per_row;  // rows (heads) of a slot, slots of a row of `slots`
  int64_t rows;               // N * H
  int32_t D;
  uint32_t* status;
};

__device__ __forceinline__ void store8(float* o, const float (&y)[8]) {
  reinterpret_cast<float4*>(o)[0] = make_float4(y[0], y[1], y[2], y[3]);
  reinterpret_cast<float4*>(o)[1] = make_float4(y[4], y[5], y[6], y[7]);
}
template <typename T>
__device__ __forceinline__ void store8(T* o, const float (&y)[8]) {
  *reinterpret_cast<uint4*>(o) = make_uint4(narrow2(y[0], y[1], T()), narrow2(y[2], y[3], T()), narrow2(y[4], y[5], T()), narrow2(y[6], y[7], T()));
}

// kLanes lanes a row, 8 codes each; kRows rows a group, one behind the other
template <typename T, int kLanes, int kRows, bool kVec>
__global__ void __launch_bounds__(kRowThreads) cache_read_kernel(const __grid_constant__ ReadParams p) {
  const int lane = threadIdx.x & (kLanes - 1);
  constexpr int kGroups = kRowThreads / kLanes;
  const int64_t first = (int64_t)blockIdx.x * (kGroups * kRows) + threadIdx.x / kLanes;
  const int at = lane * 8;
  if (at >= p.D) return;
  uint2 codes[kRows];
  float scale[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int64_t r = first + (int64_t)i * kGroups;
    codes[i] = make_uint2(0u, 0u);
    scale[i] = 0.f;
    if (r < p.rows) {
      const uint32_t n = p.per_slot.div((uint32_t)r);
      const uint32_t h = (uint32_t)r - n * p.per_slot.d;
      int64_t slot = p.slots[n];
      if (slot >= 0) {
        if (p.offsets != nullptr) slot += p.offsets[p.per_row.div(n)];
        if (slot >= 0 && slot < p.n_slots) {
          const uint8_t* x = p.cache + slot * p.slot_stride + (int64_t)h * p.head_stride + at;
          if constexpr (kVec) {
            codes[i] = *reinterpret_cast<const uint2*>(x);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) codes[i].x |= (uint32_t)x[e] << (8 * e), codes[i].y |= (uint32_t)x[4 + e] << (8 * e);
          }
          scale[i] = p.scale[slot * p.scale_slot_stride + (int64_t)h * p.scale_head_stride];
        } else if (lane == 0 && p.status) {
          atomicOr(p.status, (uint32_t)FFTOPK_ST_BAD_INDEX);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int64_t r = first + (int64_t)i * kGroups;
    if (r >= p.rows) break;
    float y[8];
    from_e4m3(y, codes[i].x);
    from_e4m3(y + 4, codes[i].y);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] *= scale[i];
    store8(static_cast<T*>(p.out) + r * p.D + at, y);
  }
}

template <typename T, int kLanes>
cudaError_t launch_read(const ReadParams& p, bool vec, int sms, cudaStream_t stream) {
  constexpr int kRows = 4;
  const int64_t per_cta = kRowThreads / kLanes;
  if (!vec) {
    cache_read_kernel<T, kLanes, 1, false><<<(unsigned)((p.rows + per_cta - 1) / per_cta), kRowThreads, 0, stream>>>(p);
  } else if (p.rows < per_cta * kRows * sms) {  // (2,048 rows: one row a group 2.1 us, four 3.1; 262,144 rows: 27 and 20)
    cache_read_kernel<T, kLanes, 1, true><<<(unsigned)((p.rows + per_cta - 1) / per_cta), kRowThreads, 0, stream>>>(p);
  } else {
    cache_read_kernel<T, kLanes, kRows, true>
        <<<(unsigned)((p.rows + per_cta * kRows - 1) / (per_cta * kRows)), kRowThreads, 0, stream>>>(p);
  }
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_read(const ReadParams& p, bool vec, int sms, cudaStream_t stream) {
  return p.D <= 64 ? launch_read<T, 8>(p, vec, sms, stream) : p.D <= 128 ? launch_read<T, 16>(p, vec, sms, stream) : launch_read<T, 32>(p, vec, sms, stream);
}

DeviceOnce g_sms_once[kMaxDevices];
int g_sms[kMaxDevices];
int device_sms(int& sms) {
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e);
  if (dev < 0 || dev >= kMaxDevices) return FFTOPK_EDEVICE;
  const int rc = g_sms_once[dev].run([&] {
    const cudaError_t e2 = cudaDeviceGetAttribute(&g_sms[dev], cudaDevAttrMultiProcessorCount, dev);
    return e2 == cudaSuccess ? 0 : cuda_fail(e2);
  });
  sms = g_sms[dev];
  return rc;
}

int elem_bytes(int32_t dtype) { return dtype == FFTOPK_DTYPE_FP32 ? 4 : 2; }
bool known_dtype(int32_t dtype) { return dtype == FFTOPK_DTYPE_FP16 || dtype == FFTOPK_DTYPE_BF16 || dtype == FFTOPK_DTYPE_FP32; }
bool on(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(bytes - 1)) == 0; }

// axes: NULL where a token has one position; merged: NULL, or [tokens, rotary] for what kernels of many rows read
int head_rows_call(const fftopk_head_part* parts, int32_t n_parts, int64_t tokens, int32_t D, int32_t dtype, const int32_t* positions,
                   int64_t axis_stride, int32_t n_axes, const uint8_t* axes, float* merged, const float* cos_sin, int64_t table_rows, int32_t rotary,
                   int32_t interleaved, uint32_t* status, void* cuda_stream) {
  if (parts == nullptr || n_parts < 1 || n_parts > kMaxParts || tokens < 0 || !known_dtype(dtype)) return FFTOPK_EINVAL;
  if (D < 8 || D > 256 || (D & 7) != 0) return FFTOPK_ERANGE;
  const int es = elem_bytes(dtype);
  AxesParams p;
  memset(&p, 0, sizeof(p));
  bool vec = true, rotates = false;
  int64_t all_heads = 0;
  for (int i = 0; i < n_parts; ++i) {
    const fftopk_head_part& a = parts[i];
    if (a.heads < 0 || a.norm < FFTOPK_NORM_NONE || a.norm > FFTOPK_NORM_LAYER) return FFTOPK_EINVAL;
    if (a.norm == FFTOPK_NORM_NONE && (a.weight != nullptr || a.bias != nullptr)) return FFTOPK_EINVAL;
    if ((a.weight != nullptr || a.bias != nullptr) && !known_dtype(a.weight_dtype)) return FFTOPK_EINVAL;
    if (a.slots != nullptr && a.n_slots < 0) return FFTOPK_EINVAL;
    if (a.mul != nullptr && a.scale == nullptr) return FFTOPK_EINVAL;
    if (a.heads == 0) continue;
    const bool nowhere = a.slots != nullptr && a.n_slots == 0;  // (an empty cache has no address)
    if (a.x == nullptr || (a.out == nullptr && !nowhere)) {
      if (tokens > 0) return FFTOPK_EINVAL;
      continue;
    }
    const int we = elem_bytes(a.weight_dtype), oe = a.scale != nullptr ? 1 : es;
    if (!on(a.x, es) || !on(a.out, oe) || !on(a.scale, 4) || !on(a.slots, 4) || !on(a.mul, 4) || !on(a.weight, we) || !on(a.bias, we))
      return FFTOPK_EINVAL;
    // pieces of four channels (the stride of a lone token or head says nothing)
    vec = vec && on(a.x, 4 * es) && (tokens == 1 || a.x_token_stride % 4 == 0) && (a.heads == 1 || a.x_head_stride % 4 == 0);
    vec = vec && on(a.out, 4 * oe) && ((tokens == 1 && a.slots == nullptr) || a.out_token_stride % 4 == 0) &&
          (a.heads == 1 || a.out_head_stride % 4 == 0);
    rotates = rotates || a.rotate != 0;
    all_heads += a.heads;
  }
  if (rotates) {
    if (rotary < 16 || rotary > D || (rotary & 15) != 0) return FFTOPK_ERANGE;
    if (tokens > 0 && (positions == nullptr || cos_sin == nullptr || table_rows < 0 || !on(cos_sin, 16) || !on(positions, 4)))
      return FFTOPK_EINVAL;
    for (int i = 0; axes != nullptr && i < rotary / 2; ++i) {
      if (axes[i] >= n_axes) return FFTOPK_EINVAL;
      p.axis_of[i >> 4] |= (uint32_t)axes[i] << (2 * (i & 15));
    }
  }
  if (tokens == 0 || all_heads == 0) return FFTOPK_OK;
  if (tokens > 0x7fffffff) return FFTOPK_ERANGE;  // (in front of every product: none wraps)
  // (one head a group only where there are few rows)
  for (int i = 0; i < n_parts; ++i)
    if (tokens * (((int64_t)parts[i].heads + (vec ? kHeadsItem - 1 : 0)) / (vec ? kHeadsItem : 1)) > (int64_t)0x7fffffff - 64) return FFTOPK_ERANGE;
  // several heads a group once there are rows for every group of lanes the device holds (16,384 tokens of 72 heads: four heads 126 us,
  // one 276; 64 tokens of the indexer's step: 5.2 and 3.5)
  int sms = 0;
  const int rc = device_sms(sms);
  if (rc) return rc;
  const int64_t enough = (int64_t)sms * 64 * kHeadsItem;
  const bool by_axes = axes != nullptr && rotates;
  const int heads = vec && all_heads >= (enough + tokens - 1) / tokens && !(by_axes && merged == nullptr) ? kHeadsItem : 1;
  for (int i = 0; i < n_parts; ++i) {
    p.part[i] = parts[i];
    const int64_t per_token = ((int64_t)parts[i].heads + heads - 1) / heads;
    p.per_token[i] = FastDiv(per_token > 0 ? (uint32_t)per_token : 1u);
    p.items[i] = (uint32_t)(tokens * per_token);
    p.aligned_w[i] = on(parts[i].weight, 16) && on(parts[i].bias, 16);
    if (p.padding == nullptr && parts[i].heads > 0) p.padding = parts[i].slots;
  }
  p.positions = positions;
  p.cos_sin = cos_sin;
  p.table_rows = table_rows;
  p.D = D;
  p.inv_d = 1.f / (float)D;
  p.R = rotary;
  p.interleaved = interleaved;
  p.status = status;
  p.axis_stride = axis_stride;
  cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  cudaError_t e = cudaSuccess;
  if (by_axes && heads == 1) {
    e = launch_rows_axes(p, dtype, vec, stream);
  } else {
    if (by_axes) {
      e = launch_merge_rows(p, merged, (uint32_t)tokens, stream);
      p.positions = nullptr, p.cos_sin = merged, p.table_rows = tokens;
    }
    if (e == cudaSuccess) e = launch_rows<false>(p, dtype, vec, heads, stream);
  }
  return e == cudaSuccess ? FFTOPK_OK : cuda_fail(e);
}

}  // namespace
}  // namespace fftopk

using namespace fftopk;

extern "C" {

int fftopk_head_rows(const fftopk_head_part* parts, int32_t n_parts, int64_t tokens, int32_t D, int32_t dtype,
                     const int32_t* positions, const float* cos_sin, int64_t table_rows, int32_t rotary, int32_t interleaved,
                     uint32_t* status, void* cuda_stream) {
  return head_rows_call(parts, n_parts, tokens, D, dtype, positions, 0, 0, nullptr, nullptr, cos_sin, table_rows, rotary, interleaved, status, cuda_stream);
}

int fftopk_head_rows_axes(const fftopk_head_part* parts, int32_t n_parts, int64_t tokens, int32_t D, int32_t dtype,
                          const int32_t* positions, int64_t axis_stride, int32_t n_axes, const uint8_t* axes, const float* cos_sin,
                          int64_t table_rows, int32_t rotary, int32_t interleaved, float* workspace, uint32_t* status, void* cuda_stream) {
  if (axes == nullptr || n_axes < 1 || !on(workspace, 16)) return FFTOPK_EINVAL;
  if (n_axes > kMaxAxes) return FFTOPK_ERANGE;
  return head_rows_call(parts, n_parts, tokens, D, dtype, positions, axis_stride, n_axes, axes, workspace, cos_sin, table_rows, rotary, interleaved,
                        status, cuda_stream);
}

int fftopk_cache_read(const void* cache, int64_t slot_stride, int64_t head_stride, int64_t n_slots, int32_t heads, int32_t D,
                      const float* scale, int64_t scale_slot_stride, int64_t scale_head_stride, const int32_t* slots, int64_t rows,
                      int64_t per_row, const int32_t* offsets, void* out, int32_t out_dtype, uint32_t* status, void* cuda_stream) {
  if (n_slots < 0 || heads < 0 || rows < 0 || per_row < 0 || !known_dtype(out_dtype)) return FFTOPK_EINVAL;
  if (D < 8 || D > 256 || (D & 7) != 0) return FFTOPK_ERANGE;
  if (rows == 0 || per_row == 0 || heads == 0) return FFTOPK_OK;
  if (slots == nullptr || out == nullptr || (n_slots > 0 && (cache == nullptr || scale == nullptr))) return FFTOPK_EINVAL;
  if (!on(scale, 4) || !on(slots, 4) || !on(offsets, 4) || !on(out, 16)) return FFTOPK_EINVAL;
  if (rows > 0x7fffffff || per_row > 0x7fffffff || rows * per_row > 0x7fffffff || rows * per_row * heads > (int64_t)0x7fffffff - 4096)
    return FFTOPK_ERANGE;
  int sms = 0;
  const int rc = device_sms(sms);
  if (rc) return rc;
  ReadParams p;
  memset(&p, 0, sizeof(p));
  p.cache = static_cast<const uint8_t*>(cache);
  p.slot_stride = slot_stride;
  p.head_stride = head_stride;
  p.n_slots = n_slots;
  p.scale = scale;
  p.scale_slot_stride = scale_slot_stride;
  p.scale_head_stride = scale_head_stride;
  p.slots = slots;
  p.offsets = offsets;
  p.out = out;
  p.per_slot = FastDiv((uint32_t)heads);
  p.per_row = FastDiv((uint32_t)per_row);
  p.rows = rows * per_row * heads;
  p.D = D;
  p.status = status;
  const bool vec = on(cache, 8) && slot_stride % 8 == 0 && (heads == 1 || head_stride % 8 == 0);
  cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  const cudaError_t e = out_dtype == FFTOPK_DTYPE_FP32   ? launch_read<float>(p, vec, sms, stream)
                        : out_dtype == FFTOPK_DTYPE_BF16 ? launch_read<__nv_bfloat16>(p, vec, sms, stream)
                                                         : launch_read<__half>(p, vec, sms, stream);
  return e == cudaSuccess ? FFTOPK_OK : cuda_fail(e);
}

}  // extern "C"
