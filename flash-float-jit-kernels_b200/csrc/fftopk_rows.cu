// Head rows: what lies in front of the indexer and of the attention behind the selector. One pass over the heads of q, k and v
// that normalises each head, rotates it by its token's position, and writes it as it came, quantised, or quantised into a cache
// row; and the way back, rows of a quantised cache gathered and widened.
//
// A head row of D channels x:
//   norm    rms:   y = x * rsqrt(mean(x^2) + eps) * w          layer: y = (x - mean(x)) * rsqrt(var(x) + eps) * w + b
//   rotate  the first R channels in pairs (i, i + R/2), or (2i, 2i + 1), by the angle whose cosine and sine the table holds for
//           the token's position: a' = a c - b s, b' = b c + a s
//   quantise  amax = largest finite |y|, at least 2^-96 (a row of zeros gets a positive scale); codes = e4m3(y * (448 / amax)),
//           to nearest even, infinities to 448, NaN kept; scale = amax / 448
// in 32 bits throughout, rounded once, where it is written. The reference has no counterpart: it starts from finished logits.
//
// What bounds it is memory: 8 channels a lane, one 16-byte load and store each (16-bit types), 8 to 32 lanes a row, so a row's
// sums are three to five shuffles. A group of lanes takes several heads of ONE token where there are rows enough: it loads the
// token's cosines and sines (64 bytes a lane for 16 bytes of a head) and the norm's weights once, and has that many loads in flight.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

#include "../../include/fftopk.h"
#include "fftopk_host.h"
#include "fftopk_internal.h"
#include "fftopk_rows.cuh"

namespace fftopk {
namespace {

constexpr int kRowThreads = 256;
constexpr int kMaxParts = 3;
constexpr float kAmaxFloor = 1.262177448353618888658765704452e-29f;  // 2^-96

struct RowParams {
  fftopk_head_part part[kMaxParts];
  int32_t first_item[kMaxParts + 1];  // items of a token: a part's first, and their number
  int32_t aligned_w[kMaxParts];       // weight and bias may be read 16 bytes at a time
  FastDiv per_token;
  int64_t items;                      // tokens * items of a token
  const int32_t* positions;
  const float* cos_sin;
  int64_t table_rows;
  int32_t D, R, interleaved;
  uint32_t* status;
};

__device__ __forceinline__ void load_weights(float (&w)[8], const void* p, int32_t dtype, int at, bool aligned) {
  if (dtype == FFTOPK_DTYPE_FP32) {
    load8<float>(w, static_cast<const float*>(p) + at, aligned);
  } else if (dtype == FFTOPK_DTYPE_BF16) {
    load8<__nv_bfloat16>(w, static_cast<const __nv_bfloat16*>(p) + at, aligned);
  } else {
    load8<__half>(w, static_cast<const __half*>(p) + at, aligned);
  }
}

// T: the rows' type; kLanes: lanes of a group (8 channels each); kHeads: heads an item takes; kVec: rows start on 16 bytes
template <typename T, int kLanes, int kHeads, bool kVec>
__global__ void __launch_bounds__(kRowThreads) head_rows_kernel(const __grid_constant__ RowParams p) {
  const int lane = threadIdx.x & (kLanes - 1);
  const int64_t item = (int64_t)blockIdx.x * (kRowThreads / kLanes) + threadIdx.x / kLanes;
  // (groups beyond the last item stay for the shuffles, and touch nothing)
  const bool in = item < p.items;
  const uint32_t it = in ? (uint32_t)item : 0u;
  const uint32_t token = p.per_token.div(it);
  const int of_token = (int)(it - token * p.per_token.d);
  const int which = of_token >= p.first_item[2] ? 2 : of_token >= p.first_item[1] ? 1 : 0;
  const fftopk_head_part& part = p.part[which];
  const int h0 = (of_token - p.first_item[which]) * kHeads;
  const int at = lane * 8;
  const bool mine = in && at < p.D;
  const uint32_t mask = group_mask<kLanes>();

  Row8<T> raw[kHeads];
  const T* x = static_cast<const T*>(part.x) + (int64_t)token * part.x_token_stride + at;
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    raw[i].zero();
    if (mine && h0 + i < part.heads) raw[i].template load<kVec>(x + (int64_t)(h0 + i) * part.x_head_stride);
  }
  // where the row goes
  int64_t to = token;
  bool keep = mine;
  if (part.slots != nullptr && in) {
    to = part.slots[token];
    if (to < 0) keep = false;
    if (to >= part.n_slots) {
      keep = false;
      if (lane == 0 && h0 == 0 && p.status) atomicOr(p.status, (uint32_t)FFTOPK_ST_BAD_INDEX);
    }
  }
  float c[8], s[8];
  const int R = part.rotate ? p.R : 0;
  const bool turned = mine && at < R;
  if (turned) {
    const int64_t pos = p.positions[token];
    const int half = R >> 1;
    const bool ok = pos >= 0 && pos < p.table_rows;
    if (ok) {
      const float* row = p.cos_sin + pos * p.R;
      if (p.interleaved) {
        const float4 cc = *reinterpret_cast<const float4*>(row + (at >> 1)), ss = *reinterpret_cast<const float4*>(row + half + (at >> 1));
        c[0] = cc.x, c[1] = cc.y, c[2] = cc.z, c[3] = cc.w;
        s[0] = ss.x, s[1] = ss.y, s[2] = ss.z, s[3] = ss.w;
      } else {
        const int i = at < half ? at : at - half;
        load8<float>(c, row + i, true);
        load8<float>(s, row + half + i, true);
      }
    } else {
      // no such row in the table: the rotated channels become NaN
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] = s[i] = __int_as_float(0x7fffffff);
      if (lane == 0 && p.status) atomicOr(p.status, (uint32_t)FFTOPK_ST_BAD_INDEX);
    }
  }
  float w[8], b[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = 1.f, b[i] = 0.f;
  if (mine && part.weight != nullptr) load_weights(w, part.weight, part.weight_dtype, at, p.aligned_w[which] != 0);
  if (mine && part.bias != nullptr) load_weights(b, part.bias, part.weight_dtype, at, p.aligned_w[which] != 0);

  const float inv_d = 1.f / (float)p.D;
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    float y[8];
    raw[i].widen(y);
    if (part.norm == FFTOPK_NORM_LAYER) {
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += y[e];
      const float mean = group_sum<kLanes>(sum, mask) * inv_d;
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = mine ? y[e] - mean : 0.f;
    }
    if (part.norm != FFTOPK_NORM_NONE) {
      float sq = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) sq = fmaf(y[e], y[e], sq);
      const float r = rsqrtf(group_sum<kLanes>(sq, mask) * inv_d + part.eps);
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = fmaf(y[e] * r, w[e], b[e]);
    }
    if (R) {  // the same for a whole group: R belongs to the part
      if (p.interleaved) {
        if (turned) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float u = y[2 * e], v = y[2 * e + 1];
            y[2 * e] = u * c[e] - v * s[e];
            y[2 * e + 1] = v * c[e] + u * s[e];
          }
        }
      } else {
        const int step = R >> 4;  // lanes from a channel to its partner's
        const bool low = lane < step;
        const int from = turned ? (low ? lane + step : lane - step) : lane;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float other = __shfl_sync(mask, y[e], from, kLanes);
          if (turned) y[e] = low ? y[e] * c[e] - other * s[e] : y[e] * c[e] + other * s[e];
        }
      }
    }
    const int h = h0 + i;
    const bool put = keep && h < part.heads;
    if (part.scale == nullptr) {
      if (put) {
        T* o = static_cast<T*>(part.out) + to * part.out_token_stride + (int64_t)h * part.out_head_stride + at;
        Row8<T> r;
        r.narrow(y);
        r.template store<kVec>(o);
      }
    } else {
      float amax = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float a = fabsf(y[e]);
        amax = fmaxf(amax, a <= 3.402823466e38f ? a : 0.f);
      }
      if (!mine) amax = 0.f;
      amax = fmaxf(group_max<kLanes>(amax, mask), kAmaxFloor);
      const float inv = __fdiv_rn(448.f, amax);
      if (put) {
        uint8_t* o = static_cast<uint8_t*>(part.out) + to * part.out_token_stride + (int64_t)h * part.out_head_stride + at;
        const uint2 codes = to_e4m3(y, inv);
        if constexpr (kVec) {
          *reinterpret_cast<uint2*>(o) = codes;
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] = (uint8_t)((e < 4 ? codes.x : codes.y) >> (8 * (e & 3)));
        }
        if (lane == 0) {
          const float scale = __fdiv_rn(amax, 448.f);
          part.scale[to * part.scale_token_stride + (int64_t)h * part.scale_head_stride] =
              part.mul != nullptr ? part.mul[(int64_t)token * part.heads + h] * scale : scale;
        }
      }
    }
  }
}

template <typename T, int kLanes>
cudaError_t launch_rows(const RowParams& p, bool vec, int heads, cudaStream_t stream) {
  const int64_t per_cta = kRowThreads / kLanes;
  const unsigned grid = (unsigned)((p.items + per_cta - 1) / per_cta);
  if (!vec)
    head_rows_kernel<T, kLanes, 1, false><<<grid, kRowThreads, 0, stream>>>(p);
  else if (heads == 1)
    head_rows_kernel<T, kLanes, 1, true><<<grid, kRowThreads, 0, stream>>>(p);
  else
    head_rows_kernel<T, kLanes, 4, true><<<grid, kRowThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_rows(const RowParams& p, bool vec, int heads, cudaStream_t stream) {
  return p.D <= 64 ? launch_rows<T, 8>(p, vec, heads, stream)
                   : p.D <= 128 ? launch_rows<T, 16>(p, vec, heads, stream) : launch_rows<T, 32>(p, vec, heads, stream);
}

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
    from_e4m3(y, codes[i]);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] *= scale[i];
    Row8<T> o;
    o.narrow(y);
    o.template store<true>(static_cast<T*>(p.out) + r * p.D + at);
  }
}

template <typename T, int kLanes>
cudaError_t launch_read(const ReadParams& p, bool vec, cudaStream_t stream) {
  constexpr int kRows = 4;
  const int64_t per_cta = kRowThreads / kLanes;
  if (!vec) {
    cache_read_kernel<T, kLanes, 1, false><<<(unsigned)((p.rows + per_cta - 1) / per_cta), kRowThreads, 0, stream>>>(p);
  } else if (p.rows < per_cta * kRows * 148) {
    cache_read_kernel<T, kLanes, 1, true><<<(unsigned)((p.rows + per_cta - 1) / per_cta), kRowThreads, 0, stream>>>(p);
  } else {
    cache_read_kernel<T, kLanes, kRows, true>
        <<<(unsigned)((p.rows + per_cta * kRows - 1) / (per_cta * kRows)), kRowThreads, 0, stream>>>(p);
  }
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_read(const ReadParams& p, bool vec, cudaStream_t stream) {
  return p.D <= 64 ? launch_read<T, 8>(p, vec, stream) : p.D <= 128 ? launch_read<T, 16>(p, vec, stream) : launch_read<T, 32>(p, vec, stream);
}

int elem_bytes(int32_t dtype) { return dtype == FFTOPK_DTYPE_FP32 ? 4 : 2; }
bool known_dtype(int32_t dtype) { return dtype == FFTOPK_DTYPE_FP16 || dtype == FFTOPK_DTYPE_BF16 || dtype == FFTOPK_DTYPE_FP32; }
bool on(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(bytes - 1)) == 0; }

}  // namespace
}  // namespace fftopk

using namespace fftopk;

extern "C" {

int fftopk_head_rows(const fftopk_head_part* parts, int32_t n_parts, int64_t tokens, int32_t D, int32_t dtype,
                     const int32_t* positions, const float* cos_sin, int64_t table_rows, int32_t rotary, int32_t interleaved,
                     uint32_t* status, void* cuda_stream) {
  if (parts == nullptr || n_parts < 1 || n_parts > kMaxParts || tokens < 0 || !known_dtype(dtype)) return FFTOPK_EINVAL;
  if (D < 8 || D > 256 || (D & 7) != 0) return FFTOPK_ERANGE;
  const int es = elem_bytes(dtype);
  RowParams p;
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
    if (a.x == nullptr || a.out == nullptr) {
      if (tokens > 0) return FFTOPK_EINVAL;
      continue;
    }
    const int we = elem_bytes(a.weight_dtype), oe = a.scale != nullptr ? 1 : es;
    if (!on(a.x, es) || !on(a.out, oe) || !on(a.scale, 4) || !on(a.slots, 4) || !on(a.mul, 4) || !on(a.weight, we) || !on(a.bias, we))
      return FFTOPK_EINVAL;
    const int ob = a.scale != nullptr ? 8 : 16;  // bytes a lane stores at once
    // (the stride of a lone token or head says nothing)
    vec = vec && on(a.x, 16) && (tokens == 1 || a.x_token_stride * es % 16 == 0) && (a.heads == 1 || a.x_head_stride * es % 16 == 0);
    vec = vec && on(a.out, ob) && ((tokens == 1 && a.slots == nullptr) || a.out_token_stride * oe % ob == 0) &&
          (a.heads == 1 || a.out_head_stride * oe % ob == 0);
    rotates = rotates || a.rotate != 0;
    all_heads += a.heads;
  }
  if (rotates) {
    if (rotary < 16 || rotary > D || (rotary & 15) != 0) return FFTOPK_ERANGE;
    if (tokens > 0 && (positions == nullptr || cos_sin == nullptr || table_rows < 0 || !on(cos_sin, 16) || !on(positions, 4)))
      return FFTOPK_EINVAL;
  }
  if (tokens == 0 || all_heads == 0) return FFTOPK_OK;
  // Four heads a group once there are rows for every group of the device: see the figures at the top
  const int heads = vec && tokens * all_heads >= 148 * 64 * 4 ? 4 : 1;
  int64_t per_token = 0;
  for (int i = 0; i < n_parts; ++i) {
    p.part[i] = parts[i];
    p.first_item[i] = (int32_t)per_token;
    per_token += (parts[i].heads + heads - 1) / heads;
    p.aligned_w[i] = on(parts[i].weight, 16) && on(parts[i].bias, 16);
  }
  for (int i = n_parts; i <= kMaxParts; ++i) p.first_item[i] = (int32_t)per_token;
  if (per_token > 0x7fffffff || tokens > 0x7fffffff || tokens * per_token > (int64_t)0x7fffffff - 64) return FFTOPK_ERANGE;
  p.per_token = FastDiv((uint32_t)per_token);
  p.items = tokens * per_token;
  p.positions = positions;
  p.cos_sin = cos_sin;
  p.table_rows = table_rows;
  p.D = D;
  p.R = rotary;
  p.interleaved = interleaved;
  p.status = status;
  cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  const cudaError_t e = dtype == FFTOPK_DTYPE_FP32   ? launch_rows<float>(p, vec, heads, stream)
                        : dtype == FFTOPK_DTYPE_BF16 ? launch_rows<__nv_bfloat16>(p, vec, heads, stream)
                                                     : launch_rows<__half>(p, vec, heads, stream);
  return e == cudaSuccess ? FFTOPK_OK : cuda_fail(e);
}

int fftopk_cache_read(const void* cache, int64_t slot_stride, int64_t head_stride, int64_t n_slots, int32_t heads, int32_t D,
                      const float* scale, int64_t scale_slot_stride, int64_t scale_head_stride, const int32_t* slots, int64_t rows,
                      int64_t per_row, const int32_t* offsets, void* out, int32_t out_dtype, uint32_t* status, void* cuda_stream) {
  if (n_slots < 0 || heads < 0 || rows < 0 || per_row < 0 || !known_dtype(out_dtype)) return FFTOPK_EINVAL;
  if (D < 8 || D > 256 || (D & 7) != 0) return FFTOPK_ERANGE;
  if (rows == 0 || per_row == 0 || heads == 0) return FFTOPK_OK;
  if (cache == nullptr || scale == nullptr || slots == nullptr || out == nullptr) return FFTOPK_EINVAL;
  if (!on(scale, 4) || !on(slots, 4) || !on(offsets, 4) || !on(out, 16)) return FFTOPK_EINVAL;
  if (rows > 0x7fffffff || per_row > 0x7fffffff || rows * per_row > 0x7fffffff || rows * per_row * heads > (int64_t)0x7fffffff - 4096)
    return FFTOPK_ERANGE;
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
  const cudaError_t e = out_dtype == FFTOPK_DTYPE_FP32   ? launch_read<float>(p, vec, stream)
                        : out_dtype == FFTOPK_DTYPE_BF16 ? launch_read<__nv_bfloat16>(p, vec, stream)
                                                         : launch_read<__half>(p, vec, stream);
  return e == cudaSuccess ? FFTOPK_OK : cuda_fail(e);
}

}  // extern "C"
