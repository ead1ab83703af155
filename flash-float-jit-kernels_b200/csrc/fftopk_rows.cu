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
#include "fftopk_host.h"
#include "fftopk_internal.h"
#include "fftopk_rows.cuh"

namespace fftopk {
namespace {

constexpr int kRowThreads = 128;
constexpr int kMaxParts = 3;
constexpr int kHeadsItem = 4;  // heads of a token that a group of lanes takes where there are rows enough
constexpr float kAmaxFloor = 1.262177448353618888658765704452e-29f;  // 2^-96

struct RowParams {
  fftopk_head_part part[kMaxParts];
  uint32_t first_block[kMaxParts];  // of a part; the grid is theirs in turn
  FastDiv per_token[kMaxParts];     // items of a token
  uint32_t items[kMaxParts];        // tokens * items of a token
  int32_t aligned_w[kMaxParts];     // weight and bias may be read four at a time
  const int32_t* positions;
  const float* cos_sin;
  int64_t table_rows;
  const int32_t* padding;  // slots of the first part that has some: a token whose entry is negative is padding, and has no position
  int32_t D, R, interleaved;
  float inv_d;
  uint32_t* status;
};

__device__ __forceinline__ void load_weights(float* w, const void* p, int32_t dtype, int at, bool aligned) {
  if (dtype == FFTOPK_DTYPE_FP32) {
    load4(w, static_cast<const float*>(p) + at, aligned);
  } else if (dtype == FFTOPK_DTYPE_BF16) {
    load4(w, static_cast<const __nv_bfloat16*>(p) + at, aligned);
  } else {
    load4(w, static_cast<const __half*>(p) + at, aligned);
  }
}

enum : int { kRotNone = 0, kRotApart = 1, kRotNext = 2 };  // partners: none, i and i + R / 2, 2 i and 2 i + 1

// T: the rows' type; kLanes: lanes of a group; kHeads: heads an item takes; kVec: pieces may be read and written as one
template <typename T, int kLanes, int kHeads, bool kVec, int kNorm, int kRot, bool kQuant>
__device__ __forceinline__ void head_rows(const RowParams& p, const int which) {
  const fftopk_head_part& part = p.part[which];
  const int lane = threadIdx.x & (kLanes - 1);
  const uint32_t mask = group_mask<kLanes>();
  const uint32_t item = (blockIdx.x - p.first_block[which]) * (uint32_t)(kRowThreads / kLanes) + threadIdx.x / kLanes;
  // (groups beyond the last item stay for the shuffles, and touch nothing)
  const bool in = item < p.items[which];
  const uint32_t token = in ? p.per_token[which].div(item) : 0u;
  const int h0 = in ? (int)(item - token * p.per_token[which].d) * kHeads : 0;
  // the lane's pieces: channels at[0] .. at[0] + 3 and at[1] .. at[1] + 3
  const int pairs = kRot == kRotApart ? p.R : 0;  // channels that lie with their partners
  const int back = lane - (pairs >> 3);
  int at[2];
  at[0] = kRot == kRotApart && back < 0 ? 4 * lane : pairs + 4 * back;
  at[1] = at[0] + ((kRot == kRotApart && back < 0 ? pairs : p.D - pairs) >> 1);
  const bool mine = in && lane * 8 < p.D;
  const int there = in ? min(kHeads, part.heads - h0) : 0;  // rows of the item
  const int rows = mine ? there : 0;

  Four<T> raw[kHeads][2];
  {
    const int64_t step = part.x_head_stride;
    const T* x = static_cast<const T*>(part.x) + ((int64_t)token * part.x_token_stride + h0 * step);
#pragma unroll
    for (int i = 0; i < kHeads; ++i, x += step) {
      raw[i][0].zero();
      raw[i][1].zero();
      if (i < rows) {
        raw[i][0].template load<kVec>(x + at[0]);
        raw[i][1].template load<kVec>(x + at[1]);
      }
    }
  }
  // where the rows go
  int64_t to = token;
  bool keep = true;
  if (part.slots != nullptr && in) {
    to = part.slots[token];
    keep = to >= 0 && to < part.n_slots;
    if (to >= part.n_slots && lane == 0 && h0 == 0 && p.status) atomicOr(p.status, (uint32_t)FFTOPK_ST_BAD_INDEX);
  }
  const int puts = keep ? rows : 0;
  // Cosines and sines. Partners apart: of channels at[0] .. at[0] + 3; side by side: of two pairs of each piece, each twice, the sines
  // with the signs the pair's two channels take the other one with.
  Pair c[4], sn[4];
  if constexpr (kRot != kRotNone) {
    const Pair one = pair(1.f, 1.f), none = pair(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < (kRot == kRotApart ? 2 : 4); ++i) c[i] = one, sn[i] = none;
    if (mine) {
      const int64_t pos = p.positions[token];
      const bool ok = pos >= 0 && pos < p.table_rows;
      if (!ok && lane == 0 && p.status && (p.padding == nullptr || p.padding[token] >= 0))
        atomicOr(p.status, (uint32_t)FFTOPK_ST_BAD_INDEX);
      const float nan = __int_as_float(0x7fffffff);  // (no such row in the table: the rotated channels become NaN)
      const float* row = p.cos_sin + (ok ? pos : 0) * p.R;
      const int half = p.R >> 1;
      if constexpr (kRot == kRotNext) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (at[e] < p.R) {
            float2 a = make_float2(nan, nan), b = a;
            if (ok) a = *reinterpret_cast<const float2*>(row + (at[e] >> 1)), b = *reinterpret_cast<const float2*>(row + half + (at[e] >> 1));
            c[2 * e] = pair(a.x, a.x), c[2 * e + 1] = pair(a.y, a.y);
            sn[2 * e] = pair(-b.x, b.x), sn[2 * e + 1] = pair(-b.y, b.y);
          }
        }
      } else if (back < 0) {
        float4 a = make_float4(nan, nan, nan, nan), b = a;
        if (ok) a = *reinterpret_cast<const float4*>(row + at[0]), b = *reinterpret_cast<const float4*>(row + half + at[0]);
        c[0] = pair(a.x, a.y), c[1] = pair(a.z, a.w);
        sn[0] = pair(b.x, b.y), sn[1] = pair(b.z, b.w);
      }
    }
    if constexpr (kRot == kRotApart) {
      const Pair minus = pair(-1.f, -1.f);
      sn[2] = mul2(sn[0], minus), sn[3] = mul2(sn[1], minus);
    }
  }
  Pair w[4], b[4];
  const bool scaled = kNorm != FFTOPK_NORM_NONE && part.weight != nullptr, moved = kNorm != FFTOPK_NORM_NONE && part.bias != nullptr;
  if constexpr (kNorm != FFTOPK_NORM_NONE) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float f[4] = {1.f, 1.f, 1.f, 1.f}, g[4] = {0.f, 0.f, 0.f, 0.f};
      if (scaled && mine) load_weights(f, part.weight, part.weight_dtype, at[e], p.aligned_w[which] != 0);
      if (moved && mine) load_weights(g, part.bias, part.weight_dtype, at[e], p.aligned_w[which] != 0);
      w[2 * e] = pair(f[0], f[1]), w[2 * e + 1] = pair(f[2], f[3]);
      b[2 * e] = pair(g[0], g[1]), b[2 * e + 1] = pair(g[2], g[3]);
    }
  }

  const int64_t step = part.out_head_stride;
  char* o = static_cast<char*>(part.out) + (to * part.out_token_stride + h0 * step) * (kQuant ? 1 : (int)sizeof(T));
  float amax_of[kHeads];
#pragma unroll
  for (int i = 0; i < kHeads; ++i, o += step * (kQuant ? 1 : (int)sizeof(T))) {
    Pair y[4];  // channels of piece 0, of piece 1
    raw[i][0].widen(y);
    raw[i][1].widen(y + 2);
    if constexpr (kNorm != FFTOPK_NORM_NONE) {
      if constexpr (kNorm == FFTOPK_NORM_LAYER) {
        const float2 t = apart(add2(add2(y[0], y[1]), add2(y[2], y[3])));
        const float all = group_sum<kLanes>(t.x + t.y, mask);
        const float mean = mine ? all * p.inv_d : 0.f;  // (lanes beyond D stay zero)
        const Pair less = pair(-mean, -mean);
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = add2(y[e], less);
      }
      const float2 t = apart(add2(fma2(y[0], y[0], mul2(y[1], y[1])), fma2(y[2], y[2], mul2(y[3], y[3]))));
      const float r = rsqrtf(fmaf(group_sum<kLanes>(t.x + t.y, mask), p.inv_d, part.eps));
      const Pair rr = pair(r, r);
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = fma2(mul2(y[e], rr), w[e], b[e]);
    }
    if constexpr (kRot == kRotNext) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (at[e >> 1] < p.R) y[e] = fma2(turned(y[e]), sn[e], mul2(y[e], c[e]));
      }
    } else if constexpr (kRot == kRotApart) {
      if (back < 0) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const Pair u = y[e], v = y[e + 2];
          y[e] = fma2(v, sn[e + 2], mul2(u, c[e]));
          y[e + 2] = fma2(u, sn[e], mul2(v, c[e]));
        }
      }
    }
    if constexpr (!kQuant) {
      if (i < puts) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          Four<T> r;
          r.narrow(y + 2 * e);
          r.template store<kVec>(reinterpret_cast<T*>(o) + at[e]);
        }
      }
    } else {
      float amax = 0.f;  // (NaN is passed over)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = apart(y[e]);
        amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
      }
      amax = group_max<kLanes>(mine ? amax : 0.f, mask);
      if (amax > 3.402823466e38f) {  // an infinity: the largest of the others
        amax = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = apart(y[e]);
          if (fabsf(f.x) <= 3.402823466e38f) amax = fmaxf(amax, fabsf(f.x));
          if (fabsf(f.y) <= 3.402823466e38f) amax = fmaxf(amax, fabsf(f.y));
        }
        amax = group_max<kLanes>(mine ? amax : 0.f, mask);
      }
      amax = fmaxf(amax, kAmaxFloor);
      amax_of[i] = amax;
      const float inv = __fdiv_rn(448.f, amax);
      if (i < puts) {
        const Pair ii = pair(inv, inv);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t codes = to_e4m3(mul2(y[2 * e], ii), mul2(y[2 * e + 1], ii));
          if constexpr (kVec) {
            *reinterpret_cast<uint32_t*>(o + at[e]) = codes;
          } else {
#pragma unroll
            for (int i2 = 0; i2 < 4; ++i2) o[at[e] + i2] = (char)(codes >> (8 * i2));
          }
        }
      }
    }
  }
  if constexpr (kQuant) {  // lane i writes the scale of the item's row i
    float amax = amax_of[0];
#pragma unroll
    for (int i = 1; i < kHeads; ++i)
      if (lane == i) amax = amax_of[i];
    if (keep && lane < there) {  // (whether the lane has channels of its own or not)
      const int h = h0 + lane;
      const float scale = __fdiv_rn(amax, 448.f);
      part.scale[to * part.scale_token_stride + (int64_t)h * part.scale_head_stride] =
          part.mul != nullptr ? part.mul[(int64_t)token * part.heads + h] * scale : scale;
    }
  }
}

// What a part is like is known to the whole block, and is a constant of the code that runs (norm, rotation and quantisation as
// branches inside one body cost 9 % when that was measured). Eight blocks of 128 threads per SM, 64 registers (fp32: five): a block
// loads, works and stores once, so the blocks beside it have to keep memory busy. Those 64 registers are shared by eighteen bodies, and ptxas
// reports 296 bytes of spill stores for 16 lanes (216 with 32, 288 with 8); more registers spill less and hold fewer blocks, which costs
// more. 16,384 tokens of 72 heads, norm and rotation: 126 us; six blocks 145, seven 134, ten (48 registers) 143; two, three or eight
// heads an item 171, 146, 149.
template <typename T, int kLanes, int kHeads, bool kVec, int kNorm, int kRot>
__device__ __forceinline__ void head_rows(const RowParams& p, int which) {
  if (p.part[which].scale != nullptr)
    head_rows<T, kLanes, kHeads, kVec, kNorm, kRot, true>(p, which);
  else
    head_rows<T, kLanes, kHeads, kVec, kNorm, kRot, false>(p, which);
}
template <typename T, int kLanes, int kHeads, bool kVec, int kNorm>
__device__ __forceinline__ void head_rows(const RowParams& p, int which) {
  if (!p.part[which].rotate)
    head_rows<T, kLanes, kHeads, kVec, kNorm, kRotNone>(p, which);
  else if (p.interleaved)
    head_rows<T, kLanes, kHeads, kVec, kNorm, kRotNext>(p, which);
  else
    head_rows<T, kLanes, kHeads, kVec, kNorm, kRotApart>(p, which);
}
template <typename T, int kLanes, int kHeads, bool kVec>
__global__ void __launch_bounds__(kRowThreads, sizeof(T) == 4 && kHeads > 1 ? 5 : 8) head_rows_kernel(const __grid_constant__ RowParams p) {
  const int which = blockIdx.x >= p.first_block[2] ? 2 : blockIdx.x >= p.first_block[1] ? 1 : 0;
  const int norm = p.part[which].norm;
  if (norm == FFTOPK_NORM_NONE)
    head_rows<T, kLanes, kHeads, kVec, FFTOPK_NORM_NONE>(p, which);
  else if (norm == FFTOPK_NORM_RMS)
    head_rows<T, kLanes, kHeads, kVec, FFTOPK_NORM_RMS>(p, which);
  else
    head_rows<T, kLanes, kHeads, kVec, FFTOPK_NORM_LAYER>(p, which);
}

template <typename T, int kLanes>
cudaError_t launch_rows(RowParams& p, bool vec, int heads, cudaStream_t stream) {
  const uint32_t per_cta = kRowThreads / kLanes;
  uint32_t grid = 0;
  for (int i = 0; i < kMaxParts; ++i) {
    p.first_block[i] = grid;
    grid += (p.items[i] + per_cta - 1) / per_cta;
  }
  if (!vec)
    head_rows_kernel<T, kLanes, 1, false><<<grid, kRowThreads, 0, stream>>>(p);
  else if (heads == 1)
    head_rows_kernel<T, kLanes, 1, true><<<grid, kRowThreads, 0, stream>>>(p);
  else
    head_rows_kernel<T, kLanes, kHeadsItem, true><<<grid, kRowThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_rows(RowParams& p, bool vec, int heads, cudaStream_t stream) {
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
  const int heads = vec && all_heads >= (enough + tokens - 1) / tokens ? kHeadsItem : 1;
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
