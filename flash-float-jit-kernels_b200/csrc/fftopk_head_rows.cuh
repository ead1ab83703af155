// Head rows: the kernel that normalises, rotates and quantises heads of q, k and v (fftopk_rows.cu says what it does), for tokens with one
// position and - an instantiation of its own, compiled in fftopk_rows_axes.cu - with one on each of several axes.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/fftopk.h"
#include "fftopk_rows.cuh"

namespace fftopk {

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
  const int32_t* positions;  // NULL: a token's row of the table is its number
  const float* cos_sin;
  int64_t table_rows;
  const int32_t* padding;  // slots of the first part that has some: a token whose entry is negative is padding, and has no position
  int32_t D, R, interleaved;
  float inv_d;
  uint32_t* status;
};
constexpr int kMaxAxes = 4;
struct AxesParams : RowParams {
  int64_t axis_stride;     // from a token's position on one axis to that on the next
  uint32_t axis_of[8];     // two bits a pair
};
template <bool kAxes>
using ParamsOf = typename std::conditional<kAxes, AxesParams, RowParams>::type;

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

// Several axes: rows of cosines and sines for tokens token0 .. token0 + tokens - 1, every pair's from its own axis' row of the table; NaN where there is no such row.
// `thread` of `threads` writes its share.
__device__ __forceinline__ void merge_rows(const AxesParams& p, float* merged, uint32_t token0, uint32_t tokens, uint32_t thread, uint32_t threads) {
  const uint32_t R = (uint32_t)p.R, half = R >> 1, table_rows = (uint32_t)min(p.table_rows, (int64_t)0x80000000ll);
  uint32_t token = token0, pair = thread;
  for (uint32_t i = thread; i < tokens * half; i += threads, pair += threads) {
    while (pair >= half) pair -= half, ++token, merged += R;
    const uint32_t pos = (uint32_t)p.positions[(p.axis_of[pair >> 4] >> (2 * (pair & 15)) & 3u) * p.axis_stride + token];
    float c = __int_as_float(0x7fffffff), s = c;
    if (pos < table_rows) {
      const float* row = p.cos_sin + (uint64_t)pos * R + pair;
      c = row[0], s = row[half];
    } else if (p.status && (p.padding == nullptr || p.padding[token] >= 0)) {
      atomicOr(p.status, (uint32_t)FFTOPK_ST_BAD_INDEX);
    }
    merged[pair] = c, merged[half + pair] = s;
  }
}

// T: the rows' type; kLanes: lanes of a group; kHeads: heads an item takes; kVec: pieces may be read and written as one
template <typename T, int kLanes, int kHeads, bool kVec, int kNorm, int kRot, bool kQuant, bool kAxes>
__device__ __forceinline__ void head_rows(const ParamsOf<kAxes>& p, const int which, float* merged) {
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
    const float* row = nullptr;
    bool ok = true;
    if constexpr (kAxes) {
      const uint32_t item0 = (blockIdx.x - p.first_block[which]) * (uint32_t)(kRowThreads / kLanes);
      const uint32_t token0 = p.per_token[which].div(item0);
      merge_rows(p, merged, token0, p.per_token[which].div(min(item0 + kRowThreads / kLanes, p.items[which]) - 1u) - token0 + 1u, threadIdx.x, kRowThreads);
      __syncthreads();
      row = merged + (in ? token - token0 : 0u) * (uint32_t)p.R;
    } else if (mine) {
      const int64_t pos = p.positions != nullptr ? p.positions[token] : (int64_t)token;
      ok = pos >= 0 && pos < p.table_rows;
      if (!ok && lane == 0 && p.status && (p.padding == nullptr || p.padding[token] >= 0))
        atomicOr(p.status, (uint32_t)FFTOPK_ST_BAD_INDEX);
      row = p.cos_sin + (ok ? pos : 0) * p.R;
    }
    if (mine) {
      const float nan = __int_as_float(0x7fffffff);  // (no such row in the table: the rotated channels become NaN)
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
template <typename T, int kLanes, int kHeads, bool kVec, int kNorm, int kRot, bool kAxes>
__device__ __forceinline__ void head_rows(const ParamsOf<kAxes>& p, int which, float* merged) {
  if (p.part[which].scale != nullptr)
    head_rows<T, kLanes, kHeads, kVec, kNorm, kRot, true, kAxes>(p, which, merged);
  else
    head_rows<T, kLanes, kHeads, kVec, kNorm, kRot, false, kAxes>(p, which, merged);
}
template <typename T, int kLanes, int kHeads, bool kVec, int kNorm, bool kAxes>
__device__ __forceinline__ void head_rows(const ParamsOf<kAxes>& p, int which, float* merged) {
  if (!p.part[which].rotate)
    head_rows<T, kLanes, kHeads, kVec, kNorm, kRotNone, kAxes>(p, which, merged);
  else if (p.interleaved)
    head_rows<T, kLanes, kHeads, kVec, kNorm, kRotNext, kAxes>(p, which, merged);
  else
    head_rows<T, kLanes, kHeads, kVec, kNorm, kRotApart, kAxes>(p, which, merged);
}
template <typename T, int kLanes, int kHeads, bool kVec, bool kAxes>
__global__ void __launch_bounds__(kRowThreads, sizeof(T) == 4 && kHeads > 1 ? 5 : 8) head_rows_kernel(const __grid_constant__ ParamsOf<kAxes> p) {
  float* merged = nullptr;  // several axes: the block's tokens' cosines and sines
  if constexpr (kAxes) {
    __shared__ __align__(16) float rows[kRowThreads * 8];
    merged = rows;
  }
  const int which = blockIdx.x >= p.first_block[2] ? 2 : blockIdx.x >= p.first_block[1] ? 1 : 0;
  const int norm = p.part[which].norm;
  if (norm == FFTOPK_NORM_NONE)
    head_rows<T, kLanes, kHeads, kVec, FFTOPK_NORM_NONE, kAxes>(p, which, merged);
  else if (norm == FFTOPK_NORM_RMS)
    head_rows<T, kLanes, kHeads, kVec, FFTOPK_NORM_RMS, kAxes>(p, which, merged);
  else
    head_rows<T, kLanes, kHeads, kVec, FFTOPK_NORM_LAYER, kAxes>(p, which, merged);
}

template <typename T, int kLanes, bool kAxes>
cudaError_t launch_rows(ParamsOf<kAxes>& p, bool vec, int heads, cudaStream_t stream) {
  const uint32_t per_cta = kRowThreads / kLanes;
  uint32_t grid = 0;
  for (int i = 0; i < kMaxParts; ++i) {
    p.first_block[i] = grid;
    grid += (p.items[i] + per_cta - 1) / per_cta;
  }
  if (!vec)
    head_rows_kernel<T, kLanes, 1, false, kAxes><<<grid, kRowThreads, 0, stream>>>(p);
  else if (kAxes || heads == 1)
    head_rows_kernel<T, kLanes, 1, true, kAxes><<<grid, kRowThreads, 0, stream>>>(p);
  else if constexpr (!kAxes)
    head_rows_kernel<T, kLanes, kHeadsItem, true, kAxes><<<grid, kRowThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

template <typename T, bool kAxes>
cudaError_t launch_rows(ParamsOf<kAxes>& p, bool vec, int heads, cudaStream_t stream) {
  return p.D <= 64 ? launch_rows<T, 8, kAxes>(p, vec, heads, stream)
                   : p.D <= 128 ? launch_rows<T, 16, kAxes>(p, vec, heads, stream) : launch_rows<T, 32, kAxes>(p, vec, heads, stream);
}

template <bool kAxes>
cudaError_t launch_rows(ParamsOf<kAxes>& p, int32_t dtype, bool vec, int heads, cudaStream_t stream) {
  return dtype == FFTOPK_DTYPE_FP32   ? launch_rows<float, kAxes>(p, vec, heads, stream)
         : dtype == FFTOPK_DTYPE_BF16 ? launch_rows<__nv_bfloat16, kAxes>(p, vec, heads, stream)
                                      : launch_rows<__half, kAxes>(p, vec, heads, stream);
}

// fftopk_rows_axes.cu: one head an item; rows of cosines and sines of all tokens
cudaError_t launch_rows_axes(AxesParams& p, int32_t dtype, bool vec, cudaStream_t stream);
cudaError_t launch_merge_rows(const AxesParams& p, float* merged, uint32_t tokens, cudaStream_t stream);

}  // namespace fftopk
