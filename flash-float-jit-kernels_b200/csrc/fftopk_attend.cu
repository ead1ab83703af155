// Attention over selected tokens: what follows the selector. Every query token t attends to the cache rows its selection names,
//   o[t, h] = sum_j p_j v[row_j, h / g] / sum_j p_j,   p_j = exp(scale * q[t, h] . k[row_j, h / g] - max),   row_j = indices[t, j]
// g query heads to a key head, negative indices left out, a token that names none gets zeros and a log-sum of -inf.
// k and v are of q's type, or e4m3 with a 32-bit scale per row and head. (The reference ends with the indices.)
//
// attend_narrow_kernel, up to 16 query heads to a key head at a time (which calls take it: attend_is_wide in fftopk_decide.h). A row of
// k or v is used by those heads alone, so reading the rows bounds it: 16 flop a byte at most in 16 bits, 32 in fp8, where the tensor
// cores want over 200 (64 tokens, 64 heads on 8 key heads, 2,048 picks: bf16 98 us = 5.5 TB/s; e4m3 82 us, where widening codes and
// pairing rows take half of the ALU). The rows lie anywhere,
// and nothing but their own heads shares them: every warp has a ring of its own in shared memory that cp.async fills, blocks of 16
// (e4m3: 32) keys ahead of the one it works on, and waits for no other warp.
//   q.k: the contraction's order is free, so a lane's 16-byte piece of a key row serves as B fragments of consecutive steps
//        and q is loaded in the same order: no ldmatrix, no padding to its layout.
//   p.v: the contraction runs over keys, so B fragments pair two rows' elements: a lane loads the same 16-byte piece of the
//        four rows its fragments hold and interleaves them (byte permutes); which column a fragment's lane stands for is free too.
// A warp keeps running maxima and sums (one pass); the warps of a CTA are joined in shared memory, the CTAs of a cluster (few
// tokens: a token's keys are split over up to 8 CTAs) through distributed shared memory. No workspace.
//   e4m3 rows are widened to fp16, which holds every code exactly; a row's k scale multiplies its score, its v scale its weight.
//   Queries are brought to magnitudes below 2 by a power of two per head first (fp16 has fewer exponents than bf16; what is
//   lost lies 2^-25 below the head's largest). What a row adds is p * |v scale|, so that is what the running maximum is of:
//   weights p * v scale become fp16 relative to the head's largest of them, off by 2^-11 of their size, the smallest ones by 2^-25
//   of that largest; a large v scale with hardly any weight behind it sets nothing. Sums of p are held against the same reference.
//   16-bit caches: weights are rounded to the cache's type.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include <string.h>

#include <atomic>

#include "../../include/fftopk.h"
#include "fftopk_host.h"
#include "fftopk_internal.h"
#include "fftopk_attend.cuh"
#include "fftopk_decide.h"
#include "fftopk_rows.cuh"
#include "fftopk_tcgen05.cuh"

namespace fftopk {
namespace {

namespace cg = cooperative_groups;

// Four warps, two CTAs per SM: while one CTA starts or joins, the other one streams (64 tokens, 8 key heads, bf16: 98 us; eight warps
// and one CTA per SM: 108). Heads of 64 hold half the accumulators and half the ring: three CTAs per SM, with rings of three stages
// (61 tokens of 3 key heads, fp16: 14.8 us, two CTAs with four stages 18.3; e4m3: 15.0 and 17.4. 512 tokens of 2 key heads, bf16: 82 and
// 102; e4m3: 82 and 92. 64 tokens of 8 key heads, whose 512 CTAs make a second wave of either: 75 and 72; 57 and 56)
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kHeadsM = kAttendHeads;  // query heads a CTA works on: rows of the MMA
constexpr int sm_ctas(int D) { return D == 64 ? 3 : 2; }

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <int kBytes>
__device__ __forceinline__ void copy_or_zero(uint32_t dst, const void* src, bool there) {
  if constexpr (kBytes == 16)
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(there ? 4 : 0) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t addr) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(addr) : "memory");
  return r;
}
__device__ __forceinline__ float2 lds8(uint32_t addr) {
  float2 r;
  asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(r.x), "=f"(r.y) : "r"(addr) : "memory");
  return r;
}
__device__ __forceinline__ float quad_max(float x) {
  x = fmaxf(x, __shfl_xor_sync(kAll, x, 1));
  return fmaxf(x, __shfl_xor_sync(kAll, x, 2));
}
__device__ __forceinline__ float quad_sum(float x) {
  x += __shfl_xor_sync(kAll, x, 1);
  return x + __shfl_xor_sync(kAll, x, 2);
}

// A warp's ring of blocks on their way. Rows are padded so that the lanes that are served together touch all banks: k, where a
// quad reads 64 neighbouring bytes of each of two rows, by 64 bytes beyond a multiple of 128; v, where eight lanes read two
// neighbouring pieces of rows 0, 2, 4, 6, by 16.
template <bool kFp8, int D>
struct Ring {
  static constexpr int kKeys = kFp8 ? 32 : 16;  // keys of a block: 8 KB of k and v at D = 128
  static constexpr int kRowBytes = D * (kFp8 ? 1 : 2);
  static constexpr int kKPitch = kRowBytes == 64 ? 64 : kRowBytes + 64, kVPitch = kRowBytes + 16;
  static constexpr int kV = kKeys * kKPitch, kScales = kV + kKeys * kVPitch;
  static constexpr int kStage = kScales + (kFp8 ? 2 * kKeys * 4 : 0);
  static constexpr int kStages = kFp8 && D != 64 ? 2 : 3;
  static constexpr int kBytes = kStages * kStage;  // of a warp
};
// Shared memory of a CTA: the warps' rings; in their place, in the end, the warps' accumulators, maxima, sums, and joined the CTA's own.
template <int D>
struct JoinSmem {
  float o[kWarps][kHeadsM][D];
  float m[kWarps][kHeadsM], l[kWarps][kHeadsM];
  float joined[kHeadsM][D];
  float2 jml[kHeadsM];  // maximum and sum
};
template <bool kFp8, int D>
constexpr size_t narrow_smem_bytes() {
  return sizeof(JoinSmem<D>) > (size_t)kWarps * Ring<kFp8, D>::kBytes ? sizeof(JoinSmem<D>) : (size_t)kWarps * Ring<kFp8, D>::kBytes;
}

// T: type of q and out, and of the cache where kFp8 is false
template <typename T, bool kFp8, int D>
__global__ void __launch_bounds__(kThreads, sm_ctas(D)) attend_narrow_kernel(const __grid_constant__ AttendParams p) {
  using M = typename std::conditional<kFp8, __half, T>::type;  // the MMAs' type
  constexpr int kCE = kFp8 ? 16 : 8;                            // elements of a 16-byte piece
  constexpr int kPieces = D / (4 * kCE);                        // pieces of a key row per lane (a quad reads a row)
  constexpr int kVWords = D * (kFp8 ? 1 : 2) / 32;              // 32-bit words of a value row per lane (8 lanes read a row)
  using G = Ring<kFp8, D>;
  constexpr int kKeys = G::kKeys;
  constexpr int kStages = G::kStages;
  constexpr int kSub = kKeys / 16;
  constexpr int kTiles = D / 8;                                 // columns tiles of the output
  extern __shared__ __align__(16) unsigned char smem_raw[];
  JoinSmem<D>& sm = *reinterpret_cast<JoinSmem<D>*>(smem_raw);

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, qd = lane & 3;
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  uint32_t unit = blockIdx.x / (uint32_t)ctas;
  const int hb = (int)(unit % (uint32_t)p.head_blocks);
  unit /= (uint32_t)p.head_blocks;
  const int kvh = (int)(unit % (uint32_t)p.kv_heads);
  const int token = (int)(unit / (uint32_t)p.kv_heads);
  const int heads = min(kHeadsM, p.group - hb * kHeadsM);
  const int head0 = kvh * p.group + hb * kHeadsM;

  // q fragments in the order of the key pieces: element pair u of piece i of lane qd
  uint32_t qa[D / 16][4];
  float qmul[2];  // what the rows' scores are to be multiplied with
  {
    const T* q0 = static_cast<const T*>(p.q) + (int64_t)token * p.q_token + (int64_t)head0 * p.q_head;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const bool have = g + 8 * r < heads;
      const T* q = q0 + (int64_t)(g + 8 * r) * p.q_head;
      uint2 w[D / 16];
#pragma unroll
      for (int m = 0; m < D / 16; ++m) {
        const int i = m / (kCE / 4), u = m % (kCE / 4);
        w[m] = have ? *reinterpret_cast<const uint2*>(q + i * 4 * kCE + qd * kCE + 4 * u) : make_uint2(0u, 0u);
      }
      qmul[r] = p.scale_log2;
      if constexpr (kFp8 && !std::is_same<T, __half>::value) {
        float amax = 0.f;
#pragma unroll
        for (int m = 0; m < D / 16; ++m) {
          const float2 a = widen2(w[m].x, T()), b = widen2(w[m].y, T());
          amax = fmaxf(amax, fmaxf(fmaxf(fabsf(a.x), fabsf(a.y)), fmaxf(fabsf(b.x), fabsf(b.y))));
        }
        amax = quad_max(amax);
        const uint32_t e = __float_as_uint(amax) >> 23;  // amax in [2^(e-127), 2^(e-126)); 255: an infinity
        const uint32_t ee = e == 255u ? 127u : max(1u, min(e, 253u));
        const float down = __uint_as_float((254u - ee) << 23), up = __uint_as_float(ee << 23);
        qmul[r] *= up;
#pragma unroll
        for (int m = 0; m < D / 16; ++m) {
          const float2 a = widen2(w[m].x, T()), b = widen2(w[m].y, T());
          w[m] = make_uint2(narrow2(a.x * down, a.y * down, __half()), narrow2(b.x * down, b.y * down, __half()));
        }
      }
#pragma unroll
      for (int m = 0; m < D / 16; ++m) qa[m][r] = w[m].x, qa[m][2 + r] = w[m].y;
    }
  }

  float o[kTiles][4];
#pragma unroll
  for (int i = 0; i < kTiles; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  // what weights are taken against (log2): the largest score; fp8: the largest score + log2 |v scale|, by the scale's exponent
  float mx[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};

  const int32_t* idx = p.indices + (int64_t)token * p.idx_row;
  const int64_t offset = p.offsets != nullptr ? p.offsets[token] : 0;
  constexpr int kLanesRow = G::kRowBytes / 16, kRowsOnce = 32 / kLanesRow, kTurns = kKeys / kRowsOnce;
  const int piece = lane % kLanesRow, sub = lane / kLanesRow;
  const char* const kbase = static_cast<const char*>(p.k) + (int64_t)kvh * p.k_head * (kFp8 ? 1 : 2) + piece * 16;
  const char* const vbase = static_cast<const char*>(p.v) + (int64_t)kvh * p.v_head * (kFp8 ? 1 : 2) + piece * 16;
  const int64_t kstep = p.k_slot * (kFp8 ? 1 : 2), vstep = p.v_slot * (kFp8 ? 1 : 2);
  const uint32_t ring = smem_u32(smem_raw) + (uint32_t)warp * G::kBytes;
  const int blocks = (int)(((uint32_t)p.picks + kKeys - 1u) / kKeys);
  const int stride = ctas * kWarps;

  auto pick = [&](int block) {  // lane's index in a block; -1: none
    const uint32_t j = (uint32_t)block * kKeys + (uint32_t)(lane & (kKeys - 1));
    return block < blocks && j < (uint32_t)p.picks ? idx[j] : -1;
  };
  // asks for a block's rows and scales; which of them are there
  auto ask = [&](uint32_t stage, int32_t index) {
    int64_t slot = index;
    bool ok = slot >= 0;
    if (ok) {
      slot += offset;
      if (slot < 0 || slot >= p.slots) {
        ok = false;
        if (p.status) atomicOr(p.status, (uint32_t)FFTOPK_ST_BAD_INDEX);
      }
    }
    const unsigned live = __ballot_sync(kAll, ok) & (kKeys == 16 ? 0xffffu : kAll);
    if (live != 0u) {
      const int row = ok ? (int)slot : -1;
#pragma unroll
      for (int i = 0; i < kTurns; ++i) {
        const int at = i * kRowsOnce + sub;
        const int r = __shfl_sync(kAll, row, at);
        copy_or_zero<16>(stage + (uint32_t)(at * G::kKPitch + piece * 16), r >= 0 ? kbase + (int64_t)r * kstep : kbase, r >= 0);
        copy_or_zero<16>(stage + (uint32_t)(G::kV + at * G::kVPitch + piece * 16), r >= 0 ? vbase + (int64_t)r * vstep : vbase, r >= 0);
      }
      if constexpr (kFp8) {
        const uint32_t at = stage + (uint32_t)(G::kScales + lane * 8);
        copy_or_zero<4>(at, p.k_scale + (ok ? slot * p.ks_slot + (int64_t)kvh * p.ks_head : 0), ok);
        copy_or_zero<4>(at + 4u, p.v_scale + (ok ? slot * p.vs_slot + (int64_t)kvh * p.vs_head : 0), ok);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    return live;
  };
  int block = rank * kWarps + warp;
  unsigned live_of[kStages];
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) live_of[s] = ask(ring + s * G::kStage, pick(block + s * stride));
  int32_t next = pick(block + (kStages - 1) * stride);
  uint32_t here = ring, there = ring + (kStages - 1) * G::kStage;  // stages: of this block, of the one that is asked for
  for (; block < blocks; block += stride) {
    live_of[kStages - 1] = ask(there, next);
    next = pick(block + kStages * stride);
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
    __syncwarp();
    const unsigned live = live_of[0];
    const uint32_t stage = here;
    here = here + G::kStage == ring + G::kBytes ? ring : here + G::kStage;
    there = there + G::kStage == ring + G::kBytes ? ring : there + G::kStage;
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) live_of[s] = live_of[s + 1];
    if (live == 0u) continue;
    float ks = 0.f, vs = 0.f, vlog = 0.f;  // the scales of the lane's key
    if constexpr (kFp8) {
      const float2 both = lds8(stage + (uint32_t)(G::kScales + lane * 8));
      ks = both.x, vs = both.y;
      vlog = (float)scale_exponent(vs);
    }
    // scores, in units of log2
    float sc[kSub * 2][4];
#pragma unroll
    for (int n = 0; n < kSub * 2; ++n) {
      sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
      const uint32_t at = stage + (uint32_t)((n * 8 + g) * G::kKPitch + qd * 16);
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const uint4 x = lds16(at + 64u * i);
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int u = 0; u < kCE / 4; ++u) {
          const int m = i * (kCE / 4) + u;
          if constexpr (kFp8) {
            mma16816(sc[n], qa[m], e4m3x2_to_half2((uint16_t)w[u]), e4m3x2_to_half2((uint16_t)(w[u] >> 16)), M());
          } else {
            mma16816(sc[n], qa[m], w[2 * u], w[2 * u + 1], M());
          }
        }
      }
    }
    float bmax[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < kSub * 2; ++n) {
      const unsigned mask = live >> (n * 8 + 2 * qd);
      float k0 = 1.f, k1 = 1.f, l0 = 0.f, l1 = 0.f;
      if constexpr (kFp8) {
        k0 = __shfl_sync(kAll, ks, n * 8 + 2 * qd);
        k1 = __shfl_sync(kAll, ks, n * 8 + 2 * qd + 1);
        l0 = __shfl_sync(kAll, vlog, n * 8 + 2 * qd);
        l1 = __shfl_sync(kAll, vlog, n * 8 + 2 * qd + 1);
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        sc[n][2 * r] = (mask & 1u) ? sc[n][2 * r] * k0 * qmul[r] : -INFINITY;
        sc[n][2 * r + 1] = (mask & 2u) ? sc[n][2 * r + 1] * k1 * qmul[r] : -INFINITY;
        bmax[r] = fmaxf(bmax[r], kFp8 ? fmaxf(sc[n][2 * r] + l0, sc[n][2 * r + 1] + l1) : fmaxf(sc[n][2 * r], sc[n][2 * r + 1]));
      }
    }
    // (a reference is let stand until a score exceeds it by 2^8: fp16 weights and 32-bit sums have the room)
    float grow[2], was[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float top = quad_max(bmax[r]);
      const float m = top > mx[r] + 8.f ? top : mx[r];
      grow[r] = mx[r] == m ? 1.f : ex2(mx[r] - m);  // (-inf both: nothing seen yet)
      was[r] = mx[r];
      mx[r] = m;
    }
    if (__any_sync(kAll, grow[0] != 1.f || grow[1] != 1.f)) {
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        o[i][0] *= grow[0], o[i][1] *= grow[0];
        o[i][2] *= grow[1], o[i][3] *= grow[1];
      }
      if constexpr (kFp8) sum[0] = brought(sum[0], was[0], mx[0]), sum[1] = brought(sum[1], was[1], mx[1]);
    }
    if constexpr (!kFp8) sum[0] *= grow[0], sum[1] *= grow[1];
    uint32_t pa[kSub][4];
#pragma unroll
    for (int n = 0; n < kSub * 2; ++n) {
      float v0 = 1.f, v1 = 1.f;
      if constexpr (kFp8) {
        v0 = __shfl_sync(kAll, vs, n * 8 + 2 * qd);
        v1 = __shfl_sync(kAll, vs, n * 8 + 2 * qd + 1);
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float m = mx[r] == -INFINITY ? 0.f : mx[r];
        const float a = ex2(sc[n][2 * r] - m), b = ex2(sc[n][2 * r + 1] - m);
        sum[r] += a + b;
        pa[n >> 1][(n & 1) * 2 + r] = narrow2(a * v0, b * v1, M());
      }
    }
#pragma unroll
    for (int s = 0; s < kSub; ++s) {
      // the lane's pieces of rows 16 s + {2 qd, 2 qd + 1, 2 qd + 8, 2 qd + 9}
      const uint32_t at = stage + (uint32_t)(G::kV + (16 * s + 2 * qd) * G::kVPitch + g * (kVWords >= 4 ? 16 : 8));
#pragma unroll
      for (int h = 0; h < (kVWords >= 4 ? kVWords / 4 : 1); ++h) {
        uint32_t vw[4][4];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const uint32_t from = at + (uint32_t)(((n & 1) + (n >> 1) * 8) * G::kVPitch) + 128u * h;
          if constexpr (kVWords >= 4) {
            const uint4 x = lds16(from);
            vw[n][0] = x.x, vw[n][1] = x.y, vw[n][2] = x.z, vw[n][3] = x.w;
          } else {
            const float2 x = lds8(from);
            vw[n][0] = __float_as_uint(x.x), vw[n][1] = __float_as_uint(x.y);
          }
        }
#pragma unroll
        for (int e = 0; e < (kVWords >= 4 ? 4 : kVWords); ++e) {
          const int w = 4 * h + e;
          const uint32_t a = vw[0][e], b = vw[1][e], c = vw[2][e], d = vw[3][e];
          if constexpr (kFp8) {
            // columns 4 w .. 4 w + 3 of the lane's piece: bytes of rows 2 qd and 2 qd + 1 side by side
            const uint32_t ab0 = __byte_perm(a, b, 0x5140), ab1 = __byte_perm(a, b, 0x7362);
            const uint32_t cd0 = __byte_perm(c, d, 0x5140), cd1 = __byte_perm(c, d, 0x7362);
            mma16816(o[4 * w], pa[s], e4m3x2_to_half2((uint16_t)ab0), e4m3x2_to_half2((uint16_t)cd0), M());
            mma16816(o[4 * w + 1], pa[s], e4m3x2_to_half2((uint16_t)(ab0 >> 16)), e4m3x2_to_half2((uint16_t)(cd0 >> 16)), M());
            mma16816(o[4 * w + 2], pa[s], e4m3x2_to_half2((uint16_t)ab1), e4m3x2_to_half2((uint16_t)cd1), M());
            mma16816(o[4 * w + 3], pa[s], e4m3x2_to_half2((uint16_t)(ab1 >> 16)), e4m3x2_to_half2((uint16_t)(cd1 >> 16)), M());
          } else {
            mma16816(o[2 * w], pa[s], __byte_perm(a, b, 0x5410), __byte_perm(c, d, 0x5410), M());
            mma16816(o[2 * w + 1], pa[s], __byte_perm(a, b, 0x7632), __byte_perm(c, d, 0x7632), M());
          }
        }
      }
    }
    __syncwarp();  // (the next block but kStages - 2 goes where this one was)
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();  // the rings make room for the join

  // ---- join: warps, then CTAs ----
  sum[0] = quad_sum(sum[0]);
  sum[1] = quad_sum(sum[1]);
  if (qd == 0) {
    sm.m[warp][g] = mx[0], sm.m[warp][g + 8] = mx[1];
    sm.l[warp][g] = sum[0], sm.l[warp][g + 8] = sum[1];
  }
#pragma unroll
  for (int t = 0; t < kTiles; ++t) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      // which column tile t of lane n stands for: see the value pieces above
      const int n = 2 * qd + (e & 1);
      const int col = kFp8 ? n * (kVWords * 4) + t : (t >> 3) * 64 + n * 8 + (t & 7);
      sm.o[warp][g + 8 * (e >> 1)][col] = o[t][e];
    }
  }
  __syncthreads();
  for (int i = tid; i < kHeadsM * D; i += kThreads) {
    const int h = i / D, d = i % D;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) m = fmaxf(m, sm.m[w][h]);
    float acc = 0.f, l = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = sm.m[w][h] == m ? 1.f : ex2(sm.m[w][h] - m);  // (a warp without keys: 0 of both; 0 * NaN stays NaN)
      acc += f * sm.o[w][h][d];
      l += kFp8 ? brought(sm.l[w][h], sm.m[w][h], m) : f * sm.l[w][h];
    }
    sm.joined[h][d] = acc;
    if (d == 0) sm.jml[h] = make_float2(m, l);
  }
  if (ctas > 1)
    cluster.sync();
  else
    __syncthreads();
  // every CTA of the cluster finishes its share of the rows, four channels a thread
  for (int i = tid + rank * kThreads; i < heads * (D / 4); i += kThreads * ctas) {
    const int h = i / (D / 4), d = i % (D / 4) * 4;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float m = -INFINITY, l = 0.f;
    if (ctas == 1) {
      o = *reinterpret_cast<const float4*>(&sm.joined[h][d]);
      m = sm.jml[h].x, l = sm.jml[h].y;
    } else {
      // (every CTA's part is asked for before any is used)
      const uint32_t ml_at = smem_u32(&sm.jml[h]), o_at = smem_u32(&sm.joined[h][d]);
      float2 ml[kAttendMaxCluster];
      float4 part[kAttendMaxCluster];
#pragma unroll
      for (int c = 0; c < kAttendMaxCluster; ++c) {
        ml[c] = make_float2(-INFINITY, 0.f);
        if (c < ctas) {
          ml[c] = lds_cluster2(shared_of(ml_at, c));
          part[c] = lds_cluster4(shared_of(o_at, c));
        }
      }
#pragma unroll
      for (int c = 0; c < kAttendMaxCluster; ++c) m = fmaxf(m, ml[c].x);
#pragma unroll
      for (int c = 0; c < kAttendMaxCluster; ++c) {
        if (c < ctas) {
          const float f = ml[c].x == m ? 1.f : ex2(ml[c].x - m);
          o.x += f * part[c].x, o.y += f * part[c].y, o.z += f * part[c].z, o.w += f * part[c].w;
          l += kFp8 ? brought(ml[c].y, ml[c].x, m) : f * ml[c].y;
        }
      }
    }
    const float y[4] = {l == 0.f ? 0.f : o.x / l, l == 0.f ? 0.f : o.y / l, l == 0.f ? 0.f : o.z / l, l == 0.f ? 0.f : o.w / l};
    T* out = static_cast<T*>(p.out) + (int64_t)token * p.out_token + (int64_t)(head0 + h) * p.out_head + d;
    Four<T> r;
    r.narrow(y);
    if (p.out_vec)
      r.template store<true>(out);
    else
      r.template store<false>(out);
    if (d == 0 && p.lse != nullptr)
      p.lse[(int64_t)token * p.kv_heads * p.group + head0 + h] = l == 0.f ? -INFINITY : m * 0.693147180559945309f + logf(l);
  }
  if (ctas > 1) cluster.sync();  // (nobody leaves while its memory is read)
}

std::atomic<int64_t> g_wait_ns{(int64_t)kMbarWaitNs};
std::atomic<uint32_t> g_stop_after{0xffffffffu};

DeviceOnce g_attend_once[kMaxDevices];
struct Limits {
  int sms = 0;
  int narrow_eights[2][2] = {}, wide_eights = 0;  // clusters of eight CTAs the device holds at once; narrow: [e4m3][heads of 128]
};
Limits g_attend_limits[kMaxDevices];

template <typename T, bool kFp8, int D>
int setup_one() {
  const cudaError_t e =
      cudaFuncSetAttribute(attend_narrow_kernel<T, kFp8, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)narrow_smem_bytes<kFp8, D>());
  return e == cudaSuccess ? 0 : cuda_fail(e);
}

template <typename T, bool kFp8, int D>
int eights_of(int& clusters) {
  return clusters_of(clusters, attend_narrow_kernel<T, kFp8, D>, kThreads, narrow_smem_bytes<kFp8, D>());
}

int attend_setup(Limits& limits) {
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e);
  if (dev < 0 || dev >= kMaxDevices) return FFTOPK_EDEVICE;
  const int rc = g_attend_once[dev].run([&] {
    const cudaError_t e2 = cudaDeviceGetAttribute(&g_attend_limits[dev].sms, cudaDevAttrMultiProcessorCount, dev);
    if (e2 != cudaSuccess) return cuda_fail(e2);
    int r = setup_one<__nv_bfloat16, false, 64>();
    if (!r) r = setup_one<__nv_bfloat16, false, 128>();
    if (!r) r = setup_one<__nv_bfloat16, true, 64>();
    if (!r) r = setup_one<__nv_bfloat16, true, 128>();
    if (!r) r = setup_one<__half, false, 64>();
    if (!r) r = setup_one<__half, false, 128>();
    if (!r) r = setup_one<__half, true, 64>();
    if (!r) r = setup_one<__half, true, 128>();
    int(&eights)[2][2] = g_attend_limits[dev].narrow_eights;
    if (!r) r = eights_of<__nv_bfloat16, false, 64>(eights[0][0]);
    if (!r) r = eights_of<__nv_bfloat16, false, 128>(eights[0][1]);
    if (!r) r = eights_of<__nv_bfloat16, true, 64>(eights[1][0]);
    if (!r) r = eights_of<__nv_bfloat16, true, 128>(eights[1][1]);
    if (!r) r = attend_wide_setup(g_attend_limits[dev].wide_eights);
    return r;
  });
  limits = g_attend_limits[dev];
  return rc;
}

template <typename T, bool kFp8, int D>
cudaError_t launch_narrow(const AttendParams& p, int ctas, int64_t units, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(units * ctas), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = narrow_smem_bytes<kFp8, D>();
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)ctas;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, attend_narrow_kernel<T, kFp8, D>, p);
}

template <typename T>
cudaError_t launch_narrow(const AttendParams& p, bool fp8, int D, int ctas, int64_t units, cudaStream_t stream) {
  if (fp8) return D == 64 ? launch_narrow<T, true, 64>(p, ctas, units, stream) : launch_narrow<T, true, 128>(p, ctas, units, stream);
  return D == 64 ? launch_narrow<T, false, 64>(p, ctas, units, stream) : launch_narrow<T, false, 128>(p, ctas, units, stream);
}

// rows of 16-byte pieces whatever their token (slot) and head; the stride of a lone one says nothing
bool on16(const void* p, int64_t n, int64_t a, int64_t heads, int64_t b, int bytes) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (n <= 1 || a * bytes % 16 == 0) && (heads <= 1 || b * bytes % 16 == 0);
}

}  // namespace
}  // namespace fftopk

using namespace fftopk;

extern "C" int fftopk_sparse_attention(const fftopk_attend* a, uint32_t* status, void* cuda_stream) {
  if (a == nullptr) return FFTOPK_EINVAL;
  if (a->tokens < 0 || a->kv_heads < 0 || a->q_heads < 0 || a->picks < 0 || a->slots < 0) return FFTOPK_EINVAL;
  if (a->dtype != FFTOPK_DTYPE_FP16 && a->dtype != FFTOPK_DTYPE_BF16) return FFTOPK_EINVAL;
  if (a->D != 64 && a->D != 128) return FFTOPK_ERANGE;
  if (a->tokens == 0 || a->q_heads == 0) return FFTOPK_OK;
  if (a->kv_heads == 0 || a->q_heads % a->kv_heads != 0) return FFTOPK_EINVAL;
  const bool fp8 = a->k_scale != nullptr;
  if (fp8 != (a->v_scale != nullptr)) return FFTOPK_EINVAL;
  if (!a->q || !a->out) return FFTOPK_EINVAL;
  if (a->picks > 0 && !a->indices) return FFTOPK_EINVAL;
  if (a->picks > 0 && a->slots > 0 && (!a->k || !a->v)) return FFTOPK_EINVAL;
  const int ce = fp8 ? 1 : 2;
  if (!on16(a->q, a->tokens, a->q_token, a->q_heads, a->q_head, 2) || !on16(a->k, a->slots, a->k_slot, a->kv_heads, a->k_head, ce) ||
      !on16(a->v, a->slots, a->v_slot, a->kv_heads, a->v_head, ce))
    return FFTOPK_EINVAL;
  if ((reinterpret_cast<uintptr_t>(a->out) & 1u) || ((reinterpret_cast<uintptr_t>(a->indices) | reinterpret_cast<uintptr_t>(a->offsets) |
                                                      reinterpret_cast<uintptr_t>(a->lse) | reinterpret_cast<uintptr_t>(a->k_scale) |
                                                      reinterpret_cast<uintptr_t>(a->v_scale)) & 3u))
    return FFTOPK_EINVAL;
  if (a->slots > 0x7fffffff || a->tokens > 0x7fffffff) return FFTOPK_ERANGE;
  // (pieces of work: no more than tokens * q_heads, below 2^62, so that nothing has wrapped; what passes is a grid, too)
  if (attend_narrow_units(a->tokens, a->kv_heads, a->q_heads / a->kv_heads) > 0x7fffffff) return FFTOPK_ERANGE;
  Limits limits;
  const int rc = attend_setup(limits);
  if (rc) return rc;
  const int sms = limits.sms;

  AttendParams p;
  memset(&p, 0, sizeof(p));
  p.q = a->q, p.q_token = a->q_token, p.q_head = a->q_head;
  // (an empty cache has no address, and rows that are left out are copies of no bytes: from somewhere)
  p.k = a->slots > 0 ? a->k : a->q, p.v = a->slots > 0 ? a->v : a->q;
  p.k_slot = a->k_slot, p.k_head = a->k_head, p.v_slot = a->v_slot, p.v_head = a->v_head;
  p.k_scale = a->k_scale, p.v_scale = a->v_scale;
  p.ks_slot = a->ks_slot, p.ks_head = a->ks_head, p.vs_slot = a->vs_slot, p.vs_head = a->vs_head;
  p.indices = a->indices, p.idx_row = a->idx_row, p.offsets = a->offsets;
  p.out = a->out, p.out_token = a->out_token, p.out_head = a->out_head, p.lse = a->lse;
  p.slots = a->slots;
  p.tokens = (int32_t)a->tokens, p.kv_heads = a->kv_heads, p.group = a->q_heads / a->kv_heads, p.picks = a->picks;
  const bool wide = attend_is_wide(a->tokens, a->kv_heads, p.group, fp8, sms);
  const int rows = wide ? 128 : kHeadsM;
  p.head_blocks = (p.group + rows - 1) / rows;
  p.scale_log2 = a->softmax_scale * 1.44269504088896340736f;
  p.out_vec = on16(a->out, a->tokens, a->out_token, a->q_heads, a->out_head, 2);
  p.status = status;
  p.wait_ns = (uint64_t)g_wait_ns.load(std::memory_order_relaxed);
  p.stop_after = g_stop_after.load(std::memory_order_relaxed);

  // CTAs a token: as many as keep the device's SMs busy, and no more than give every warp (wide: every CTA) keys
  const int64_t units = a->tokens * p.kv_heads * p.head_blocks;
  const int keys = wide ? 128 : kWarps * (fp8 ? 32 : 16);
  int ctas = 1;
  // (clusters of eight fit in fewer places than their CTAs alone: 16 of the wide kernel's took 26 us, eight 14)
  const int64_t room = wide ? sms : sm_ctas(a->D) * (int64_t)sms, eights = wide ? limits.wide_eights : limits.narrow_eights[fp8][a->D == 128];
  while (ctas < kAttendMaxCluster && units * ctas * 2 <= room && (ctas * 2 < 8 || units <= eights) && (int64_t)ctas * keys < p.picks) ctas *= 2;
  cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  if (wide) {
    const cudaError_t e = attend_wide(p, a->dtype == FFTOPK_DTYPE_BF16, fp8, a->D, ctas, units, sms, stream);
    return e == cudaSuccess ? FFTOPK_OK : cuda_fail(e);
  }
  const cudaError_t e = a->dtype == FFTOPK_DTYPE_BF16 ? launch_narrow<__nv_bfloat16>(p, fp8, a->D, ctas, units, stream)
                                                      : launch_narrow<__half>(p, fp8, a->D, ctas, units, stream);
  return e == cudaSuccess ? FFTOPK_OK : cuda_fail(e);
}

extern "C" int fftopk_set_attend_stop(int64_t wait_ns, int64_t tiles) {
  if (wait_ns > (int64_t)kMbarWaitNs || tiles > 0x7fffffff) return FFTOPK_ERANGE;
  g_wait_ns.store(wait_ns < 0 ? (int64_t)kMbarWaitNs : wait_ns, std::memory_order_relaxed);
  g_stop_after.store(tiles < 0 ? 0xffffffffu : (uint32_t)tiles, std::memory_order_relaxed);
  return FFTOPK_OK;
}
