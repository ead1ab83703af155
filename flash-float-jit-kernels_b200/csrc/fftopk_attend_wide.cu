// Attention over selected rows for more than 16 query heads to a key head: the tensor cores' share of fftopk_attend.cu (the
// formulas stand there).
//
// 128 query heads use a row of k and v here, 2 * 2 * 128 flop per element: in 16 bits as many flop per byte as the device has
// (250), in fp8 and wherever tokens share rows out of L2 twice that and more. So the products run on tcgen05, one CTA per SM:
//   S[128 heads x 128 keys] = Q K^T    Q, K in shared memory (K-major, 128-byte swizzle), S in tensor memory
//   O[128 heads x D]       += P V      P in tensor memory (16 bits, over the S it came from), V in shared memory as it lies in the
//                                      cache, [key][channel]: an MN-major operand
// 17 warps: two groups of four softmax warps, one thread per head, that take alternate tiles of keys, each with an S, an O and a
// running maximum of its own, so that one group's exponentials run while the other's products do; eight that gather rows (four
// k, four v), and one thread that issues the MMAs: QK of tile j + 1, then PV of tile j. The rows lie anywhere: 16-bit ones are
// copied with cp.async, e4m3 ones go through registers and are widened to fp16 on the way (eight 16-byte loads a thread in
// flight: as a piece is widened the next tile's takes its registers). Rows that are not there are zeros, and masked in S.
//
// A row's maximum is let stand until a score exceeds it by 2^8 (fp16 and 32-bit sums have the room), so O, which lives in tensor
// memory, is hardly ever rescaled. fp8: the k scales multiply S, the v scales P, relative to a power of two near the largest v scale that is
// let stand likewise: it is part of the reference the exponentials are taken against. At the end the groups' O are added, row by
// row, with the factors their maxima give.
// A CTA takes one piece of work after the other (token, key head, 128 query heads), and its gathering warps run ahead into the next
// one. Few tokens: the CTAs of a cluster take every n-th tile, and join through distributed shared memory.
// Every wait on an mbarrier has a time limit; when one runs out the CTA raises FFTOPK_ST_STAGE_TIMEOUT and winds down.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/fftopk.h"
#include "fftopk_attend.cuh"
#include "fftopk_host.h"
#include "fftopk_internal.h"
#include "fftopk_rows.cuh"
#include "fftopk_tcgen05.cuh"

namespace fftopk {
namespace {

namespace cg = cooperative_groups;

constexpr int kHeadsW = 128;   // rows of the MMAs
constexpr int kTileKeys = 128; // keys of a tile
constexpr int kSoftmaxWarps = 8, kGatherWarps = 8;
constexpr int kMmaWarp = kSoftmaxWarps + kGatherWarps;
constexpr int kWideThreads = (kMmaWarp + 1) * 32;
constexpr uint32_t kTmemCols = 512;
constexpr float kLetStand = 8.f;  // log2 by which a score may exceed the reference

template <int D>
struct WideCfg {
  static constexpr uint32_t kTileBytes = kTileKeys * D * 2;  // of Q too
  static constexpr int kKStages = D == 128 ? 3 : 4, kVStages = D == 128 ? 2 : 4;
  // Softmax reads a tile's TileMeta after its K stage may have been filled again. The gather of tile n + kKStages + 2 waits for
  // QK of tile n + 2, which is issued behind PV of tile n, which waits for softmax of tile n: so many places are enough.
  static constexpr int kMeta = kKStages + 2;
};
struct TileMeta {  // of a tile's keys
  float ks[kTileKeys], vs[kTileKeys];
  uint32_t live[4];
  float vmax[4];
};
template <int D>
struct WideSmem {  // behind the operand tiles
  TileMeta meta[WideCfg<D>::kMeta];
  float qmul[2][kHeadsW];    // by parity of the piece of work
  float2 ml[2][2][kHeadsW];  // by parity of the piece of work, and group: maximum and sum
  uint64_t kfull[WideCfg<D>::kKStages], kempty[WideCfg<D>::kKStages];
  uint64_t vfull[WideCfg<D>::kVStages], vempty[WideCfg<D>::kVStages];
  uint64_t mfull[WideCfg<D>::kMeta];
  uint64_t qfull, qempty, oempty, mlbar;
  uint64_t sfull[2], pfull[2], pvdone[2];
  uint32_t tmem, abort_flag;
};
template <int D>
constexpr size_t wide_smem_bytes() {
  return 1024 + (size_t)WideCfg<D>::kTileBytes * (1 + WideCfg<D>::kKStages + WideCfg<D>::kVStages) + sizeof(WideSmem<D>);
}

// V as it lies in the cache: an MN-major operand, 128-byte swizzle. Blocks of 64 channels x 128 keys, 128 bytes a key; 8 keys are
// 1024 bytes apart (stride offset), blocks of channels 16 KiB (leading offset).
__device__ __forceinline__ uint64_t desc_mn_sw128(uint32_t smem_addr) {
  return umma_desc_sw128(smem_addr) & ~((uint64_t)0x3fffu << 16) | (uint64_t)((kTileKeys * 128u) >> 4) << 16;
}
template <typename M, int N, bool kMnMajorB>
__host__ __device__ constexpr uint32_t instr_desc() {  // D fp32; A and B fp16 or bf16; M = 128
  constexpr uint32_t f = std::is_same<M, __half>::value ? 0u : 1u;
  return (1u << 4) | (f << 7) | (f << 10) | ((kMnMajorB ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(kHeadsW >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
      "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
      "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]),
      "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {  // zeros where it is not
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void put16(uint32_t dst, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// 16-byte chunk c of row r of a tile: blocks of 64 channels, 128 bytes a row, swizzled
__device__ __forceinline__ uint32_t chunk_at(uint32_t tile, int r, int c) {
  return tile + (uint32_t)(c >> 3) * (kTileKeys * 128u) + (uint32_t)r * 128u + (uint32_t)(((c & 7) ^ (r & 7)) << 4);
}

// tiles of a token's picks up to the last entry that is not negative (by a whole warp)
__device__ __forceinline__ int tiles_of(const int32_t* idx, int picks, int lane) {
  for (int hi = picks; hi > 0; hi -= 512) {
    int last = -1;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int j = hi - 1 - (i * 32 + lane);
      if (j >= 0 && idx[j] >= 0) last = max(last, j);
    }
    last = __reduce_max_sync(kAll, last);
    if (last >= 0) return last / kTileKeys + 1;
  }
  return 0;
}

struct Work {
  int token, kvh, head0, heads;
};
__device__ __forceinline__ Work work_of(const AttendParams& p, uint32_t unit) {
  Work w;
  const int hb = (int)(unit % (uint32_t)p.head_blocks);
  unit /= (uint32_t)p.head_blocks;
  w.kvh = (int)(unit % (uint32_t)p.kv_heads);
  w.token = (int)(unit / (uint32_t)p.kv_heads);
  w.heads = min(kHeadsW, p.group - hb * kHeadsW);
  w.head0 = w.kvh * p.group + hb * kHeadsW;
  return w;
}

// 32 consecutive scores of a thread's row out of tensor memory: times the k scales (fp8), masked
template <bool kFp8>
__device__ __forceinline__ void load_scores(float (&s)[32], uint32_t taddr, const float* ks, uint32_t live) {
  uint32_t v[32];
  tmem_ld32(taddr, v);
  tmem_wait_ld();
#pragma unroll
  for (int i = 0; i < 32; ++i) s[i] = __uint_as_float(v[i]);
  if constexpr (kFp8) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float4 k = reinterpret_cast<const float4*>(ks)[i];
      s[4 * i] *= k.x, s[4 * i + 1] *= k.y, s[4 * i + 2] *= k.z, s[4 * i + 3] *= k.w;
    }
  }
  if (live != kAll) {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (!(live >> i & 1u)) s[i] = -INFINITY;
  }
}

template <typename T, int N>
__device__ __forceinline__ void store_row(T* out, const float (&y)[N], bool vec) {
  if (vec) {
#pragma unroll
    for (int i = 0; i < N; i += 8)
      *reinterpret_cast<uint4*>(out + i) = make_uint4(narrow2(y[i], y[i + 1], T()), narrow2(y[i + 2], y[i + 3], T()),
                                                      narrow2(y[i + 4], y[i + 5], T()), narrow2(y[i + 6], y[i + 7], T()));
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const uint32_t v = narrow2(y[i], y[i + 1], T());
      reinterpret_cast<uint16_t*>(out)[i] = (uint16_t)v;
      reinterpret_cast<uint16_t*>(out)[i + 1] = (uint16_t)(v >> 16);
    }
  }
}

template <typename T, bool kFp8, int D>
__global__ void __launch_bounds__(kWideThreads, 1) attend_wide_kernel(const __grid_constant__ AttendParams p, const uint32_t units) {
  using M = typename std::conditional<kFp8, __half, T>::type;
  using C = WideCfg<D>;
  constexpr uint32_t kTileBytes = C::kTileBytes;
  constexpr int kKS = C::kKStages, kVS = C::kVStages;
  extern __shared__ unsigned char wide_raw[];
  const uint32_t pad = (1024u - (smem_u32(wide_raw) & 1023u)) & 1023u;
  unsigned char* base = wide_raw + pad;
  const uint32_t q_tile = smem_u32(base), k_tiles = q_tile + kTileBytes, v_tiles = k_tiles + kKS * kTileBytes;
  WideSmem<D>& sm = *reinterpret_cast<WideSmem<D>*>(base + (size_t)kTileBytes * (1 + kKS + kVS));
  volatile uint32_t* abort_flag = &sm.abort_flag;

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const uint32_t first = blockIdx.x / (uint32_t)ctas, step = gridDim.x / (uint32_t)ctas;

  if (tid == 0) {
    for (int i = 0; i < kKS; ++i) mbar_init(&sm.kfull[i], 4), mbar_init(&sm.kempty[i], 1);
    for (int i = 0; i < kVS; ++i) mbar_init(&sm.vfull[i], 4), mbar_init(&sm.vempty[i], 1);
    for (int i = 0; i < C::kMeta; ++i) mbar_init(&sm.mfull[i], 4);
    mbar_init(&sm.qfull, 4);
    mbar_init(&sm.qempty, 1);
    mbar_init(&sm.oempty, kSoftmaxWarps);
    mbar_init(&sm.mlbar, kSoftmaxWarps);
    for (int i = 0; i < 2; ++i) mbar_init(&sm.sfull[i], 1), mbar_init(&sm.pfull[i], 4), mbar_init(&sm.pvdone[i], 1);
    sm.abort_flag = 0u;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem)), "r"(kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  const uint32_t tmem = sm.tmem;

  // Tiles this CTA has been through (it), pieces of work with tiles (wn): they select stages and the barriers' phases.
  uint32_t it = 0, wn = 0;
  bool ok = true;

  if (warp >= kSoftmaxWarps && warp < kMmaWarp) {
    // ---- gather ----
    const bool is_k = warp < kSoftmaxWarps + 4;
    const int gw = (warp - kSoftmaxWarps) & 3;  // rows 32 gw .. 32 gw + 31 of a tile
    uint64_t* const full = is_k ? sm.kfull : sm.vfull;
    uint64_t* const empty = is_k ? sm.kempty : sm.vempty;
    const int stages = is_k ? kKS : kVS;
    const uint32_t tiles = is_k ? k_tiles : v_tiles;
    constexpr int kLanesRow = D * (kFp8 ? 1 : 2) / 16;  // lanes that read a row
    constexpr int kRowsOnce = 32 / kLanesRow, kTurns = 32 / kRowsOnce;
    const int piece = lane % kLanesRow;
    const int64_t row_bytes = (is_k ? p.k_slot : p.v_slot) * (kFp8 ? 1 : 2);
    for (uint32_t unit = first; ok && unit < units; unit += step) {
      const Work w = work_of(p, unit);
      const int32_t* idx = p.indices + (int64_t)w.token * p.idx_row;
      const int all = tiles_of(idx, p.picks, lane);
      const int nt = all > rank ? (all - rank + ctas - 1) / ctas : 0;
      if (nt == 0) continue;
      const int64_t offset = p.offsets != nullptr ? p.offsets[w.token] : 0;
      const char* const src = static_cast<const char*>(is_k ? p.k : p.v) + (int64_t)w.kvh * (is_k ? p.k_head : p.v_head) * (kFp8 ? 1 : 2) + piece * 16;
      auto pick = [&](int j) {  // the lane's row of local tile j
        const int at = (rank + j * ctas) * kTileKeys + gw * 32 + lane;
        return j < nt && at < p.picks ? idx[at] : -1;
      };
      auto row_of = [&](int32_t i) {
        if (i < 0) return -1;
        const int64_t slot = i + offset;
        if (slot < 0 || slot >= p.slots) {
          if (is_k && p.status) atomicOr(p.status, (uint32_t)FFTOPK_ST_BAD_INDEX);
          return -1;
        }
        return (int)slot;
      };
      int row = row_of(pick(0));
      int32_t ahead = pick(1);  // (an index is asked for a tile before its row is)
      uint4 held[kFp8 ? kTurns : 1];  // fp8: the lane's pieces of the rows on their way
      float ks = 0.f, vs = 0.f;
      auto fetch = [&](int i, int r) {
        const int of = __shfl_sync(kAll, r, i * kRowsOnce + lane / kLanesRow);
        held[i] = of >= 0 ? ldg16(src + (int64_t)of * row_bytes) : make_uint4(0u, 0u, 0u, 0u);
      };
      auto fetch_scales = [&](int r) {
        ks = vs = 0.f;
        if (is_k && r >= 0) {
          ks = __ldg(p.k_scale + (int64_t)r * p.ks_slot + (int64_t)w.kvh * p.ks_head);
          vs = __ldg(p.v_scale + (int64_t)r * p.vs_slot + (int64_t)w.kvh * p.vs_head);
        }
      };
      if constexpr (kFp8) {
#pragma unroll
        for (int i = 0; i < kTurns; ++i) fetch(i, row);
        fetch_scales(row);
      }
      if (is_k) {
        // q: rows 32 gw .. of the tile
        if (!__all_sync(kAll, mbar_wait(&sm.qempty, (wn & 1u) ^ 1u, abort_flag))) {
          ok = false;
          break;
        }
        constexpr int kQLanes = D / 8, kQOnce = 32 / kQLanes;
        const int c = lane % kQLanes;
        const float negative = p.scale_log2 < 0.f ? -1.f : 1.f;
        const uint32_t flip = p.scale_log2 < 0.f ? 0x80008000u : 0u;
        const T* q0 = static_cast<const T*>(p.q) + (int64_t)w.token * p.q_token + (int64_t)w.head0 * p.q_head + c * 8;
#pragma unroll 4
        for (int i = 0; i < 32 / kQOnce; ++i) {
          const int h = gw * 32 + i * kQOnce + lane / kQLanes;
          uint4 v = h < w.heads ? *reinterpret_cast<const uint4*>(q0 + (int64_t)h * p.q_head) : make_uint4(0u, 0u, 0u, 0u);
          float mul = p.scale_log2 * negative;
          if constexpr (kFp8 && !std::is_same<T, __half>::value) {
            // to magnitudes below 2, as fp16 (see fftopk_attend.cu)
            const float2 a = widen2(v.x, T()), b = widen2(v.y, T()), d = widen2(v.z, T()), e = widen2(v.w, T());
            float amax = fmaxf(fmaxf(fmaxf(fabsf(a.x), fabsf(a.y)), fmaxf(fabsf(b.x), fabsf(b.y))),
                               fmaxf(fmaxf(fabsf(d.x), fabsf(d.y)), fmaxf(fabsf(e.x), fabsf(e.y))));
#pragma unroll
            for (int o = kQLanes / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(kAll, amax, o));
            const uint32_t ex = __float_as_uint(amax) >> 23;
            const uint32_t ee = ex == 255u ? 127u : max(1u, min(ex, 253u));
            const float down = __uint_as_float((254u - ee) << 23);
            mul *= __uint_as_float(ee << 23);
            v = make_uint4(narrow2(a.x * down, a.y * down, __half()), narrow2(b.x * down, b.y * down, __half()),
                           narrow2(d.x * down, d.y * down, __half()), narrow2(e.x * down, e.y * down, __half()));
          }
          put16(chunk_at(q_tile, h, c), v.x ^ flip, v.y ^ flip, v.z ^ flip, v.w ^ flip);
          if (c == 0) sm.qmul[wn & 1u][h] = fmaxf(mul, 1.17549435e-38f);  // (times a masked score it must stay -inf)
        }
        fence_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.qfull);
      }
      for (int j = 0; j < nt; ++j) {
        const uint32_t n = it + (uint32_t)j;
        const int stage = (int)(n % (uint32_t)stages);
        const uint32_t phase = (n / (uint32_t)stages) & 1u;
        const uint32_t tile = tiles + (uint32_t)stage * kTileBytes;
        const int next_row = row_of(ahead);
        ahead = pick(j + 2);
        if (!__all_sync(kAll, mbar_wait(&empty[stage], phase ^ 1u, abort_flag))) {
          ok = false;
          break;
        }
        if (is_k) {
          const int place = (int)(n % (uint32_t)C::kMeta);
          TileMeta& m = sm.meta[place];
          const unsigned live = __ballot_sync(kAll, row >= 0);
          if (lane == 0) m.live[gw] = live;
          if constexpr (kFp8) {
            m.ks[gw * 32 + lane] = ks;
            m.vs[gw * 32 + lane] = vs;
            float top = vs;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kAll, top, o));
            if (lane == 0) m.vmax[gw] = top;
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.mfull[place]);
        }
        if constexpr (kFp8) {
#pragma unroll
          for (int i = 0; i < kTurns; ++i) {
            const int r = gw * 32 + i * kRowsOnce + lane / kLanesRow;
            const uint32_t x[4] = {held[i].x, held[i].y, held[i].z, held[i].w};
            uint32_t h[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              h[2 * e] = e4m3x2_to_half2((uint16_t)x[e]);
              h[2 * e + 1] = e4m3x2_to_half2((uint16_t)(x[e] >> 16));
            }
            // (lanes of a row's second half write their chunks the other way around: eight lanes, all banks)
            const bool swap = (piece & 4) != 0;
            const uint32_t lo = chunk_at(tile, r, 2 * piece), hi = chunk_at(tile, r, 2 * piece + 1);
            put16(swap ? hi : lo, swap ? h[4] : h[0], swap ? h[5] : h[1], swap ? h[6] : h[2], swap ? h[7] : h[3]);
            put16(swap ? lo : hi, swap ? h[0] : h[4], swap ? h[1] : h[5], swap ? h[2] : h[6], swap ? h[3] : h[7]);
            fetch(i, next_row);  // the next tile's piece takes its place
          }
          fetch_scales(next_row);
          fence_async_shared();
          __syncwarp();
          if (lane == 0) mbar_arrive(&full[stage]);
        } else {
#pragma unroll
          for (int i = 0; i < kTurns; ++i) {
            const int r = i * kRowsOnce + lane / kLanesRow;
            const int of = __shfl_sync(kAll, row, r);
            copy16(chunk_at(tile, gw * 32 + r, piece), of >= 0 ? src + (int64_t)of * row_bytes : src, of >= 0);
          }
          asm volatile("cp.async.commit_group;" ::: "memory");
          // the tile before this one has landed: hand it over (the last one: below)
          if (j > 0) {
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            fence_async_shared();
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[(n - 1) % (uint32_t)stages]);
          }
        }
        row = next_row;
      }
      if constexpr (!kFp8) {
        if (ok) {
          asm volatile("cp.async.wait_group 0;" ::: "memory");
          fence_async_shared();
          __syncwarp();
          if (lane == 0) mbar_arrive(&full[(it + (uint32_t)nt - 1) % (uint32_t)stages]);
        }
      }
      it += (uint32_t)nt;
      ++wn;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp == kMmaWarp) {
    // ---- the MMAs ----
    uint32_t turns[2] = {0u, 0u};  // tiles of each group in the pieces of work before
    for (uint32_t unit = first; unit < units; unit += step) {
      const Work w = work_of(p, unit);
      const int all = tiles_of(p.indices + (int64_t)w.token * p.idx_row, p.picks, lane);
      const int nt = all > rank ? (all - rank + ctas - 1) / ctas : 0;
      if (nt == 0) continue;
      if (lane == 0) {
        ok = mbar_wait(&sm.qfull, wn & 1u, abort_flag);
        for (int j = 0; ok && j <= nt; ++j) {
          if (j < nt) {  // S of tile j
            const uint32_t n = it + (uint32_t)j;
            const int stage = (int)(n % kKS);
            if (!(ok = mbar_wait(&sm.kfull[stage], (n / kKS) & 1u, abort_flag))) break;
            tmem_fence_after();
            const uint32_t kt = k_tiles + (uint32_t)stage * kTileBytes;
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
              const uint32_t at = (uint32_t)(k >> 2) * (kTileKeys * 128u) + (uint32_t)(k & 3) * 32u;
              mma_ss(tmem + (uint32_t)(j & 1) * 128u, umma_desc_sw128(q_tile + at), umma_desc_sw128(kt + at),
                     instr_desc<M, kTileKeys, false>(), k != 0);
            }
            umma_commit(&sm.sfull[j & 1]);
            umma_commit(&sm.kempty[stage]);
            if (j == nt - 1) umma_commit(&sm.qempty);
          }
          if (j > 0) {  // O of tile j - 1
            const int i = j - 1, g = i & 1;
            const uint32_t n = it + (uint32_t)i;
            const int stage = (int)(n % kVS);
            if (i == 0 && !(ok = mbar_wait(&sm.oempty, (wn & 1u) ^ 1u, abort_flag))) break;
            if (!(ok = mbar_wait(&sm.vfull[stage], (n / kVS) & 1u, abort_flag))) break;
            if (!(ok = mbar_wait(&sm.pfull[g], (turns[g] + (uint32_t)(i >> 1)) & 1u, abort_flag))) break;
            tmem_fence_after();
            const uint32_t vt = v_tiles + (uint32_t)stage * kTileBytes;
#pragma unroll
            for (int k = 0; k < kTileKeys / 16; ++k)
              mma_ts(tmem + 256u + (uint32_t)g * 128u, tmem + (uint32_t)g * 128u + (uint32_t)k * 8u, desc_mn_sw128(vt + (uint32_t)k * 2048u),
                     instr_desc<M, D, true>(), i > 1 || k != 0);
            umma_commit(&sm.pvdone[g]);
            umma_commit(&sm.vempty[stage]);
          }
        }
      }
      __syncwarp();
      turns[0] += (uint32_t)(nt + 1) / 2u, turns[1] += (uint32_t)nt / 2u;
      it += (uint32_t)nt;
      ++wn;
      if (*abort_flag) break;
    }
  } else {
    // ---- softmax: group g takes tiles g, g + 2, ..; thread r of a group has head r ----
    const int g = warp >> 2, r = (warp & 3) * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t s_cols = lanes + (uint32_t)g * 128u, o_cols = lanes + 256u + (uint32_t)g * 128u;
    uint32_t turns[2] = {0u, 0u};
    constexpr int kHalf = D / 2;  // columns of O a thread writes
    for (uint32_t unit = first; ok && unit < units; unit += step) {
      const Work w = work_of(p, unit);
      const int all = tiles_of(p.indices + (int64_t)w.token * p.idx_row, p.picks, lane);
      const int nt = all > rank ? (all - rank + ctas - 1) / ctas : 0;
      const bool busy = (warp & 3) * 32 < w.heads, mine = r < w.heads;
      T* const out = static_cast<T*>(p.out) + (int64_t)w.token * p.out_token + (int64_t)(w.head0 + r) * p.out_head + g * kHalf;
      float* const lse = p.lse == nullptr ? nullptr : p.lse + (int64_t)w.token * p.kv_heads * p.group + w.head0 + r;
      if (nt == 0 && ctas == 1) {
        if (mine) {
          float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
          for (int c = 0; c < kHalf; c += 8) store_row(out + c, zero, p.out_vec != 0);
          if (g == 0 && lse != nullptr) *lse = -INFINITY;
        }
        continue;
      }
      float ref = -INFINITY, vlog = 0.f, sum = 0.f;
      const uint32_t turn0 = turns[g];
      for (int j = g; j < nt; j += 2) {
        const uint32_t n = it + (uint32_t)j, turn = turn0 + (uint32_t)(j >> 1);
        const int place = (int)(n % C::kMeta);
        ok = mbar_wait(&sm.mfull[place], (n / C::kMeta) & 1u, abort_flag) && mbar_wait(&sm.sfull[g], turn & 1u, abort_flag);
        if (!(ok = __all_sync(kAll, ok))) break;
        tmem_fence_after();
        if (busy) {
          const TileMeta& m = sm.meta[place];
          const float qmul = sm.qmul[wn & 1u][r];
          float top = -INFINITY;
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            float s[32];
            load_scores<kFp8>(s, s_cols + 32u * c, m.ks + 32 * c, m.live[c]);
#pragma unroll
            for (int i = 0; i < 32; ++i) top = fmaxf(top, s[i]);
          }
          top *= qmul;
          // the references: this head's largest score, and the exponent of the tile's largest v scale
          float vnew = vlog;
          if constexpr (kFp8) {
            const float4 v = *reinterpret_cast<const float4*>(m.vmax);
            const int e = (int)(__float_as_uint(fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w))) >> 23) - 127;
            const float ve = (float)max(-100, min(e, 100));
            if (j == g || ve > vlog + 6.f) vnew = ve;
          }
          const float next = top > ref + kLetStand ? top : ref;
          if (j != g) {
            const bool changed = next != ref || vnew != vlog;
            if (__any_sync(kAll, changed)) {
              const float f = !changed ? 1.f : ref == -INFINITY ? (next == -INFINITY ? 1.f : 0.f) : ex2((ref + vlog) - (next + vnew));
              ok = mbar_wait(&sm.pvdone[g], (turn - 1u) & 1u, abort_flag);
              if (!(ok = __all_sync(kAll, ok))) break;
              tmem_fence_after();
#pragma unroll 1
              for (int c = 0; c < D / 32; ++c) {
                uint32_t v[32];
                tmem_ld32(o_cols + 32u * c, v);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * f);
                tmem_st32(o_cols + 32u * c, v);
              }
              sum *= f;
            }
          }
          ref = next;
          vlog = vnew;
          const float sub = (ref == -INFINITY ? 0.f : ref) + vlog;
          float part = 0.f;
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            float s[32];
            uint32_t pk[16];
            load_scores<kFp8>(s, s_cols + 32u * c, m.ks + 32 * c, m.live[c]);
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              const float a = ex2(fmaf(s[i], qmul, -sub)), b = ex2(fmaf(s[i + 1], qmul, -sub));
              const float d = ex2(fmaf(s[i + 2], qmul, -sub)), e = ex2(fmaf(s[i + 3], qmul, -sub));
              sum += a + b;
              part += d + e;
              float4 v = make_float4(1.f, 1.f, 1.f, 1.f);
              if constexpr (kFp8) v = *reinterpret_cast<const float4*>(m.vs + 32 * c + i);
              pk[i / 2] = kFp8 ? narrow2(a * v.x, b * v.y, M()) : narrow2(a, b, M());
              pk[i / 2 + 1] = kFp8 ? narrow2(d * v.z, e * v.w, M()) : narrow2(d, e, M());
            }
            tmem_st16(s_cols + 16u * c, pk);  // (over scores that have been read)
          }
          sum += part;
          tmem_wait_st();
        }
        tmem_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.pfull[g]);
      }
      if (!ok) break;
      // ---- this piece's end: both groups' products, maxima and sums ----
      const int nga = (nt + 1) / 2, ngb = nt / 2;
      float2 a = make_float2(-INFINITY, 0.f), b = a;
      if (nt > 0) {
        sm.ml[wn & 1u][g][r] = make_float2(ref == -INFINITY ? -INFINITY : ref + vlog, sum);
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.mlbar);
        ok = mbar_wait(&sm.mlbar, wn & 1u, abort_flag) && mbar_wait(&sm.pvdone[0], (turns[0] + (uint32_t)nga - 1u) & 1u, abort_flag);
        if (ngb > 0) ok = ok && mbar_wait(&sm.pvdone[1], (turns[1] + (uint32_t)ngb - 1u) & 1u, abort_flag);
        if (!(ok = __all_sync(kAll, ok))) break;
        tmem_fence_after();
        a = sm.ml[wn & 1u][0][r], b = sm.ml[wn & 1u][1][r];
      }
      const float top = fmaxf(a.x, b.x);
      const float fa = a.x == top ? 1.f : ex2(a.x - top), fb = b.x == top ? 1.f : ex2(b.x - top);
      const float l = fa * a.y + fb * b.y;
      const float inv = ctas > 1 ? 1.f : l == 0.f ? 0.f : 1.f / l;
      float* const stage_row = reinterpret_cast<float*>(base + kTileBytes) + (size_t)r * (D + 4) + g * kHalf;  // (several CTAs: over the k tiles)
      if (busy) {
#pragma unroll 1
        for (int c = 0; c < kHalf; c += 32) {
          float y[32];
          const uint32_t col = lanes + 256u + (uint32_t)(g * kHalf + c);
#pragma unroll
          for (int i = 0; i < 32; ++i) y[i] = 0.f;
#pragma unroll 1
          for (int i = 0; i < 2; ++i) {
            if (i < nt) {
              uint32_t v[32];
              tmem_ld32(col + 128u * i, v);
              tmem_wait_ld();
              const float f = (i == 0 ? fa : fb) * inv;
#pragma unroll
              for (int e = 0; e < 32; ++e) y[e] = fmaf(f, __uint_as_float(v[e]), y[e]);
            }
          }
          if (ctas > 1) {
#pragma unroll
            for (int i = 0; i < 32; i += 4) *reinterpret_cast<float4*>(stage_row + c + i) = make_float4(y[i], y[i + 1], y[i + 2], y[i + 3]);
          } else if (mine) {
            store_row(out + c, y, p.out_vec != 0);
          }
        }
      }
      tmem_fence_before();
      __syncwarp();
      if (nt > 0 && lane == 0) mbar_arrive(&sm.oempty);
      if (g == 0) {
        if (ctas > 1)
          sm.ml[1][0][r] = make_float2(top, l);  // (one piece of work a CTA: the other half is not in use)
        else if (mine && lse != nullptr)
          *lse = l == 0.f ? -INFINITY : top * 0.693147180559945309f + logf(l);
      }
      turns[0] += (uint32_t)nga, turns[1] += (uint32_t)ngb;
      it += (uint32_t)nt;
      wn += nt > 0 ? 1u : 0u;
    }
  }
  __syncwarp();
  tmem_fence_before();
  __syncthreads();
  if (*abort_flag) {
    // a wait ran out: give MMAs that may still be in flight a moment before shared and tensor memory go away
    unsigned long long t0, t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
    do {
      asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    } while (t - t0 < 100000ull);
    if (tid == 0 && p.status) atomicOr(p.status, (uint32_t)FFTOPK_ST_STAGE_TIMEOUT);
  }
  tmem_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  if (ctas > 1) {
    cluster.sync();
    const Work w = work_of(p, first);
    constexpr int kPer = D / 32;  // channels a lane
    const float* mine_o = reinterpret_cast<const float*>(base + kTileBytes);
    for (int h = rank + ctas * warp; h < w.heads; h += ctas * (kWideThreads / 32)) {
      float top = -INFINITY;
      for (int c = 0; c < ctas; ++c) top = fmaxf(top, cluster.map_shared_rank(&sm.ml[1][0][h], c)->x);
      float l = 0.f, acc[kPer];
#pragma unroll
      for (int e = 0; e < kPer; ++e) acc[e] = 0.f;
      for (int c = 0; c < ctas; ++c) {
        const float2 ml = *cluster.map_shared_rank(&sm.ml[1][0][h], c);
        const float f = ml.x == top ? 1.f : ex2(ml.x - top);
        l += f * ml.y;
        const float* o = cluster.map_shared_rank(mine_o, c) + (size_t)h * (D + 4) + lane * kPer;
#pragma unroll
        for (int e = 0; e < kPer; ++e) acc[e] += f * o[e];
      }
      T* out = static_cast<T*>(p.out) + (int64_t)w.token * p.out_token + (int64_t)(w.head0 + h) * p.out_head + lane * kPer;
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const uint32_t v = narrow2(l == 0.f ? 0.f : acc[e] / l, 0.f, T());
        reinterpret_cast<uint16_t*>(out)[e] = (uint16_t)v;
      }
      if (lane == 0 && p.lse != nullptr)
        p.lse[(int64_t)w.token * p.kv_heads * p.group + w.head0 + h] = l == 0.f ? -INFINITY : top * 0.693147180559945309f + logf(l);
    }
    cluster.sync();  // (nobody leaves while its memory is read)
  }
}

template <typename T, bool kFp8, int D>
int setup_wide() {
  const cudaError_t e =
      cudaFuncSetAttribute(attend_wide_kernel<T, kFp8, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)wide_smem_bytes<D>());
  return e == cudaSuccess ? 0 : cuda_fail(e);
}

template <typename T, bool kFp8, int D>
cudaError_t launch_wide(const AttendParams& p, int ctas, int64_t units, int sms, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  const int64_t grid = ctas > 1 ? units * ctas : units < sms ? units : sms;
  cfg.gridDim = dim3((unsigned)grid, 1, 1);
  cfg.blockDim = dim3(kWideThreads, 1, 1);
  cfg.dynamicSmemBytes = wide_smem_bytes<D>();
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)ctas;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, attend_wide_kernel<T, kFp8, D>, p, (uint32_t)units);
}

template <typename T>
cudaError_t launch_wide(const AttendParams& p, bool fp8, int D, int ctas, int64_t units, int sms, cudaStream_t stream) {
  if (fp8) return D == 64 ? launch_wide<T, true, 64>(p, ctas, units, sms, stream) : launch_wide<T, true, 128>(p, ctas, units, sms, stream);
  return D == 64 ? launch_wide<T, false, 64>(p, ctas, units, sms, stream) : launch_wide<T, false, 128>(p, ctas, units, sms, stream);
}

}  // namespace

int attend_wide_setup() {
  int r = setup_wide<__nv_bfloat16, false, 64>();
  if (!r) r = setup_wide<__nv_bfloat16, false, 128>();
  if (!r) r = setup_wide<__nv_bfloat16, true, 64>();
  if (!r) r = setup_wide<__nv_bfloat16, true, 128>();
  if (!r) r = setup_wide<__half, false, 64>();
  if (!r) r = setup_wide<__half, false, 128>();
  if (!r) r = setup_wide<__half, true, 64>();
  if (!r) r = setup_wide<__half, true, 128>();
  return r;
}

cudaError_t attend_wide(const AttendParams& p, bool bf16, bool fp8, int D, int ctas, int64_t units, int sms, cudaStream_t stream) {
  return bf16 ? launch_wide<__nv_bfloat16>(p, fp8, D, ctas, units, sms, stream) : launch_wide<__half>(p, fp8, D, ctas, units, sms, stream);
}

}  // namespace fftopk
