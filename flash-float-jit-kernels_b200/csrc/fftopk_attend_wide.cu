// Attention over selected rows for many query heads to a key head: the tensor cores' share of fftopk_attend.cu (the formulas
// stand there; which calls come here: attend_is_wide in fftopk_decide.h).
//
// 128 query heads use a row of k and v here, 2 * 128 flop per element: 128 a byte in 16 bits, where a cache whose rows no tokens share
// is bound by memory (the device has 250), 256 in fp8, and a multiple of that wherever tokens share rows out of L2. So the products run
// on tcgen05, one CTA per SM:
//   S[128 heads x 128 keys] = Q K^T    Q, K in shared memory (K-major, 128-byte swizzle), S in tensor memory
//   O[128 heads x D]       += P V      P in tensor memory (16 bits, over the S it came from), V in shared memory as it lies in the
//                                      cache, [key][channel]: an MN-major operand
// 20 warps: two groups of four softmax warps, one thread per head, that take alternate tiles of keys, each with an S, an O and a
// running maximum of its own, so that one group's exponentials run while the other's products do; one that looks up which rows
// the tiles to come are made of (and, fp8, their scales) and hands them out as a stream of TileMeta; four that gather k rows and
// four that gather v rows; two that bring the queries of the next piece of work; and one thread that issues the MMAs, whichever
// are ready: QK of a tile as soon as PV of the tile two before it has been issued, PV in halves of a tile's keys. The rows lie
// anywhere: 16-bit ones are copied into their tile with cp.async; e4m3 codes into a ring of the gathering warp's own, which widens
// them to fp16 in the tile. Rows that are not there are zeros, and masked in S.
//
// What bounds it (1,024 tokens of 128 heads on one key head, 2,048 picks of 65,536 shared rows; 112 tiles a CTA, clock 1,965 MHz): bf16
// 198 us, 690 TFLOP/s, 3,500 cycles a tile where its products take 1,030. Nothing is used up (tcgen05 32 %, issue slots 42 %): a tile waits
// in turn for its rows out of L2, for softmax (1,024 cycles of exponentials a warp) and to be handed on. e4m3 313 us, 5,500 cycles a tile:
// the same (tcgen05 23 %, issue slots 43 %), with codes of one tile on their way at a time at D = 128 (kRaw) and 8,800 warp instructions a
// tile where bf16 has 6,050, for the scales in softmax and widening the codes. ptxas spills 104 to 132 bytes of stores at D = 128 (by role
// 128, 80 and 64 registers), 8 to 50 at 64.
//
// A row's maximum is let stand until a score exceeds it by 2^8 (fp16 and 32-bit sums have the room), so O, which lives in tensor
// memory, is hardly ever rescaled. fp8: the k scales multiply S, the v scales P, and the reference is the largest score + log2 |v scale|,
// what a row adds being its weight times its scale; where a tile's v scales lie within 2^kEvenLog the largest of them stands for all,
// which saves looking at them one by one (1,024 tokens of 128 heads: 313 us, 346 with scales further apart). At the end the groups' O
// are added, row by row, with the factors their references give.
// A CTA takes one piece of work after the other (token, key head, 128 query heads), and its gathering warps run ahead into the next
// one. Few tokens: the CTAs of a cluster take every n-th tile, and join through distributed shared memory.
// Every wait on an mbarrier has a time limit; when one runs out the CTA raises FFTOPK_ST_STAGE_TIMEOUT, writes NaN for what it has
// not finished and winds down.
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
constexpr int kSoftmaxWarps = 8, kGatherWarps = 8, kQueryWarps = 2;
constexpr int kMmaWarp = kSoftmaxWarps + kGatherWarps, kScoutWarp = kMmaWarp + 1, kQueryWarp = kScoutWarp + 1;
constexpr int kWideThreads = (kQueryWarp + kQueryWarps) * 32;
// Registers a thread: 640 threads are launched with 96 each; by warpgroup 2 x 128 (softmax: 64 scores at once), 2 x 80 (gather) and
// 64 (the rest) are the same 480.
constexpr int kRegsLaunch = 96, kRegsSoftmax = 128, kRegsGather = 80, kRegsRest = 64;
static_assert(2 * kRegsSoftmax + 2 * kRegsGather + kRegsRest == kWideThreads / 128 * kRegsLaunch, "no more registers than the block has");
template <int N>
__device__ __forceinline__ void more_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void fewer_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
constexpr uint32_t kTmemCols = 512;
constexpr float kLetStand = 8.f;  // log2 by which a score may exceed the reference
constexpr int kEvenLog = 4;       // weights may be smaller than the reference says by that many bits: of the 25 that fp16 reaches down

// What lies in shared memory beside the query tile: k and v tiles as the MMAs read them; and, e4m3, every gathering warp's share of
// the codes of tiles on their way.
template <bool kFp8, int D>
struct WideCfg {
  static constexpr uint32_t kTileBytes = kTileKeys * D * 2;  // of Q too
  // (1,024 tokens of 128 heads on one e4m3 key head, when the kernel took 344 us: one k and one v tile, codes of two and a query tile
  // ahead 362)
  static constexpr int kQTiles = D == 128 && kFp8 ? 1 : 2, kKStages = 2, kVStages = 2;
  static_assert(kKStages >= 2, "softmax may be a tile behind QK, whose barriers are the k stages'");
  static constexpr int kRaw = kFp8 ? (D == 64 ? 4 : 1) : 0;
  static constexpr uint32_t kRawBytes = 32 * D;              // of a warp and tile
  static constexpr size_t kTiles = (size_t)kTileBytes * (kQTiles + kKStages + kVStages), kOperands = kTiles + (size_t)kRaw * kGatherWarps * kRawBytes;
};
static_assert(kTileKeys == 128);
constexpr int kChunk = 64;    // scores of a row that a softmax thread works on at once
constexpr int kMeta = 4;      // tiles the scout is ahead at most; a place is free again when its tile's PV is done
constexpr int kPauseNs = 64;  // of the thread that issues the MMAs, between two looks at what it waits for
constexpr int kInfo = 4;      // pieces of work it is ahead
constexpr int kLast = 1, kEnd = 2, kWhole = 4, kSeen = 8, kEven = 16;
struct TileMeta {             // a tile of 128 keys
  int64_t k_at[kTileKeys], v_at[kTileKeys];  // byte offsets of the rows in the caches; negative: none
  float ks[kTileKeys], vs[kTileKeys], vlog[kTileKeys];  // vlog: the v scales' exponents
  uint32_t live[4];
  float vmost;                // the largest of them
  int32_t flags;              // last tile of its piece of work; end of the stream (no tile); all rows are there; their v scales are alike
  int32_t kvh;
};
template <bool kFp8, int D>
struct WideSmem {  // behind the operand tiles
  TileMeta meta[kMeta];
  float qmul[4][kHeadsW];    // by piece of work: softmax may be two behind the queries
  float2 ml[2][2][kHeadsW];  // by parity of the piece of work, and group: maximum and sum
  int32_t tiles[kInfo];      // tiles of a piece of work
  // A place of a ring is free again when the MMAs that read it are done, which one commit tells all who wait for them.
  uint64_t kfull[WideCfg<kFp8, D>::kKStages], sdone[WideCfg<kFp8, D>::kKStages];  // k has landed; QK is done: S is there, k may be replaced
  uint64_t vfull[WideCfg<kFp8, D>::kVStages];
  uint64_t mfull[kMeta], pvdone[kMeta];  // TileMeta is there; PV is done: v and TileMeta may be replaced, O is up to this tile
  uint64_t ifull[kInfo], iempty[kInfo];
  uint64_t qfull[WideCfg<kFp8, D>::kQTiles], qempty[WideCfg<kFp8, D>::kQTiles], oempty, mlbar;
  uint64_t pfull[2][2], halfdone[2];     // by group: a half of P is there; PV of the first half is done
  uint32_t tmem, abort_flag;
};
template <bool kFp8, int D>
constexpr size_t wide_smem_bytes() {
  return 1024 + WideCfg<kFp8, D>::kOperands + sizeof(WideSmem<kFp8, D>);
}

// Matrix descriptors as their two halves: only the lower one, address and leading offset, differs from operand to operand, and
// 16-byte units may be added to it. K-major (Q, K): see umma_desc_sw128. V as it lies in the cache is an MN-major operand, 128-byte
// swizzle: blocks of 64 channels x 128 keys, 128 bytes a key; 8 keys are 1024 bytes apart (stride offset), blocks of channels 16 KiB
// (leading offset).
__device__ __forceinline__ uint32_t desc_k(uint32_t smem_addr) { return (uint32_t)umma_desc_sw128(smem_addr); }
__device__ __forceinline__ uint32_t desc_mn(uint32_t smem_addr) {  // (of a cluster's CTAs, addresses have more bits)
  return ((smem_addr >> 4) & 0x3fffu) | ((kTileKeys * 128u) >> 4) << 16;
}
constexpr uint32_t kDescHigh = (1024u >> 4) | 1u << 14 | 2u << 29;  // stride offset, version, 128-byte swizzle
template <typename M, int N, bool kMnMajorB>
__host__ __device__ constexpr uint32_t instr_desc() {  // D fp32; A and B fp16 or bf16; M = 128
  constexpr uint32_t f = std::is_same<M, __half>::value ? 0u : 1u;
  return (1u << 4) | (f << 7) | (f << 10) | ((kMnMajorB ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(kHeadsW >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "n"(kDescHigh)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "n"(kDescHigh)
      : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
        "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
      "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void load_chunk(uint32_t taddr, float (&s)[64]) {
  tmem_ld32(taddr, reinterpret_cast<uint32_t(&)[32]>(s[0]));
  tmem_ld32(taddr + 32u, reinterpret_cast<uint32_t(&)[32]>(s[32]));
}
__device__ __forceinline__ void store_chunk(uint32_t taddr, const uint32_t (&v)[32]) {
  tmem_st16(taddr, reinterpret_cast<const uint32_t(&)[16]>(v[0]));
  tmem_st16(taddr + 16u, reinterpret_cast<const uint32_t(&)[16]>(v[16]));
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {  // zeros where it is not
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void get16(uint32_t (&v)[4], uint32_t src) {
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(src) : "memory");
}
__device__ __forceinline__ void put16(uint32_t dst, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// 16-byte chunk c of row r of a tile: blocks of 64 channels, 128 bytes a row, swizzled
__device__ __forceinline__ uint32_t chunk_at(uint32_t tile, int r, int c) {
  return tile + (uint32_t)(c >> 3) * (kTileKeys * 128u) + (uint32_t)r * 128u + (uint32_t)(((c & 7) ^ (r & 7)) << 4);
}

__device__ __forceinline__ int tiles_up_to(int picks) { return (int)(((uint32_t)picks + kTileKeys - 1u) / kTileKeys); }
// tiles of a token's picks up to the last entry that is not negative (by a whole warp). It is looked for among the last kLookBack
// entries, a millisecond at most: everybody waits meanwhile, and a list of 2^28 would outlast the limit of their waits.
constexpr int kLookBack = 1 << 20;
__device__ __forceinline__ int tiles_of(const int32_t* idx, int picks, int lane) {
  const int until = max(picks - kLookBack, 0);
  for (int hi = picks; hi > until; hi -= 512) {
    int last = -1;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int j = hi - 1 - (i * 32 + lane);
      if (j >= 0 && idx[j] >= 0) last = max(last, j);
    }
    last = __reduce_max_sync(kAll, last);
    if (last >= 0) return last / kTileKeys + 1;
  }
  return tiles_up_to(until);
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

// the largest of a thread's kChunk scores
__device__ __forceinline__ float top_of(const float (&s)[kChunk]) {
  float top[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) top[i] = fmaxf(s[2 * i], s[2 * i + 1]);
#pragma unroll
  for (int i = 8; i < kChunk; i += 8) {
#pragma unroll
    for (int e = 0; e < 4; ++e) top[e] = fmaxf(top[e], fmaxf(s[i + 2 * e], s[i + 2 * e + 1]));
  }
  return fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
}

// the largest of them, times qmul, with their rows' v scales
__device__ __forceinline__ float top_with(const float (&s)[kChunk], float qmul, const float* vlog) {
  const Pair mul = pair(qmul, qmul);
  float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int i = 0; i < kChunk; i += 4) {
    const float4 x = *reinterpret_cast<const float4*>(vlog + i);
    const float2 a = apart(fma2(pair(s[i], s[i + 1]), mul, pair(x.x, x.y))), b = apart(fma2(pair(s[i + 2], s[i + 3]), mul, pair(x.z, x.w)));
    top[0] = fmaxf(top[0], a.x), top[1] = fmaxf(top[1], a.y), top[2] = fmaxf(top[2], b.x), top[3] = fmaxf(top[3], b.y);
  }
  return fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
}

// pairs of 16-bit values
template <typename T, int N>
__device__ __forceinline__ void store_row(T* out, const uint32_t (&v)[N], bool vec) {
  if (vec) {
#pragma unroll
    for (int i = 0; i < N; i += 4) *reinterpret_cast<uint4*>(out + 2 * i) = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      reinterpret_cast<uint16_t*>(out)[2 * i] = (uint16_t)v[i];
      reinterpret_cast<uint16_t*>(out)[2 * i + 1] = (uint16_t)(v[i] >> 16);
    }
  }
}

// what softmax thread (r, g) leaves for the pieces of work from `unit` on where a wait ran out (a function of its own: hardly ever run,
// and its registers are not the loop's)
template <typename T, int D>
__device__ __noinline__ void leave_nan(const AttendParams& p, uint32_t unit, uint32_t units, uint32_t step, int r, int g) {
  const uint32_t nan[4] = {0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu};
  for (; unit < units; unit += step) {
    const Work w = work_of(p, unit);
    if (r >= w.heads) continue;
    T* const out = static_cast<T*>(p.out) + (int64_t)w.token * p.out_token + (int64_t)(w.head0 + r) * p.out_head + g * (D / 2);
    for (int c = 0; c < D / 2; c += 8) store_row(out + c, nan, p.out_vec != 0);
    if (g == 0 && p.lse != nullptr) p.lse[(int64_t)w.token * p.kv_heads * p.group + w.head0 + r] = __int_as_float(0x7fffffff);
  }
}

template <typename T, bool kFp8, int D>
__global__ void __launch_bounds__(kWideThreads, 1) attend_wide_kernel(const __grid_constant__ AttendParams p, const uint32_t units) {
  using M = typename std::conditional<kFp8, __half, T>::type;
  using C = WideCfg<kFp8, D>;
  constexpr uint32_t kTileBytes = C::kTileBytes;
  constexpr int kKS = C::kKStages, kVS = C::kVStages;
  extern __shared__ unsigned char wide_raw[];
  const uint32_t pad = (1024u - (smem_u32(wide_raw) & 1023u)) & 1023u;
  unsigned char* base = wide_raw + pad;
  constexpr uint32_t kQTiles = C::kQTiles;
  const uint32_t q_tiles = smem_u32(base), k_tiles = q_tiles + kQTiles * kTileBytes, v_tiles = k_tiles + kKS * kTileBytes;
  WideSmem<kFp8, D>& sm = *reinterpret_cast<WideSmem<kFp8, D>*>(base + C::kOperands);
  volatile uint32_t* abort_flag = &sm.abort_flag;

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const uint32_t first = blockIdx.x / (uint32_t)ctas, step = gridDim.x / (uint32_t)ctas;

  if (tid == 0) {
    for (int i = 0; i < kKS; ++i) mbar_init(&sm.kfull[i], 4), mbar_init(&sm.sdone[i], 1);
    for (int i = 0; i < kVS; ++i) mbar_init(&sm.vfull[i], 4);
    for (int i = 0; i < kMeta; ++i) mbar_init(&sm.mfull[i], 1), mbar_init(&sm.pvdone[i], 1);
    for (int i = 0; i < kInfo; ++i) mbar_init(&sm.ifull[i], 1), mbar_init(&sm.iempty[i], kSoftmaxWarps + kQueryWarps);
    for (int i = 0; i < C::kQTiles; ++i) mbar_init(&sm.qfull[i], kQueryWarps), mbar_init(&sm.qempty[i], 1);
    mbar_init(&sm.oempty, kSoftmaxWarps);
    mbar_init(&sm.mlbar, kSoftmaxWarps);
    for (int i = 0; i < 2; ++i) mbar_init(&sm.pfull[i][0], 4), mbar_init(&sm.pfull[i][1], 4), mbar_init(&sm.halfdone[i], 1);
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
  // Tiles are counted through all pieces of work (n, it), and so are pieces (un) and those that have tiles (wn): the counts select
  // places and stages and the phases of their barriers.

  if (warp >= kSoftmaxWarps && warp < kMmaWarp) {
    // ---- gather: four warps for k, four for v; rows 32 gw .. 32 gw + 31 of every tile ----
    fewer_registers<kRegsGather>();
    const bool is_k = warp < kSoftmaxWarps + 4;
    const int gw = (warp - kSoftmaxWarps) & 3;
    uint64_t* const full = is_k ? sm.kfull : sm.vfull;
    uint64_t* const empty = is_k ? sm.sdone : sm.pvdone;  // of the tile `stages` before
    const uint32_t ring = is_k ? kKS : kMeta;
    const uint32_t stages = is_k ? kKS : kVS;
    const uint32_t tiles = is_k ? k_tiles : v_tiles;
    constexpr int kLanesRow = D * (kFp8 ? 1 : 2) / 16;  // lanes that read a row
    constexpr int kRowsOnce = 32 / kLanesRow, kTurns = 32 / kRowsOnce;
    // Eight lanes that write to shared memory together touch all its banks: 16-bit, a row's 128 bytes; e4m3, where a lane writes
    // two neighbouring chunks one after the other, half of those of two neighbouring rows.
    const int piece = kFp8 && kLanesRow == 8 ? (lane & 3) | ((lane >> 3 & 1) << 2) : lane % kLanesRow;
    const int sub = gw * 32 + (kFp8 && kLanesRow == 8 ? (lane >> 2 & 1) | ((lane >> 4) << 1) : lane / kLanesRow);
    const int64_t head_bytes = (is_k ? p.k_head : p.v_head) * (kFp8 ? 1 : 2);
    const char* const src0 = static_cast<const char*>(is_k ? p.k : p.v) + piece * 16;
    auto posted = [&](uint32_t n) { return __all_sync(kAll, mbar_test(&sm.mfull[n % kMeta], (n / kMeta) & 1u)); };
    // (in a test the first of all waits to run out; the others see abort_flag)
    auto wait_posted = [&](uint32_t n) { return __all_sync(kAll, mbar_wait(&sm.mfull[n % kMeta], (n / kMeta) & 1u, abort_flag, p.wait_ns)); };
    auto wait_empty = [&](uint32_t n) {
      const uint32_t of = n - stages;
      return n < stages || __all_sync(kAll, mbar_wait(&empty[of % ring], (of / ring) & 1u, abort_flag));
    };
    auto is_empty = [&](uint32_t n) {
      const uint32_t of = n - stages;
      return n < stages || __all_sync(kAll, mbar_test(&empty[of % ring], (of / ring) & 1u));
    };
    auto hand_over = [&](uint32_t n) {
      fence_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&full[n % stages]);
    };
    if constexpr (kFp8) {
      // Codes are copied to the warp's own ring; a tile's are widened to fp16 once they are there and the tile's place is free.
      const uint32_t raw = q_tiles + (uint32_t)C::kTiles + (uint32_t)(warp - kSoftmaxWarps) * C::kRaw * C::kRawBytes + (uint32_t)lane * 16u;
      uint32_t to[2][2];  // where the lane's two chunks go in a tile, turn 0 and turn 1 (without the turn's rows)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int e = 0; e < 2; ++e) to[i][e] = chunk_at(0u, sub + i * kRowsOnce, 2 * piece + e) - (uint32_t)(i * kRowsOnce * 128);
      }
      uint32_t asked = 0;      // tiles whose codes are asked for
      bool ended = false;      // the stream, at `asked` tiles
      auto ask = [&] {         // tile `asked`, which is posted
        const TileMeta& m = sm.meta[asked % kMeta];
        ended = (m.flags & kEnd) != 0;
        if (!ended) {
          const char* src = src0 + m.kvh * head_bytes;
          const int64_t* rows_at = (is_k ? m.k_at : m.v_at) + sub;
          const uint32_t at = raw + (asked % C::kRaw) * C::kRawBytes;
#pragma unroll
          for (int i = 0; i < kTurns; ++i) {
            const int64_t row = rows_at[i * kRowsOnce];
            copy16(at + i * 512u, src + (row >= 0 ? row : 0), row >= 0);
          }
          ++asked;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
      for (uint32_t n = 0;; ++n) {
        if (asked == n) {  // (nothing on its way: wait for the scout)
          if (!ended && !wait_posted(n)) break;
          if (!ended) ask();
          if (ended) break;
        }
        while (!ended && asked < n + C::kRaw && posted(asked)) ask();
        // (the codes of a lane are its own copies: no other lane's wait is needed)
        if (asked - n == 1u)
          asm volatile("cp.async.wait_group 0;" ::: "memory");
        else if (asked - n == 2u)
          asm volatile("cp.async.wait_group 1;" ::: "memory");
        else if (asked - n == 3u)
          asm volatile("cp.async.wait_group 2;" ::: "memory");
        else
          asm volatile("cp.async.wait_group 3;" ::: "memory");
        const uint32_t tile = tiles + (n % stages) * kTileBytes, at = raw + (n % C::kRaw) * C::kRawBytes;
        if (!wait_empty(n)) break;
#pragma unroll
        for (int i = 0; i < kTurns; ++i) {
          uint32_t x[4], h[8];
          get16(x, at + i * 512u);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            h[2 * e] = e4m3x2_to_half2((uint16_t)x[e]);
            h[2 * e + 1] = e4m3x2_to_half2((uint16_t)(x[e] >> 16));
          }
          // (rows of every second turn have their chunks in the same order)
          const uint32_t by = tile + (uint32_t)(i * kRowsOnce * 128);
          put16(by + to[i & 1][0], h[0], h[1], h[2], h[3]);
          put16(by + to[i & 1][1], h[4], h[5], h[6], h[7]);
        }
        hand_over(n);
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
    } else {
      bool pending = false;  // tile n - 1 is on its way and not handed over
      for (uint32_t n = 0;; ++n) {
        // a tile that has landed is not kept waiting for the next one's turn
        if (pending && !(posted(n) && is_empty(n))) {
          asm volatile("cp.async.wait_group 0;" ::: "memory");
          hand_over(n - 1);
          pending = false;
        }
        if (!wait_posted(n)) break;
        const TileMeta& m = sm.meta[n % kMeta];
        if (m.flags & kEnd) {
          asm volatile("cp.async.wait_group 0;" ::: "memory");
          if (pending) hand_over(n - 1);
          break;
        }
        if (!wait_empty(n)) break;
        const char* src = src0 + m.kvh * head_bytes;
        const int64_t* rows_at = (is_k ? m.k_at : m.v_at) + sub;
        const uint32_t tile = tiles + (n % stages) * kTileBytes;
#pragma unroll
        for (int i = 0; i < kTurns; ++i) {
          const int64_t row = rows_at[i * kRowsOnce];
          copy16(chunk_at(tile, sub + i * kRowsOnce, piece), src + (row >= 0 ? row : 0), row >= 0);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        if (pending) {
          asm volatile("cp.async.wait_group 1;" ::: "memory");
          hand_over(n - 1);
        }
        pending = true;
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
    }
  } else if (warp >= kMmaWarp) {
    fewer_registers<kRegsRest>();
    if (warp == kScoutWarp) {
      // ---- scout: what the tiles to come are made of ----
      uint32_t n = 0, un = 0;
      bool ok = true;
      // how many tiles a piece of work has, told to those who need not wait for the tiles themselves
      auto tell = [&](uint32_t unit, uint32_t un) {
        const int32_t* idx = p.indices + (int64_t)work_of(p, unit).token * p.idx_row;
        // (several CTAs a token: tiles without a row cost less than looking for the last)
        const int all = ctas > 1 ? tiles_up_to(p.picks) : tiles_of(idx, p.picks, lane);
        const int nt = all > rank ? (all - rank + ctas - 1) / ctas : 0;
        ok = __all_sync(kAll, mbar_wait(&sm.iempty[un % kInfo], ((un / kInfo) & 1u) ^ 1u, abort_flag));
        if (ok && lane == 0) {
          sm.tiles[un % kInfo] = nt;
          mbar_arrive(&sm.ifull[un % kInfo]);
        }
        return nt;
      };
      int nt_next = first < units ? tell(first, 0u) : 0;
      for (uint32_t unit = first; ok && unit < units; unit += step, ++un) {
        const Work w = work_of(p, unit);
        const int32_t* idx = p.indices + (int64_t)w.token * p.idx_row;
        const int nt = nt_next;
        nt_next = unit + step < units ? tell(unit + step, un + 1u) : 0;
        if (!ok) break;
        const int64_t offset = p.offsets != nullptr ? p.offsets[w.token] : 0;
        auto pick = [&](int (&to)[4], int j) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t at = (uint32_t)(rank + j * ctas) * kTileKeys + (uint32_t)(i * 32 + lane);
            to[i] = j < nt && at < (uint32_t)p.picks ? idx[at] : -1;
          }
        };
        auto rows_of = [&](int (&row)[4], float (&ks)[4], float (&vs)[4], const int (&from)[4]) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int64_t slot = from[i] + offset;
            const bool there = from[i] >= 0 && slot >= 0 && slot < p.slots;
            if (from[i] >= 0 && !there && p.status) atomicOr(p.status, (uint32_t)FFTOPK_ST_BAD_INDEX);
            row[i] = there ? (int)slot : -1;
            ks[i] = vs[i] = 0.f;
            if constexpr (kFp8) {
              if (there) {
                ks[i] = __ldg(p.k_scale + slot * p.ks_slot + (int64_t)w.kvh * p.ks_head);
                vs[i] = __ldg(p.v_scale + slot * p.vs_slot + (int64_t)w.kvh * p.vs_head);
              }
            }
          }
        };
        // an index is asked for two tiles ahead, a scale one
        int now[4], later[4], row[4];
        float ks[4], vs[4];
        pick(now, 0);
        pick(later, 1);
        rows_of(row, ks, vs, now);
        for (int j = 0; j < nt; ++j, ++n) {
          if (n >= p.stop_after) ok = false;
          if (!ok) break;
          int next_row[4];
          float next_ks[4], next_vs[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) now[i] = later[i];
          pick(later, j + 2);
          rows_of(next_row, next_ks, next_vs, now);
          if (!(ok = __all_sync(kAll, mbar_wait(&sm.pvdone[n % kMeta], ((n / kMeta) & 1u) ^ 1u, abort_flag)))) break;
          TileMeta& m = sm.meta[n % kMeta];
          int most = -100, least = 100;  // exponents of the v scales (16 bits: none)
          unsigned whole = kAll;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            m.k_at[i * 32 + lane] = row[i] < 0 ? -1 : row[i] * (p.k_slot * (kFp8 ? 1 : 2));
            m.v_at[i * 32 + lane] = row[i] < 0 ? -1 : row[i] * (p.v_slot * (kFp8 ? 1 : 2));
            const unsigned live = __ballot_sync(kAll, row[i] >= 0);
            whole &= live;
            if (lane == 0) m.live[i] = live;
            if constexpr (kFp8) {
              m.ks[i * 32 + lane] = ks[i];
              m.vs[i * 32 + lane] = vs[i];
              const int e = scale_exponent(vs[i]);
              m.vlog[i * 32 + lane] = (float)e;
              if (row[i] >= 0) most = max(most, e), least = min(least, e);
            }
          }
          if constexpr (kFp8) most = __reduce_max_sync(kAll, most), least = __reduce_min_sync(kAll, least);
          if (lane == 0) {
            m.flags = (j == nt - 1 ? kLast : 0) | (whole == kAll ? kWhole : 0) | (kFp8 && most - least <= kEvenLog ? kEven : 0);
            if constexpr (kFp8) m.vmost = (float)most;
            m.kvh = w.kvh;
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.mfull[n % kMeta]);
#pragma unroll
          for (int i = 0; i < 4; ++i) row[i] = next_row[i], ks[i] = next_ks[i], vs[i] = next_vs[i];
        }
      }
      if (ok && __all_sync(kAll, mbar_wait(&sm.pvdone[n % kMeta], ((n / kMeta) & 1u) ^ 1u, abort_flag)) && lane == 0) {
        sm.meta[n % kMeta].flags = kEnd;
        mbar_arrive(&sm.mfull[n % kMeta]);
      }
    } else if (warp >= kQueryWarp) {
      // ---- queries: two warps, 64 rows each ----
      const float negative = p.scale_log2 < 0.f ? -1.f : 1.f;
      const uint32_t flip = p.scale_log2 < 0.f ? 0x80008000u : 0u;  // (a negative scale turns q: the largest score is then the largest here)
      const uint32_t none = p.scale_log2 != p.scale_log2 ? 0x7fff7fffu : 0u;  // (a scale that is NaN makes q NaN: scores are, masked ones are not)
      constexpr int kQLanes = D / 8, kQOnce = 32 / kQLanes, kTurns = 64 / kQOnce, kBatch = 8;
      // (the piece of work to come: its rows are brought to L2 while this one's keys go by)
      auto prefetch = [&](uint32_t unit) {
        const Work w = work_of(p, unit);
        const T* q = static_cast<const T*>(p.q) + (int64_t)w.token * p.q_token + (int64_t)w.head0 * p.q_head;
        for (int h = (warp - kQueryWarp) * 32 + lane; h < w.heads; h += 64) {
#pragma unroll
          for (int b = 0; b < D * 2; b += 128)
            asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<const char*>(q + (int64_t)h * p.q_head) + b) : "memory");
        }
      };
      const int c = lane % kQLanes, sub = (warp - kQueryWarp) * 64 + lane / kQLanes;
      uint32_t un = 0, wn = 0;
      for (uint32_t unit = first; unit < units; unit += step, ++un) {
        if (!__all_sync(kAll, mbar_wait(&sm.ifull[un % kInfo], (un / kInfo) & 1u, abort_flag))) break;
        const int nt = sm.tiles[un % kInfo];
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.iempty[un % kInfo]);
        if (nt == 0) continue;
        const Work w = work_of(p, unit);
        const T* q0 = static_cast<const T*>(p.q) + (int64_t)w.token * p.q_token + (int64_t)w.head0 * p.q_head + c * 8;
#pragma unroll 1
        for (int b = 0; b < kTurns; b += kBatch) {
          uint4 x[kBatch];
#pragma unroll
          for (int i = 0; i < kBatch; ++i) {
            const int h = sub + (b + i) * kQOnce;
            x[i] = h < w.heads ? ldg16(q0 + (int64_t)h * p.q_head) : make_uint4(0u, 0u, 0u, 0u);
          }
          if (b == 0 && !__all_sync(kAll, mbar_wait(&sm.qempty[wn % kQTiles], ((wn / kQTiles) & 1u) ^ 1u, abort_flag))) break;
#pragma unroll
          for (int i = 0; i < kBatch; ++i) {
            const int h = sub + (b + i) * kQOnce;
            uint4 v = x[i];
            float mul = p.scale_log2 * negative;
            if constexpr (kFp8 && !std::is_same<T, __half>::value) {
              // to magnitudes below 2, as fp16 (see fftopk_attend.cu)
              const float2 a = widen2(v.x, T()), b2 = widen2(v.y, T()), d = widen2(v.z, T()), e = widen2(v.w, T());
              float amax = fmaxf(fmaxf(fmaxf(fabsf(a.x), fabsf(a.y)), fmaxf(fabsf(b2.x), fabsf(b2.y))),
                                 fmaxf(fmaxf(fabsf(d.x), fabsf(d.y)), fmaxf(fabsf(e.x), fabsf(e.y))));
#pragma unroll
              for (int o = kQLanes / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(kAll, amax, o));
              const uint32_t ex = __float_as_uint(amax) >> 23;
              const uint32_t ee = ex == 255u ? 127u : max(1u, min(ex, 253u));
              const float down = __uint_as_float((254u - ee) << 23);
              mul *= __uint_as_float(ee << 23);
              v = make_uint4(narrow2(a.x * down, a.y * down, __half()), narrow2(b2.x * down, b2.y * down, __half()),
                             narrow2(d.x * down, d.y * down, __half()), narrow2(e.x * down, e.y * down, __half()));
            }
            put16(chunk_at(q_tiles + (wn % kQTiles) * kTileBytes, h, c), (v.x ^ flip) | none, (v.y ^ flip) | none, (v.z ^ flip) | none, (v.w ^ flip) | none);
            if (c == 0) sm.qmul[wn & 3u][h] = fmaxf(mul, 1.17549435e-38f);  // (times a masked score it must stay -inf)
          }
        }
        fence_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.qfull[wn % kQTiles]);
        if (unit + step < units) prefetch(unit + step);
        ++wn;
      }
    } else if (warp == kMmaWarp) {
      // ---- the MMAs ----
      // A group's PV frees the place its next S goes to: QK of tile n stands right behind PV of tile n - 2, and what QK waits for is
      // looked at before PV's weights are there.
      if (lane == 0) {
        uint32_t qn = 0, pn = 0;      // tiles whose QK, whose PV has been issued
        uint32_t qwn = 0, pwn = 0;    // pieces of work they are of
        int qj = 0, pj = 0;           // and tiles of those
        uint32_t flags = 0u, pflags = 0u;  // of tile qn, once it is ready; of the tiles between QK and PV, a byte each
        bool ended = false;           // the stream, at qn tiles
        auto ready = [&] {  // tile qn's k and q are there; sets `ended` where there is no such tile
          if (flags == 0u) {
            if (!mbar_test(&sm.mfull[qn % kMeta], (qn / kMeta) & 1u)) return false;
            flags = (uint32_t)sm.meta[qn % kMeta].flags | kSeen;
            if (flags & kEnd) {
              ended = true;
              return false;
            }
          }
          return (qj != 0 || mbar_test(&sm.qfull[qwn % kQTiles], (qwn / kQTiles) & 1u)) && mbar_test(&sm.kfull[qn % kKS], (qn / kKS) & 1u);
        };
        auto qk = [&] {
          tmem_fence_after();
          const uint32_t stage = qn % kKS;
          const uint32_t kt = desc_k(k_tiles + stage * kTileBytes), q = desc_k(q_tiles + (qwn % kQTiles) * kTileBytes), d = tmem + (qn & 1u) * 128u;
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t at = ((uint32_t)(k >> 2) * (kTileKeys * 128u) + (uint32_t)(k & 3) * 32u) >> 4;
            mma_ss(d, q + at, kt + at, instr_desc<M, kTileKeys, false>(), k != 0);
          }
          umma_commit(&sm.sdone[qn % kKS]);
          const bool last = (flags & kLast) != 0;
          if (last) umma_commit(&sm.qempty[qwn % kQTiles]);
          pflags |= flags << (8u * (qn & 1u));
          flags = 0u;
          ++qn;
          qj = last ? 0 : qj + 1;
          qwn += last ? 1u : 0u;
        };
        // What can go next goes next: the products that wait for something are looked at in turn. PV of a tile goes in two halves of its
        // keys: the first half's products run beside the second half's exponentials.
        bool half = false;            // PV of tile pn: its first half has been issued
        int idle_turns = 0;           // looks in a row that found nothing to issue
        for (;;) {
          bool idle = true;
          // (two tiles at most are between their QK and their PV: one a group)
          if (!ended && qn - pn < 2u && ready()) {
            qk();
            idle = false;
          }
          if (qn == pn) {
            if (ended) break;
          } else {
            const uint32_t g = pn & 1u, stage = pn % kVS, phase = (pn >> 1) & 1u;
            const uint32_t vt = desc_mn(v_tiles + stage * kTileBytes), s_at = tmem + g * 128u;
            // (the first PV of a piece of work: O may still be on its way out)
            if (!half && mbar_test(&sm.pfull[g][0], phase) && mbar_test(&sm.vfull[stage], (pn / kVS) & 1u) &&
                (pj != 0 || mbar_test(&sm.oempty, (pwn & 1u) ^ 1u))) {
              tmem_fence_after();
#pragma unroll
              for (int k = 0; k < kTileKeys / 32; ++k)
                mma_ts(s_at + 256u, s_at + (uint32_t)k * 8u, vt + (uint32_t)k * (2048u >> 4), instr_desc<M, D, true>(), k != 0 || pj > 1);
              umma_commit(&sm.halfdone[g]);
              half = true;
              idle = false;
            }
            if (half && mbar_test(&sm.pfull[g][1], phase)) {
              tmem_fence_after();
#pragma unroll
              for (int k = kTileKeys / 32; k < kTileKeys / 16; ++k)
                mma_ts(s_at + 256u, s_at + (uint32_t)k * 8u, vt + (uint32_t)k * (2048u >> 4), instr_desc<M, D, true>(), 1u);
              umma_commit(&sm.pvdone[pn % kMeta]);
              const bool last = (pflags >> (8u * g) & kLast) != 0u;
              pflags &= 0xff00u >> (8u * g);
              ++pn;
              pj = last ? 0 : pj + 1;
              pwn += last ? 1u : 0u;
              half = false;
              idle = false;
            }
          }
          if (!idle) {
            idle_turns = 0;
          } else {
            // (a look costs issue slots that the softmax warps want; 2^22 looks with their pauses are half a second)
            if (++idle_turns >= 1 << 22) *abort_flag = 1u;
            if ((idle_turns & 255) == 0 && *abort_flag) break;
            __nanosleep(kPauseNs);
          }
        }
      }
      __syncwarp();
    }
  } else {
    // ---- softmax: group g takes every second tile of the stream; thread r of a group has head r ----
    more_registers<kRegsSoftmax>();
    const int g = warp >> 2, r = (warp & 3) * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t s_cols = lanes + (uint32_t)g * 128u, o_cols = lanes + 256u + (uint32_t)g * 128u;
    uint32_t it = 0, un = 0, wn = 0;
    bool ok = true;
    constexpr int kHalf = D / 2;  // columns of O a thread writes
    uint32_t unit = first;
    for (; unit < units; unit += step, ++un) {
      if (!(ok = __all_sync(kAll, mbar_wait(&sm.ifull[un % kInfo], (un / kInfo) & 1u, abort_flag)))) break;
      const int nt = sm.tiles[un % kInfo];
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.iempty[un % kInfo]);
      const Work w = work_of(p, unit);
      const bool busy = (warp & 3) * 32 < w.heads, mine = r < w.heads;
      T* const out = static_cast<T*>(p.out) + (int64_t)w.token * p.out_token + (int64_t)(w.head0 + r) * p.out_head + g * kHalf;
      float* const lse = p.lse == nullptr ? nullptr : p.lse + (int64_t)w.token * p.kv_heads * p.group + w.head0 + r;
      if (nt == 0 && ctas == 1) {
        if (mine) {
          const uint32_t zero[4] = {0u, 0u, 0u, 0u};
          for (int c = 0; c < kHalf; c += 8) store_row(out + c, zero, p.out_vec != 0);
          if (g == 0 && lse != nullptr) *lse = -INFINITY;
        }
        continue;
      }
      float ref = -INFINITY, sum = 0.f;
      for (int j = g ^ (int)(it & 1u); j < nt; j += 2) {
        const uint32_t n = it + (uint32_t)j;
        const int place = (int)(n % kMeta);
        ok = mbar_wait(&sm.mfull[place], (n / kMeta) & 1u, abort_flag) && mbar_wait(&sm.sdone[n % kKS], (n / kKS) & 1u, abort_flag);
        if (!(ok = __all_sync(kAll, ok))) break;
        tmem_fence_after();
        auto hand_over = [&](int half) {
          tmem_wait_st();
          tmem_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.pfull[g][half]);
        };
        if (busy) {
          const TileMeta& m = sm.meta[place];
          const float qmul = sm.qmul[wn & 3u][r];
          // A new reference: what was weighed with the old one - O up to the tile before, or with the first half of this one's keys
          // where that has been handed over, and the sum - is brought to it.
          auto refer = [&](float next, bool half) {
            const float f = next == ref ? 1.f : ex2(ref - next);
            sum = kFp8 ? brought(sum, ref, next) : sum * f;
            ref = next;
            if (half || j > 1) {
              uint64_t* const bar = half ? &sm.halfdone[g] : &sm.pvdone[(n - 2u) % kMeta];
              if (!__all_sync(kAll, mbar_wait(bar, half ? (n >> 1) & 1u : ((n - 2u) / kMeta) & 1u, abort_flag))) return;  // (the waits to come fail too)
              tmem_fence_after();
#pragma unroll 1
              for (int c = 0; c < D / 16; ++c) {
                uint32_t v[16];
                tmem_ld16(o_cols + 16u * c, v);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * f);
                tmem_st16(o_cols + 16u * c, v);
              }
            }
          };
          const bool whole = (m.flags & kWhole) != 0;
          Pair part[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
          auto parts = [&] {
            const float2 x = apart(add2(part[0], part[1]));
            part[0] = part[1] = pair(0.f, 0.f);
            return x.x + x.y;
          };
#pragma unroll 1
          for (int c = 0; c < kTileKeys / kChunk; ++c) {
            float s[kChunk];
            load_chunk(s_cols + (uint32_t)(kChunk * c), s);
            tmem_wait_ld();
            if constexpr (kFp8) {
#pragma unroll
              for (int i = 0; i < kChunk; i += 4) {
                const float4 x = *reinterpret_cast<const float4*>(m.ks + kChunk * c + i);
                const float2 a = apart(mul2(pair(s[i], s[i + 1]), pair(x.x, x.y))), b = apart(mul2(pair(s[i + 2], s[i + 3]), pair(x.z, x.w)));
                s[i] = a.x, s[i + 1] = a.y, s[i + 2] = b.x, s[i + 3] = b.y;
              }
            }
            if (!whole) {
#pragma unroll
              for (int b = 0; b < kChunk / 32; ++b) {
                const uint32_t there = m.live[kChunk / 32 * c + b];
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  if (!(there >> i & 1u)) s[32 * b + i] = -INFINITY;
              }
            }
            float top;
            if (!kFp8)
              top = top_of(s) * qmul;
            else if (m.flags & kEven)
              top = fmaf(top_of(s), qmul, m.vmost);
            else
              top = top_with(s, qmul, m.vlog + kChunk * c);
            if (__any_sync(kAll, top > ref + kLetStand)) {
              sum += parts();
              refer(top > ref + kLetStand ? top : ref, c > 0);
            }
            const float sub = ref == -INFINITY ? 0.f : ref;
            const Pair mul = pair(qmul, qmul), less = pair(-sub, -sub);
            uint32_t pk[kChunk / 2];
#pragma unroll
            for (int i = 0; i < kChunk; i += 4) {
              Pair w[2];
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float2 x = apart(fma2(pair(s[i + 2 * e], s[i + 2 * e + 1]), mul, less));
                w[e] = pair(ex2(x.x), ex2(x.y));
                part[e] = add2(part[e], w[e]);
              }
              if constexpr (kFp8) {
                const float4 x = *reinterpret_cast<const float4*>(m.vs + kChunk * c + i);
                w[0] = mul2(w[0], pair(x.x, x.y)), w[1] = mul2(w[1], pair(x.z, x.w));
              }
              const float2 a = apart(w[0]), b = apart(w[1]);
              pk[i / 2] = narrow2(a.x, a.y, M());
              pk[i / 2 + 1] = narrow2(b.x, b.y, M());
            }
            store_chunk(s_cols + (uint32_t)(kChunk / 2 * c), pk);  // (over scores that have been read)
            hand_over(c);
          }
          sum += parts();
        } else {
          hand_over(0);
          hand_over(1);
        }
      }
      if (!ok) break;
      // ---- this piece's end: both groups' products, maxima and sums ----
      const int nga = (nt + 1 - (int)(it & 1u)) / 2, ngb = nt - nga;  // tiles of group 0, of group 1
      float2 a = make_float2(-INFINITY, 0.f), b = a;
      if (nt > 0) {
        sm.ml[wn & 1u][g][r] = make_float2(ref + 0.f, sum);  // (+ 0: without it heads of 64 in 16 bits spill 36 bytes instead of 8, 173 us instead of 169)
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.mlbar);
        ok = mbar_wait(&sm.mlbar, wn & 1u, abort_flag);
        const uint32_t end = it + (uint32_t)nt - 1u;  // the last tile; the one before it is the other group's last
        ok = ok && mbar_wait(&sm.pvdone[end % kMeta], (end / kMeta) & 1u, abort_flag);
        if (nt > 1) ok = ok && mbar_wait(&sm.pvdone[(end - 1u) % kMeta], ((end - 1u) / kMeta) & 1u, abort_flag);
        if (!(ok = __all_sync(kAll, ok && *abort_flag == 0u))) break;  // (a wait may have run out in refer)
        tmem_fence_after();
        a = sm.ml[wn & 1u][0][r], b = sm.ml[wn & 1u][1][r];
      }
      const float top = fmaxf(a.x, b.x);
      const float fa = a.x == top ? 1.f : ex2(a.x - top), fb = b.x == top ? 1.f : ex2(b.x - top);
      const float l = kFp8 ? brought(a.y, a.x, top) + brought(b.y, b.x, top) : fa * a.y + fb * b.y;
      const float inv = ctas > 1 ? 1.f : l == 0.f ? 0.f : 1.f / l;
      float* const stage_row = reinterpret_cast<float*>(base) + (size_t)r * (D + 4) + g * kHalf;  // (several CTAs: over the q and k tiles)
      uint32_t packed[kHalf / 2];  // (the pieces of work to come may have O as soon as it has been read)
      if (busy) {
#pragma unroll
        for (int c = 0; c < kHalf; c += 32) {
          float y[32];
          const uint32_t col = lanes + 256u + (uint32_t)(g * kHalf + c);
#pragma unroll
          for (int i = 0; i < 32; ++i) y[i] = 0.f;
#pragma unroll 1
          for (int i = 0; i < 2; ++i) {
            if ((i == 0 ? nga : ngb) > 0) {
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
          } else {
#pragma unroll
            for (int i = 0; i < 32; i += 2) packed[(c + i) / 2] = narrow2(y[i], y[i + 1], T());
          }
        }
      }
      tmem_fence_before();
      __syncwarp();
      if (nt > 0 && lane == 0) mbar_arrive(&sm.oempty);
      if (ctas == 1 && mine) store_row(out, packed, p.out_vec != 0);
      if (g == 0) {
        if (ctas > 1)
          sm.ml[1][0][r] = make_float2(top, l);  // (one piece of work a CTA: the other half is not in use)
        else if (mine && lse != nullptr)
          *lse = l == 0.f ? -INFINITY : top * 0.693147180559945309f + logf(l);
      }
      it += (uint32_t)nt;
      wn += nt > 0 ? 1u : 0u;
    }
    if (ctas == 1 && unit < units) leave_nan<T, D>(p, unit, units, step, r, g);  // (of several CTAs: below)
  }
  __syncwarp();
  __syncthreads();
  if (warp < kSoftmaxWarps)
    fewer_registers<kRegsLaunch>();
  else
    more_registers<kRegsLaunch>();
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
    if (ctas > 1 && tid < kHeadsW) sm.ml[1][0][tid] = make_float2(-INFINITY, __int_as_float(0x7fffffff));  // (the joined rows become NaN)
  }
  tmem_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  if (ctas > 1) {
    cluster.sync();
    const Work w = work_of(p, first);
    constexpr int kPer = D / 32;  // channels a lane
    const uint32_t ml_at = smem_u32(&sm.ml[1][0][0]), o_at = smem_u32(base) + (uint32_t)(lane * kPer * 4);
    for (int h = rank + ctas * warp; h < w.heads; h += ctas * (kWideThreads / 32)) {
      // (every CTA's part is asked for before any is used)
      float2 ml[kAttendMaxCluster];
      float o[kAttendMaxCluster][kPer];
#pragma unroll
      for (int c = 0; c < kAttendMaxCluster; ++c) {
        ml[c] = make_float2(-INFINITY, 0.f);
        if (c < ctas) {
          ml[c] = lds_cluster2(shared_of(ml_at + (uint32_t)h * 8u, c));
          const uint32_t from = shared_of(o_at + (uint32_t)(h * (D + 4) * 4), c);
          if constexpr (kPer == 4) {
            const float4 v = lds_cluster4(from);
            o[c][0] = v.x, o[c][1] = v.y, o[c][2] = v.z, o[c][3] = v.w;
          } else {
            const float2 v = lds_cluster2(from);
            o[c][0] = v.x, o[c][1] = v.y;
          }
        }
      }
      float top = -INFINITY;
#pragma unroll
      for (int c = 0; c < kAttendMaxCluster; ++c) top = fmaxf(top, ml[c].x);
      float l = 0.f, acc[kPer];
#pragma unroll
      for (int e = 0; e < kPer; ++e) acc[e] = 0.f;
#pragma unroll
      for (int c = 0; c < kAttendMaxCluster; ++c) {
        if (c < ctas) {
          const float f = ml[c].x == top ? 1.f : ex2(ml[c].x - top);
          l += kFp8 ? brought(ml[c].y, ml[c].x, top) : f * ml[c].y;
#pragma unroll
          for (int e = 0; e < kPer; ++e) acc[e] += f * o[c][e];
        }
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
      cudaFuncSetAttribute(attend_wide_kernel<T, kFp8, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)wide_smem_bytes<kFp8, D>());
  return e == cudaSuccess ? 0 : cuda_fail(e);
}

template <typename T, bool kFp8, int D>
cudaError_t launch_wide(const AttendParams& p, int ctas, int64_t units, int sms, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  const int64_t grid = ctas > 1 ? units * ctas : units < sms ? units : sms;
  cfg.gridDim = dim3((unsigned)grid, 1, 1);
  cfg.blockDim = dim3(kWideThreads, 1, 1);
  cfg.dynamicSmemBytes = wide_smem_bytes<kFp8, D>();
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

int attend_wide_setup(int& eights) {
  int r = setup_wide<__nv_bfloat16, false, 64>();
  if (!r) r = setup_wide<__nv_bfloat16, false, 128>();
  if (!r) r = setup_wide<__nv_bfloat16, true, 64>();
  if (!r) r = setup_wide<__nv_bfloat16, true, 128>();
  if (!r) r = setup_wide<__half, false, 64>();
  if (!r) r = setup_wide<__half, false, 128>();
  if (!r) r = setup_wide<__half, true, 64>();
  if (!r) r = setup_wide<__half, true, 128>();
  if (!r) r = clusters_of(eights, attend_wide_kernel<__nv_bfloat16, false, 128>, kWideThreads, wide_smem_bytes<false, 128>());
  return r;
}

cudaError_t attend_wide(const AttendParams& p, bool bf16, bool fp8, int D, int ctas, int64_t units, int sms, cudaStream_t stream) {
  return bf16 ? launch_wide<__nv_bfloat16>(p, fp8, D, ctas, units, sms, stream) : launch_wide<__half>(p, fp8, D, ctas, units, sms, stream);
}

}  // namespace fftopk
