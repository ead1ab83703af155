// Attention of every sequence's newest token over its whole context, which lies in pages of a cache:
//   o[b, h] = sum_j p_j v[slot_j, h / g],  p_j = exp(scale * q[b, h] . k[slot_j, h / g] - lse),  slot_j = table[b, j / page] * page + j % page
// g query heads to a key head, j below the sequence's length. Where asked for, what every cached row has been given so far is brought up
// to date: weight_out[b, h / g, j] = weight[b, h / g, j] + sum of p_j over the key head's query heads. (The reference ends with indices.)
//
// What bounds it is reading the cache: a row of k or v is used by the g heads of its key head alone, g flop a byte in 16 bits, 2 g in e4m3 (64
// query heads on 8 key heads of 128: 64 sequences of up to 8,192 in bf16 243 us = 6.5 TB/s, of up to 16,384 in e4m3 250 = 6.5 in short runs, 271 to 285 =
// 5.7 to 6.0 after a second of such calls, when the device is at its power limit and instructions bound it; one of 131,072 in bf16 91 = 5.9, of which 5 are the
// join; one of 100: 5.1).
//
// Work split: the context, 16 or 32 keys a block, of all sequences, sequence after sequence, is one line of blocks. It is cut into equal
// runs, whatever the lengths; a CTA takes one run for one key head (8 or 16 of its query heads). The CTAs of neighbouring numbers take the same
// run for different key heads, so that what lies side by side in the cache - the heads of a row, their scales - is read at about the
// same time. What a run has of a sequence is a segment: each of four warps takes a quarter of it with running maxima and sums (one pass),
// then they are joined through the stages of their rings that are free at that moment (every fourth block to a warp instead: e4m3 299 us, the
// pages' entries are read more often). A run that holds all of a sequence writes the result, else a part, which paged_finish_kernel joins.
// Lengths are read on the device only; no CTA waits for another launch's. Where tables are short, a cluster takes a sequence and joins it through distributed shared
// memory (64 sequences of up to 300: 15 us, in equal runs 23). More than 16 query heads to a key head read its rows again for every 16 (64 on one key head, 32,768
// positions: 2.7 times the floor), and a segment costs some 4 us whatever its length (1,024 sequences of 16: 87 us).
//
// A warp has a ring of blocks in shared memory that cp.async fills ahead of it. Keys are the rows of the MMA and query heads its
// columns, 8 at a time: groups of up to 8 heads need half the products and accumulators they would need as rows.
//   k.q: the contraction's order is free, so a lane's 16-byte piece of a key row serves as A fragments of consecutive steps, and q is
//        loaded in the same order.
//   v.p: A = v transposed, by ldmatrix.trans; scores become weights where they lie and are turned by movmatrix.
//   e4m3: codes are widened to fp16, which holds each of them exactly; a matrix element of ldmatrix is then a pair of channels, whose
//        bytes are sorted by key first (the two channels are the rows i and i + 8 of the product). Queries are brought to magnitudes
//        below 2 by a power of two per head (what fp16 loses of a bf16 query lies 2^-25 below the head's largest). A row's k scale multiplies its score, its v
//        scale its weight; the running reference is of weight * |v scale|, so that no row with hardly any weight sets it.
// Roundings: weights of the second product to the cache's type (e4m3: to fp16, their v scale in them), off by half a step; everything
// else is held in 32 bits.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include <string.h>

#include "../../include/fftopk.h"
#include "fftopk_attend.cuh"
#include "fftopk_extent.h"
#include "fftopk_host.h"
#include "fftopk_internal.h"
#include "fftopk_rows.cuh"
#include "fftopk_tcgen05.cuh"

namespace fftopk {
namespace {

namespace cg = cooperative_groups;

constexpr int kMaxApart = 8;  // CTAs of a cluster that takes a sequence
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kWeighKeys = 128;  // positions that a warp has on their way at a time where it brings weights up to date
// positions of a run: below that, parts to join cost more than the blocks (one sequence of 1,000, 8 key heads: 8.8 us, with 256 positions 10.7, with 512
// 15.4; of 4,096: 9.6, 10.3 and 12.3, with 64 11.3)
constexpr int kMinKeys = 128;
// Keys of a block, 16 to a product: 8 KB of k and v (4 KB of e4m3 heads of 64), so that what goes with a block is done for enough of them (64 sequences of up to 8,192, 8 key heads, with
// 16 keys and with 32: 16 bits, heads of 64 137 us and 128; e4m3, 16 query heads to a key head 187 and 152; up to 16,384, heads of 64 174 and 138)
template <bool kFp8, int D>
constexpr int block_keys() {
  return D * (kFp8 ? 1 : 2) == 256 ? 16 : 32;
}

struct PagedParams {
  fftopk_paged a;
  int32_t group, head_blocks, units, runs, bound, weigh;
  int32_t key_shift;  // of a block's keys
  int32_t apart;      // CTAs of a cluster that takes a sequence, whatever its length: no parts; 0: equal runs
  FastDiv page;
  float scale_log2;
  int32_t weigh_here;  // the weights are brought up to date by the CTAs that have made the scores: nothing of a sequence is elsewhere
  int32_t stream;   // the rows are more than L2 holds
  int32_t out_vec;  // rows of out start on 8 bytes
  int64_t line;     // positions of a unit of the score workspace
  float* lse2;      // [seqs, q heads] log2 of the sum of exponentials, of sequences that lie in one run
  float2* ml;       // [runs * units * 2][heads of a unit] maximum (log2) and sum of a part
  float* o;         // [runs * units * 2][heads of a unit][D]
  float* scores;    // [seqs][units][line][heads of a unit], log2
  uint32_t* status;
  // paged_finish_kernel: CTAs that join, how many pairs of a sequence and a query head each of their warps takes (0: a CTA takes one), warps that weigh
  int32_t join_ctas, join_each, weigh_runs;
};

// Keys of sequence b: its length, as far as its pages reach
__device__ __forceinline__ int32_t keys_of(const PagedParams& p, int64_t b) { return min(max(p.a.lengths[b], 0), p.bound); }
__device__ __forceinline__ int64_t blocks_of(const PagedParams& p, int32_t n) { return ((int64_t)n + (1 << p.key_shift) - 1) >> p.key_shift; }

// Runs the line of `total` blocks is cut into, and where one begins: the first total % runs have a block more.
struct Runs {
  int64_t total, each, rest;
  int32_t runs;
  __device__ __forceinline__ Runs(int64_t t, int32_t most, int32_t least) : total(t) {
    runs = (int32_t)max((int64_t)1, min((int64_t)most, quotient(t, least)));
    each = quotient(t, runs);
    rest = t - each * runs;
  }
  static __device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {  // (64 bits only where they are needed: ten times as long)
    return ((a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
  }
  __device__ __forceinline__ int64_t begin(int64_t run) const { return run * each + min(run, rest); }
  __device__ __forceinline__ int64_t of(int64_t block) const {
    const int64_t wide = rest * (each + 1);  // (each = 0: every block is in front of `wide`)
    return block < wide ? quotient(block, each + 1) : rest + quotient(block - wide, each);
  }
};

__device__ __forceinline__ int64_t warp_sum(int64_t x) {
#pragma unroll
  for (int i = 16; i > 0; i >>= 1) x += __shfl_xor_sync(kAll, x, i);
  return x;
}
__device__ __forceinline__ int64_t warp_scan(int64_t x, int lane) {
#pragma unroll
  for (int i = 1; i < 32; i <<= 1) {
    const int64_t y = __shfl_up_sync(kAll, x, i);
    if (lane >= i) x += y;
  }
  return x;
}
// blocks of the sequences in front of `upto`
__device__ __forceinline__ int64_t blocks_before(const PagedParams& p, int64_t upto, int lane) {
  int64_t total = 0;
  for (int64_t b = lane; b < upto; b += 32) total += blocks_of(p, keys_of(p, b));
  return warp_sum(total);
}

// What a run has of a sequence: blocks s0 .. s1 - 1 of its `blocks`
struct Segment {
  int64_t b;
  int32_t n, blocks, s0, s1;
};
// The segment that begins at block g of the line (g < total), of at most `left` blocks
__device__ __forceinline__ Segment segment_at(const PagedParams& p, int64_t g, int64_t left, int lane) {
  Segment c;
  int64_t before = 0;
  for (int64_t first = 0;; first += 32) {
    const int32_t n = first + lane < p.a.seqs ? keys_of(p, first + lane) : 0;
    const int64_t upto = before + warp_scan(blocks_of(p, n), lane);
    const unsigned beyond = __ballot_sync(kAll, upto > g);
    if (beyond != 0u || first + 32 >= p.a.seqs) {
      const int l = beyond != 0u ? __ffs((int)beyond) - 1 : 31;
      c.b = first + l;
      c.n = __shfl_sync(kAll, n, l);
      c.blocks = (int32_t)blocks_of(p, c.n);
      c.s0 = (int32_t)(g - (__shfl_sync(kAll, upto, l) - c.blocks));
      c.s1 = (int32_t)min((int64_t)c.blocks, c.s0 + left);
      return c;
    }
    before = __shfl_sync(kAll, upto, 31);
  }
}
// The one behind it, of at most `left` > 0 blocks; false: the line ends
__device__ __forceinline__ bool next_segment(const PagedParams& p, Segment& c, int64_t left) {
  for (++c.b; c.b < p.a.seqs; ++c.b) {
    c.n = keys_of(p, c.b);
    if (c.n > 0) {
      c.blocks = (int32_t)blocks_of(p, c.n);
      c.s0 = 0;
      c.s1 = (int32_t)min((int64_t)c.blocks, left);
      return true;
    }
  }
  return false;
}
// A warp's quarter of it
__device__ __forceinline__ void quarter(const Segment& c, int warp, int32_t& at, int32_t& end) {
  const int32_t q = (c.s1 - c.s0) / kWarps, r = (c.s1 - c.s0) % kWarps;
  at = c.s0 + warp * q + min(warp, r);
  end = at + q + (warp < r ? 1 : 0);
}

__device__ __forceinline__ uint32_t turned8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// four e4m3 codes as fp16: the lower two, the upper two
__device__ __forceinline__ void widen4(uint32_t& lo, uint32_t& hi, uint32_t codes) {
  asm("{\n .reg .b16 a, b;\n mov.b32 {a, b}, %2;\n cvt.rn.f16x2.e4m3x2 %0, a;\n cvt.rn.f16x2.e4m3x2 %1, b;\n}" : "=r"(lo), "=r"(hi) : "r"(codes));
}
// 16 bytes of a row; rows that are more than L2 holds leave it before the scales - whose 32 bytes belong to several key heads - and the parts do (64 sequences of up to 16,384 in
// e4m3: 250 us, 261 without the hint; one of 131,072 in bf16: 91 and 93)
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, uint64_t once) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "l"(once) : "memory");
}
__device__ __forceinline__ void copy16_or_zero(uint32_t dst, const void* src, bool there, uint64_t once) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint.L2::128B [%0], [%1], 16, %2, %3;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0), "l"(once) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
// row r of a cache: the product of two 32-bit numbers, added in 64 bits (slots are below 2^31, slot strides below 2^32 bytes)
__device__ __forceinline__ const char* row_at(const char* base, int r, uint32_t step) { return base + (uint64_t)(uint32_t)r * step; }
__device__ __forceinline__ float lds4(uint32_t addr) {
  float r;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(r) : "r"(addr) : "memory");
  return r;
}
// over the lanes that hold the same heads
__device__ __forceinline__ float keys_max(float x) {
  x = fmaxf(x, __shfl_xor_sync(kAll, x, 4));
  x = fmaxf(x, __shfl_xor_sync(kAll, x, 8));
  return fmaxf(x, __shfl_xor_sync(kAll, x, 16));
}
__device__ __forceinline__ float keys_sum(float x) {
  x += __shfl_xor_sync(kAll, x, 4);
  x += __shfl_xor_sync(kAll, x, 8);
  return x + __shfl_xor_sync(kAll, x, 16);
}

// A warp's ring: the k rows of a block, its v rows, stage after stage; e4m3: then the stages' scales. Rows are not padded; 16-byte pieces
// change places within a row so that the lanes that are served together touch all banks: k, where a quad reads four neighbouring pieces of each of two
// rows; v, where eight rows give the same piece.
template <bool kFp8, int D>
struct PagedRing {
  static constexpr int kKeys = block_keys<kFp8, D>();
  static constexpr int kRowBytes = D * (kFp8 ? 1 : 2);
  static constexpr int kV = kKeys * kRowBytes, kStage = 2 * kV;
  static constexpr int kStages = 3;
  static constexpr int kScales = kStages * kStage, kScaleStage = kFp8 ? 2 * kKeys * 4 : 0;
  static constexpr int kBytes = kScales + kStages * kScaleStage;  // of a warp
  // (rows of 64 bytes: two of them touch all banks already)
  static __device__ __forceinline__ uint32_t k_piece(int row, int piece) { return (uint32_t)(kRowBytes == 64 ? piece : piece ^ (row & 1) << 2); }
  static __device__ __forceinline__ uint32_t v_piece(int row, int piece) { return (uint32_t)(kRowBytes == 64 ? piece ^ (row >> 1 & 3) : piece ^ (row & 7)); }
};
template <bool kFp8, int D>
constexpr size_t paged_smem() {
  return (size_t)kWarps * PagedRing<kFp8, D>::kBytes;
}
// CTAs per SM: as many as shared memory (228 KB, 1 KB of each CTA is the system's) and the registers of the accumulators allow
template <bool kFp8, int D, int kNT>
constexpr int paged_ctas() {
  constexpr int fit = (int)(228 * 1024 / (paged_smem<kFp8, D>() + 1024)), regs = kNT == 2 ? (D == 64 ? 3 : 2) : 4;
  return fit < regs ? fit : regs;
}

// T: type of q and out, and of the cache where kFp8 is false; kNT: eights of query heads; kWhole: every block lies on one page
template <typename T, bool kFp8, int D, int kNT, bool kWhole>
__global__ void __launch_bounds__(kThreads, paged_ctas<kFp8, D, kNT>()) paged_kernel(const __grid_constant__ PagedParams p) {
  using M = typename std::conditional<kFp8, __half, T>::type;  // the MMAs' type
  using G = PagedRing<kFp8, D>;
  constexpr int kCE = kFp8 ? 16 : 8;         // elements of a 16-byte piece
  constexpr int kPieces = D / (4 * kCE);     // pieces of a key row per lane (a quad reads a row)
  constexpr int kKeys = G::kKeys, kR = kKeys / 16;  // a block's keys, and products
  constexpr int kStages = G::kStages;
  constexpr int kNH = 8 * kNT;
  constexpr int kTiles = D / 16;             // of the output: rows of the MMA are channels
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  // (only where a kernel of this call follows, which waits: another one's inputs may be this one's results)
  if (p.join_ctas > 0 || (p.weigh && !p.weigh_here)) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  __shared__ float2 ml_of[kWarps][kNH];
  __shared__ uint32_t free_of[kWarps];  // the warps' free stages
  __shared__ float2 joined_ml[kNH];     // of a CTA: maximum and sum
  __shared__ float log_sum[kNH];        // of a sequence
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, qd = lane & 3;
  const uint32_t ctas = (uint32_t)max(p.apart, 1), run_unit = blockIdx.x / ctas, rank = blockIdx.x - run_unit * ctas;
  const uint32_t run = run_unit / (uint32_t)p.units;
  const int unit = (int)(run_unit - run * (uint32_t)p.units);
  const int kvh = unit / p.head_blocks, hb = unit - kvh * p.head_blocks;
  const int heads = min(kNH, p.group - hb * kNH);
  const int head0 = kvh * p.group + hb * kNH;

  // a sequence without rows; and one that reaches beyond its pages is told of
  auto empty = [&](int64_t b) {
    const int32_t n = p.a.lengths[b];
    if (n > p.bound && unit == 0 && lane == 0 && p.status) atomicOr(p.status, (uint32_t)FFTOPK_ST_BAD_INDEX);
    return min(n, p.bound) <= 0;
  };
  auto put_zeros = [&](int64_t b) {
    for (int h = 0; h < heads; ++h) {
      T* out = static_cast<T*>(p.a.out) + b * p.a.out_seq + (int64_t)(head0 + h) * p.a.out_head;
      for (int d = lane; d < D; d += 32) out[d] = T(0.f);
      if (lane == 0 && p.a.lse != nullptr) p.a.lse[b * p.a.q_heads + head0 + h] = -INFINITY;
    }
  };
  Segment here;
  int64_t left;  // blocks of the run that are not behind the segment at hand
  if (p.apart) {  // (the run is the sequence of its number, a CTA's segment its share of the cluster's)
    if (empty(run)) {
      if (warp == 0 && rank == 0) put_zeros(run);
      return;  // (the whole cluster)
    }
    here.b = run, here.n = keys_of(p, run), here.blocks = (int32_t)blocks_of(p, here.n);
    here.s0 = (int32_t)((int64_t)here.blocks * rank / ctas), here.s1 = (int32_t)((int64_t)here.blocks * (rank + 1) / ctas);
    left = here.s1 - here.s0;  // (none, where there are fewer blocks than CTAs)
  } else {
    for (int64_t b = run + (int64_t)p.runs * warp; b < p.a.seqs; b += (int64_t)p.runs * kWarps)
      if (empty(b)) put_zeros(b);
    const Runs line(blocks_before(p, p.a.seqs, lane), p.runs, kMinKeys / kKeys);
    if ((int64_t)run >= line.runs || line.total == 0) return;  // (the whole CTA)
    left = line.begin((int64_t)run + 1) - line.begin(run);
    if (left <= 0) return;
    here = segment_at(p, line.begin(run), left, lane);
  }

  constexpr int kLanesRow = G::kRowBytes / 16, kRowsOnce = 32 / kLanesRow, kTurns = kKeys / kRowsOnce;
  constexpr int kES = kFp8 ? 1 : 2;
  constexpr unsigned kFull = kKeys == 32 ? kAll : (1u << kKeys) - 1u;  // all of a block's keys
  const int piece = lane % kLanesRow, sub = lane / kLanesRow;
  const char* const kbase = static_cast<const char*>(p.a.k) + (int64_t)kvh * p.a.k_head * kES + piece * 16;
  const char* const vbase = static_cast<const char*>(p.a.v) + (int64_t)kvh * p.a.v_head * kES + piece * 16;
  static_assert(!kFp8 || kKeys == 32, "e4m3: a lane has a key of the block, and asks for both of its scales");
  const float *sbase[2] = {};
  int64_t sstep[2] = {};
  if constexpr (kFp8) {
    sbase[0] = p.a.k_scale + (int64_t)kvh * p.a.ks_head, sstep[0] = p.a.ks_slot;
    sbase[1] = p.a.v_scale + (int64_t)kvh * p.a.vs_head, sstep[1] = p.a.vs_slot;
  }
  const uint32_t kstep = (uint32_t)(p.a.k_slot * kES), vstep = (uint32_t)(p.a.v_slot * kES);
  const uint32_t ring = smem_u32(smem_raw) + (uint32_t)warp * G::kBytes;

  uint64_t once;
  if (p.stream)
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(once));
  else
    asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(once));
  Segment ahead = here;
  int64_t left_ahead = left;
  int32_t at, end, ask_at, ask_end;  // the warp's blocks of the segment at hand, and of the one it asks for
  quarter(here, warp, at, end);
  ask_at = at, ask_end = end;
  bool more = true;  // there is a block to ask for
  const int32_t* table = p.a.page_table + ahead.b * p.a.table_row;
  // of the block that is asked for next: the page of the lane's key and its place there (lanes 16 to 31: the same ones again); kWhole: of
  // the block's first key
  int32_t page = -1;
  uint32_t in_page = 0;
  int rows = 0;
  auto look = [&]() {
    if (!more) {
      page = -1;
      return;
    }
    rows = min(kKeys, ahead.n - ask_at * kKeys);
    const uint32_t j = (uint32_t)ask_at * kKeys + (kWhole ? 0u : (uint32_t)(lane & (kKeys - 1)));
    if (!kWhole || in_page == 0) {  // (kWhole: a page's blocks follow each other, and the table is read once a page)
      page = -1;
      if (j < (uint32_t)ahead.n) {
        const uint32_t n = p.page.div(j);
        in_page = j - n * p.page.d;
        page = table[n];
      }
    }
  };
  // on to the first segment with blocks of the warp
  auto find = [&]() {
    while (ask_at == ask_end) {
      left_ahead -= ahead.s1 - ahead.s0;
      if (left_ahead <= 0 || !next_segment(p, ahead, left_ahead)) {
        more = false;
        return;
      }
      quarter(ahead, warp, ask_at, ask_end);
      table = p.a.page_table + ahead.b * p.a.table_row;
      in_page = 0;
    }
  };
  // the block behind
  auto step = [&]() {
    if (!more) return;
    in_page += kKeys;
    if (in_page >= p.page.d) in_page = 0;
    ++ask_at;
    find();
  };
  // asks for the rows and scales of the block looked up; which of them are there
  auto ask = [&](int stage) {
    const uint32_t data = ring + (uint32_t)(stage * G::kStage);
    const uint32_t scales = ring + (uint32_t)(G::kScales + stage * G::kScaleStage + lane * 4);
    unsigned live = 0u;
    if constexpr (kWhole) {
      if (page >= 0) {
        const int64_t slot = (int64_t)page * p.page.d + in_page;
        const int there = slot < p.a.slots ? (int)min((int64_t)rows, p.a.slots - slot) : 0;
        if (there < rows && p.status) atomicOr(p.status, (uint32_t)FFTOPK_ST_BAD_INDEX);
        live = there == 32 ? kAll : (1u << there) - 1u;
        if (there == kKeys) {
          const char* const k = row_at(kbase, (int)slot + sub, kstep);
          const char* const v = row_at(vbase, (int)slot + sub, vstep);
#pragma unroll
          for (int i = 0; i < kTurns; ++i) {
            const int at = i * kRowsOnce + sub;
            copy16(data + at * G::kRowBytes + G::k_piece(at, piece) * 16u, row_at(k, i * kRowsOnce, kstep), once);
            copy16(data + G::kV + at * G::kRowBytes + G::v_piece(at, piece) * 16u, row_at(v, i * kRowsOnce, vstep), once);
          }
          if constexpr (kFp8) {
#pragma unroll
            for (int i = 0; i < 2; ++i) copy4(scales + i * 128u, sbase[i] + (uint64_t)(uint32_t)((int)slot + lane) * sstep[i]);
          }
        } else if (there > 0) {
#pragma unroll
          for (int i = 0; i < kTurns; ++i) {
            const int at = i * kRowsOnce + sub, r = (int)slot + min(at, there - 1);
            copy16_or_zero(data + at * G::kRowBytes + G::k_piece(at, piece) * 16u, row_at(kbase, r, kstep), at < there, once);
            copy16_or_zero(data + G::kV + at * G::kRowBytes + G::v_piece(at, piece) * 16u, row_at(vbase, r, vstep), at < there, once);
          }
          if constexpr (kFp8) {
#pragma unroll
            for (int i = 0; i < 2; ++i) copy_or_zero<4>(scales + i * 128u, sbase[i] + (uint64_t)(uint32_t)((int)slot + min(lane, there - 1)) * sstep[i], lane < there);
          }
        }
      }
    } else {
      const int64_t slot = (int64_t)page * p.page.d + in_page;
      bool ok = page >= 0;
      if (ok && slot >= p.a.slots) {
        ok = false;
        if (p.status) atomicOr(p.status, (uint32_t)FFTOPK_ST_BAD_INDEX);
      }
      live = __ballot_sync(kAll, ok) & kFull;
      if (live != 0u) {
        const int row = ok ? (int)slot : -1;
#pragma unroll
        for (int i = 0; i < kTurns; ++i) {
          const int at = i * kRowsOnce + sub;
          const int r = __shfl_sync(kAll, row, at);
          copy16_or_zero(data + at * G::kRowBytes + G::k_piece(at, piece) * 16u, row_at(kbase, max(r, 0), kstep), r >= 0, once);
          copy16_or_zero(data + G::kV + at * G::kRowBytes + G::v_piece(at, piece) * 16u, row_at(vbase, max(r, 0), vstep), r >= 0, once);
        }
        if constexpr (kFp8) {
#pragma unroll
          for (int i = 0; i < 2; ++i) copy_or_zero<4>(scales + i * 128u, sbase[i] + (uint64_t)(uint32_t)max(row, 0) * sstep[i], ok);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    return live;
  };
  unsigned live_of[kStages];
  find();
  look();  // (in_page is 0: the table is read)
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) {
    live_of[s] = ask(s);
    step();
    look();
  }
  int at_stage = 0, ask_stage = kStages - 1;

  // of the segment at hand
  uint32_t qb[kNT][D / 16][2];
  float qmul[kNT][2];  // what the scores of the lane's heads are to be multiplied with
  float o[kNT][kTiles][4];
  // what weights are taken against (log2): the largest score; fp8: the largest score + log2 |v scale|, by the scale's exponent
  float mx[kNT][2], sum[kNT][2];
  int which = 0;  // of two parts that a run may leave: 0 its first segment's, 1 its last one's
  for (;;) {
    {
      const T* q0 = static_cast<const T*>(p.a.q) + here.b * p.a.q_seq + (int64_t)head0 * p.a.q_head;
#pragma unroll
      for (int t = 0; t < kNT; ++t) {
        const bool have = 8 * t + g < heads;
        const T* q = q0 + (int64_t)(8 * t + g) * p.a.q_head;
        float down = 1.f, up = p.scale_log2;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
#pragma unroll
          for (int e = 0; e < kCE / 8; ++e) {
            const uint4 w = have ? *reinterpret_cast<const uint4*>(q + i * 4 * kCE + qd * kCE + 8 * e) : make_uint4(0u, 0u, 0u, 0u);
            const int m = i * (kCE / 4) + 2 * e;
            qb[t][m][0] = w.x, qb[t][m][1] = w.y, qb[t][m + 1][0] = w.z, qb[t][m + 1][1] = w.w;
          }
        }
        if constexpr (kFp8 && !std::is_same<T, __half>::value) {
          float amax = 0.f;
#pragma unroll
          for (int m = 0; m < D / 16; ++m) {
            const float2 a = widen2(qb[t][m][0], T()), b = widen2(qb[t][m][1], T());
            amax = fmaxf(amax, fmaxf(fmaxf(fabsf(a.x), fabsf(a.y)), fmaxf(fabsf(b.x), fabsf(b.y))));
          }
          amax = fmaxf(amax, __shfl_xor_sync(kAll, amax, 1));
          amax = fmaxf(amax, __shfl_xor_sync(kAll, amax, 2));
          const uint32_t e = __float_as_uint(amax) >> 23;  // amax in [2^(e-127), 2^(e-126)); 255: an infinity
          const uint32_t ee = e == 255u ? 127u : max(1u, min(e, 253u));
          down = __uint_as_float((254u - ee) << 23);
          up *= __uint_as_float(ee << 23);
#pragma unroll
          for (int m = 0; m < D / 16; ++m) {
            const float2 a = widen2(qb[t][m][0], T()), b = widen2(qb[t][m][1], T());
            qb[t][m][0] = narrow2(a.x * down, a.y * down, __half());
            qb[t][m][1] = narrow2(b.x * down, b.y * down, __half());
          }
        }
        qmul[t][0] = __shfl_sync(kAll, up, 8 * qd);
        qmul[t][1] = __shfl_sync(kAll, up, 8 * qd + 4);
        mx[t][0] = mx[t][1] = -INFINITY;
        sum[t][0] = sum[t][1] = 0.f;
#pragma unroll
        for (int i = 0; i < kTiles; ++i) o[t][i][0] = o[t][i][1] = o[t][i][2] = o[t][i][3] = 0.f;
      }
    }
    for (; at < end; ++at) {
    live_of[kStages - 1] = ask(ask_stage);
    step();
    look();
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
    __syncwarp();
    const unsigned live = live_of[0];
    const uint32_t stage = ring + (uint32_t)(at_stage * G::kStage);
    const uint32_t scales = ring + (uint32_t)(G::kScales + at_stage * G::kScaleStage);
    at_stage = at_stage + 1 == kStages ? 0 : at_stage + 1;
    ask_stage = ask_stage + 1 == kStages ? 0 : ask_stage + 1;
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) live_of[s] = live_of[s + 1];

    if (live != 0u || p.weigh) {
      float sc[kNT][kR][4];  // of every 16 keys: g (0, 1) and g + 8 (2, 3), heads 2 qd and 2 qd + 1
#pragma unroll
      for (int t = 0; t < kNT; ++t)
#pragma unroll
        for (int r = 0; r < kR; ++r) sc[t][r][0] = sc[t][r][1] = sc[t][r][2] = sc[t][r][3] = 0.f;
      float ks[kR][2], vs[kR][2], vl[kR][2];
#pragma unroll
      for (int r = 0; r < kR; ++r) ks[r][0] = ks[r][1] = vs[r][0] = vs[r][1] = 1.f, vl[r][0] = vl[r][1] = 0.f;
      if (live != 0u) {
#pragma unroll
        for (int r = 0; r < kR; ++r) {
          const uint32_t from_row = stage + (uint32_t)((16 * r + g) * G::kRowBytes);
#pragma unroll
          for (int i = 0; i < kPieces; ++i) {
            const uint32_t from = from_row + G::k_piece(g, 4 * i + qd) * 16u;
            const uint4 x = lds16(from), y = lds16(from + 8u * G::kRowBytes);
            const uint32_t a[4] = {x.x, x.y, x.z, x.w}, b[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int u = 0; u < kCE / 4; ++u) {
              uint32_t f[4];
              if constexpr (kFp8) {
                widen4(f[0], f[2], a[u]);
                widen4(f[1], f[3], b[u]);
              } else {
                f[0] = a[2 * u], f[2] = a[2 * u + 1], f[1] = b[2 * u], f[3] = b[2 * u + 1];
              }
#pragma unroll
              for (int t = 0; t < kNT; ++t) mma16816(sc[t][r], f, qb[t][i * (kCE / 4) + u][0], qb[t][i * (kCE / 4) + u][1], M());
            }
          }
          if constexpr (kFp8) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              ks[r][e] = lds4(scales + (uint32_t)((16 * r + g + 8 * e) * 4));
              vs[r][e] = lds4(scales + (uint32_t)((kKeys + 16 * r + g + 8 * e) * 4));
              vl[r][e] = (float)scale_exponent(vs[r][e]);
            }
          }
        }
      }
#pragma unroll
      for (int t = 0; t < kNT; ++t) {
#pragma unroll
        for (int r = 0; r < kR; ++r) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            sc[t][r][e] *= qmul[t][e & 1];
            if constexpr (kFp8) sc[t][r][e] *= ks[r][e >> 1];
          }
        }
      }
      if (live != kFull) {
#pragma unroll
        for (int r = 0; r < kR; ++r) {
          const bool lo = (live >> (16 * r + g)) & 1u, hi = (live >> (16 * r + g + 8)) & 1u;
#pragma unroll
          for (int t = 0; t < kNT; ++t) {
            sc[t][r][0] = lo ? sc[t][r][0] : -INFINITY, sc[t][r][1] = lo ? sc[t][r][1] : -INFINITY;
            sc[t][r][2] = hi ? sc[t][r][2] : -INFINITY, sc[t][r][3] = hi ? sc[t][r][3] : -INFINITY;
          }
        }
      }
      // (a reference is let stand until a score exceeds it by 2^8: fp16 weights and 32-bit sums have the room)
      float top[kNT][2];
      bool over = false;
#pragma unroll
      for (int t = 0; t < kNT; ++t) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          top[t][e] = fmaxf(sc[t][0][e] + vl[0][0], sc[t][0][2 + e] + vl[0][1]);
#pragma unroll
          for (int r = 1; r < kR; ++r) top[t][e] = fmaxf(top[t][e], fmaxf(sc[t][r][e] + vl[r][0], sc[t][r][2 + e] + vl[r][1]));
          over = over || top[t][e] > mx[t][e] + 8.f;
        }
      }
      if (p.weigh) {
        float* to = p.scores + ((here.b * p.units + unit) * p.line + (int64_t)at * kKeys + g) * kNH + 2 * qd;
#pragma unroll
        for (int r = 0; r < kR; ++r) {
#pragma unroll
          for (int t = 0; t < kNT; ++t) {
            *reinterpret_cast<float2*>(to + 16 * r * kNH + 8 * t) = make_float2(sc[t][r][0], sc[t][r][1]);
            *reinterpret_cast<float2*>(to + (16 * r + 8) * kNH + 8 * t) = make_float2(sc[t][r][2], sc[t][r][3]);
          }
        }
      }
      if (live != 0u) {
        if (__any_sync(kAll, over)) {
#pragma unroll
          for (int t = 0; t < kNT; ++t) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float all = keys_max(top[t][e]);
              const float m = all > mx[t][e] + 8.f ? all : mx[t][e];
              const float grow = mx[t][e] == m ? 1.f : ex2(mx[t][e] - m);  // (-inf both: nothing seen yet)
              sum[t][e] = kFp8 ? brought(sum[t][e], mx[t][e], m) : sum[t][e] * grow;
              mx[t][e] = m;
#pragma unroll
              for (int i = 0; i < kTiles; ++i) o[t][i][e] *= grow, o[t][i][2 + e] *= grow;
            }
          }
        }
#pragma unroll
        for (int r = 0; r < kR; ++r) {
          uint32_t pb[kNT][2];
#pragma unroll
          for (int t = 0; t < kNT; ++t) {
            const float m0 = mx[t][0] == -INFINITY ? 0.f : mx[t][0], m1 = mx[t][1] == -INFINITY ? 0.f : mx[t][1];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float a = ex2(sc[t][r][2 * e] - m0), b = ex2(sc[t][r][2 * e + 1] - m1);
              sum[t][0] += a, sum[t][1] += b;
              pb[t][e] = turned8x8(kFp8 ? narrow2(a * vs[r][e], b * vs[r][e], M()) : narrow2(a, b, M()));
            }
          }
          // lanes 0-7 and 8-15 name the rows of keys 0-7 and 8-15 at one piece, lanes 16-31 at the next
          const uint32_t vat = stage + (uint32_t)(G::kV + (16 * r + (lane & 15)) * G::kRowBytes);
#pragma unroll
          for (int c = 0; c < G::kRowBytes / 32; ++c) {
            uint32_t x[4];
            ldsm4_trans(x, vat + G::v_piece(lane & 15, 2 * c + (lane >> 4)) * 16u);
            if constexpr (kFp8) {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                uint32_t f[4];
                widen4(f[0], f[1], __byte_perm(x[2 * h], 0u, 0x3120));
                widen4(f[2], f[3], __byte_perm(x[2 * h + 1], 0u, 0x3120));
#pragma unroll
                for (int t = 0; t < kNT; ++t) mma16816(o[t][2 * c + h], f, pb[t][0], pb[t][1], M());
              }
            } else {
              const uint32_t f[4] = {x[0], x[2], x[1], x[3]};
#pragma unroll
              for (int t = 0; t < kNT; ++t) mma16816(o[t][c], f, pb[t][0], pb[t][1], M());
            }
          }
        }
      }
    }
    __syncwarp();  // (the next block but kStages - 2 goes where this one was)
    }
    // ---- the segment's end: the stage that is asked for next is free, and takes the warp's accumulators, [heads][D] ----
    static_assert(G::kStage >= kNH * D * 4, "a stage holds the accumulators");
    const bool whole = here.s0 == 0 && here.s1 == here.blocks;
    const int64_t rec = (int64_t)run_unit * 2 + which;
    const uint32_t mine = (uint32_t)(warp * G::kBytes + ask_stage * G::kStage);
#pragma unroll
    for (int t = 0; t < kNT; ++t) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int h = 8 * t + 2 * qd + e;
        const float l = keys_sum(sum[t][e]);
        if (g == 0) ml_of[warp][h] = make_float2(mx[t][e], l);
        // channels of the accumulators: 16 bits g and g + 8 of a tile, e4m3 2 g and 2 g + 1
        float* const row = reinterpret_cast<float*>(smem_raw + mine) + h * D;
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
          row[16 * i + (kFp8 ? 2 * g : g)] = o[t][i][e];
          row[16 * i + (kFp8 ? 2 * g + 1 : g + 8)] = o[t][i][2 + e];
        }
      }
    }
    if (lane == 0) free_of[warp] = mine;
    __syncthreads();
    // the warps' four channels d .. d + 3 of head h
    auto joined = [&](int h, int d, float& m, float& l) {
      m = -INFINITY, l = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) m = fmaxf(m, ml_of[w][h].x);
      float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float2 ml = ml_of[w][h];
        const float f = ml.x == m ? 1.f : ex2(ml.x - m);  // (a warp without keys: 0 of both; 0 * NaN stays NaN)
        l += kFp8 ? brought(ml.y, ml.x, m) : f * ml.y;
        const float4 x = *reinterpret_cast<const float4*>(smem_raw + free_of[w] + (h * D + d) * 4);
        y.x += f * x.x, y.y += f * x.y, y.z += f * x.z, y.w += f * x.w;
      }
      return y;
    };
    auto finish = [&](int h, int d, float m, float l, const float4& y) {
      T* out = static_cast<T*>(p.a.out) + here.b * p.a.out_seq + (int64_t)(head0 + h) * p.a.out_head + d;
      const float r[4] = {l == 0.f ? 0.f : y.x / l, l == 0.f ? 0.f : y.y / l, l == 0.f ? 0.f : y.z / l, l == 0.f ? 0.f : y.w / l};
      Four<T> narrow;
      narrow.narrow(r);
      if (p.out_vec)
        narrow.template store<true>(out);
      else
        narrow.template store<false>(out);
      if (d == 0) {
        const float l2 = l == 0.f ? -INFINITY : m + log2f(l);
        if (p.a.lse != nullptr) p.a.lse[here.b * p.a.q_heads + head0 + h] = l2 * 0.693147180559945309f;
        if (p.weigh && !p.weigh_here) p.lse2[here.b * p.a.q_heads + head0 + h] = l2;
      }
    };
    // the weights of the segment's positions, from the scores that the CTA has written and the sums of all of the sequence
    auto weigh = [&]() {
      if (threadIdx.x < kNH) {
        float m = -INFINITY, l = 0.f;
        for (uint32_t c = 0; c < ctas; ++c) {
          const float2 ml = ctas > 1 ? lds_cluster2(shared_of(smem_u32(&joined_ml[threadIdx.x]), (int)c)) : joined_ml[threadIdx.x];
          const float top = fmaxf(m, ml.x);
          l = brought(l, m, top) + brought(ml.y, ml.x, top);
          m = top;
        }
        log_sum[threadIdx.x] = l == 0.f ? INFINITY : m + log2f(l);  // (without keys: everything counts nothing against infinity)
      }
      __syncthreads();
      const float* w = p.a.weight != nullptr ? p.a.weight + here.b * p.a.w_seq + (int64_t)kvh * p.a.w_head : nullptr;
      float* wo = p.a.weight_out + here.b * p.a.wo_seq + (int64_t)kvh * p.a.wo_head;
      const float* s = p.scores + (here.b * p.units + unit) * p.line * kNH;
      const int64_t upto = min((int64_t)here.n, (int64_t)here.s1 * kKeys);
#pragma unroll 2
      for (int64_t j = (int64_t)here.s0 * kKeys + threadIdx.x; j < upto; j += kThreads) {
        if (j < p.a.weight_cols) {
          const float before = w != nullptr ? w[j] : 0.f;
          float sum = 0.f;  // (of its own: what has been added up over many calls is far larger than a head's weight, and is rounded once)
#pragma unroll
          for (int i = 0; i < kNH / 4; ++i) {
            const float4 x = *reinterpret_cast<const float4*>(s + j * kNH + 4 * i);
            const float e[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int u = 0; u < 4; ++u) sum += 4 * i + u < heads ? ex2(e[u] - log_sum[4 * i + u]) : 0.f;
          }
          wo[j] = before + sum;
        } else if (p.status) {
          atomicOr(p.status, (uint32_t)FFTOPK_ST_BAD_INDEX);
        }
      }
    };
    if (ctas > 1) {
      // The cluster's CTAs are joined through distributed shared memory. Each puts what its warps have where its rings begin - every block has been used, and
      // what comes from its warps' stages is in registers by then - and finishes its share of the rows.
      constexpr int kRows = kNH * (D / 4) / kThreads;  // of a thread
      static_assert(kRows * kThreads == kNH * (D / 4), "a thread has whole rows");
      float4 y[kRows];
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const int at = (int)threadIdx.x + i * kThreads, h = at / (D / 4), d = at % (D / 4) * 4;
        float m, l;
        y[i] = joined(h, d, m, l);
        if (d == 0) joined_ml[h] = make_float2(m, l);
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kRows; ++i) reinterpret_cast<float4*>(smem_raw)[threadIdx.x + i * kThreads] = y[i];
      cg::cluster_group cluster = cg::this_cluster();
      cluster.sync();
      for (int at = (int)(threadIdx.x + rank * kThreads); at < heads * (D / 4); at += kThreads * (int)ctas) {
        const int h = at / (D / 4), d = at % (D / 4) * 4;
        // (every CTA's part is asked for before any is used)
        const uint32_t ml_at = smem_u32(&joined_ml[h]), o_at = smem_u32(smem_raw) + (uint32_t)at * 16u;
        float2 ml[kMaxApart];
        float4 part[kMaxApart];
        float m = -INFINITY, l = 0.f;
#pragma unroll
        for (int c = 0; c < kMaxApart; ++c) {
          ml[c] = make_float2(-INFINITY, 0.f), part[c] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (c < (int)ctas) ml[c] = lds_cluster2(shared_of(ml_at, c)), part[c] = lds_cluster4(shared_of(o_at, c));
        }
#pragma unroll
        for (int c = 0; c < kMaxApart; ++c) m = fmaxf(m, ml[c].x);
        float4 all = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int c = 0; c < kMaxApart; ++c) {
          const float f = ml[c].x == m ? 1.f : ex2(ml[c].x - m);
          l += kFp8 ? brought(ml[c].y, ml[c].x, m) : f * ml[c].y;
          all.x += f * part[c].x, all.y += f * part[c].y, all.z += f * part[c].z, all.w += f * part[c].w;
        }
        finish(h, d, m, l, all);
      }
      if (p.weigh_here) weigh();
      cluster.sync();  // (nobody leaves while its memory is read)
      return;
    }
    for (int i = threadIdx.x; i < heads * (D / 4); i += kThreads) {
      const int h = i / (D / 4), d = i % (D / 4) * 4;
      float m, l;
      const float4 y = joined(h, d, m, l);
      if (whole) {
        finish(h, d, m, l, y);
        if (d == 0) joined_ml[h] = make_float2(m, l);
      } else {
        *reinterpret_cast<float4*>(p.o + (rec * kNH + h) * D + d) = y;
        if (d == 0) p.ml[rec * kNH + h] = make_float2(m, l);
      }
    }
    __syncthreads();
    if (p.weigh_here) weigh();  // (one segment a CTA)
    left -= here.s1 - here.s0;
    if (left <= 0 || !next_segment(p, here, left)) break;
    quarter(here, warp, at, end);
    which = 1;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// Parts of one unit of a sequence that lies in several runs: records `first`, and then every `step`-th from `second`
struct Parts {
  int64_t first, second, step;
  int32_t n;
  __device__ __forceinline__ Parts(const PagedParams& p, const Runs& line, int64_t begin, int64_t end, int unit) {
    const int64_t r0 = p.apart ? 0 : line.of(begin), r1 = p.apart ? 0 : line.of(end - 1);
    n = (int32_t)(r1 - r0) + 1;
    first = (r0 * p.units + unit) * 2 + (line.begin(r0) < begin ? 1 : 0);  // (the sequence begins inside its first run)
    second = ((r0 + 1) * p.units + unit) * 2;
    step = (int64_t)p.units * 2;
  }
  __device__ __forceinline__ int64_t operator[](int i) const { return i == 0 ? first : second + (i - 1) * step; }
};

// A warp's share - parts i0, i0 + step, .. - of a head's joined sums: running maximum and sum, kC channels a lane
template <int kC>
__device__ __forceinline__ void join_parts(const PagedParams& p, const Parts& parts, int nh, int h, int i0, int step, int lane, float& m, float& l,
                                           float (&acc)[kC]) {
  constexpr int kAhead = 8;
  m = -INFINITY, l = 0.f;
#pragma unroll
  for (int c = 0; c < kC; ++c) acc[c] = 0.f;
  for (int i = i0; i < parts.n; i += kAhead * step) {
    float2 ml[kAhead];
    float x[kAhead][kC];
    float top = m;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      ml[u] = make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int c = 0; c < kC; ++c) x[u][c] = 0.f;
      if (i + u * step < parts.n) {
        const int64_t r = parts[i + u * step] * nh + h;
        ml[u] = p.ml[r];
        const float* o = p.o + (r * 32 + lane) * kC;
        if constexpr (kC == 4) {
          const float4 v = *reinterpret_cast<const float4*>(o);
          x[u][0] = v.x, x[u][1] = v.y, x[u][2] = v.z, x[u][3] = v.w;
        } else {
          const float2 v = *reinterpret_cast<const float2*>(o);
          x[u][0] = v.x, x[u][1] = v.y;
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) top = fmaxf(top, ml[u].x);
    const float was = m == top ? 1.f : ex2(m - top);
    l = brought(l, m, top);
#pragma unroll
    for (int c = 0; c < kC; ++c) acc[c] *= was;
    m = top;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const float f = ml[u].x == m ? 1.f : ex2(ml[u].x - m);  // (a part without keys: 0 of both; 0 * NaN stays NaN)
      l += brought(ml[u].y, ml[u].x, m);
#pragma unroll
      for (int c = 0; c < kC; ++c) acc[c] += f * x[u][c];
    }
  }
}

template <typename T, int kC>
__device__ __forceinline__ void write_joined(const PagedParams& p, int64_t b, int head, int lane, float m, float l, const float (&acc)[kC]) {
  T* out = static_cast<T*>(p.a.out) + b * p.a.out_seq + (int64_t)head * p.a.out_head + lane * kC;
#pragma unroll
  for (int c = 0; c < kC; ++c) out[c] = T(l == 0.f ? 0.f : acc[c] / l);
  if (lane == 0 && p.a.lse != nullptr) p.a.lse[b * p.a.q_heads + head] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.693147180559945309f;
}

// What is left when every run is through. The first CTAs join the parts of sequences that lie in several runs: a warp takes a few pairs of a
// sequence and a query head, or, where there are few, a CTA one of them. The others bring the weights up to date from the scores and the
// joined sums: a warp takes a run of the line for one key head, a lane a position. Where sequences begin is found while the kernel in front still runs.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 5) paged_finish_kernel(const __grid_constant__ PagedParams p) {
  constexpr int kC = D / 32;  // channels of a lane
  __shared__ float4 part[kWarps][D / 4];
  __shared__ float2 ml_of[kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int nh = p.group > 8 ? 16 : 8;
  const int64_t total = blocks_before(p, p.a.seqs, lane);
  const Runs line(total, p.runs, kMinKeys >> p.key_shift);
  if ((int)blockIdx.x < p.join_ctas) {
    const int64_t pairs = p.a.seqs * p.a.q_heads;
    int64_t i = p.join_each == 0 ? blockIdx.x : ((int64_t)blockIdx.x * kWarps + warp) * p.join_each;
    const int64_t last = min(pairs, i + max(p.join_each, 1));
    int64_t b = i / p.a.q_heads, begin = blocks_before(p, min(b, p.a.seqs), lane);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    for (; i < last; ++i) {
      if (i / p.a.q_heads != b) {
        begin += blocks_of(p, keys_of(p, b));
        ++b;
      }
      const int64_t end = begin + blocks_of(p, keys_of(p, b));
      if (begin == end) continue;
      const int head = (int)(i - b * p.a.q_heads), kvh = head / p.group, in = head - kvh * p.group, hb = in / nh;
      const Parts parts(p, line, begin, end, kvh * p.head_blocks + hb);
      if (parts.n == 1) continue;
      float m, l, acc[kC];
      if (p.join_each != 0) {
        join_parts<kC>(p, parts, nh, in - hb * nh, 0, 1, lane, m, l, acc);
      } else {
        join_parts<kC>(p, parts, nh, in - hb * nh, warp, kWarps, lane, m, l, acc);
#pragma unroll
        for (int c = 0; c < kC; ++c) reinterpret_cast<float*>(part[warp])[lane * kC + c] = acc[c];
        if (lane == 0) ml_of[warp] = make_float2(m, l);
        __syncthreads();  // (the CTA has one pair)
        if (warp != 0) return;
        const float2 own = ml_of[0];
        m = own.x, l = own.y;
#pragma unroll
        for (int w = 1; w < kWarps; ++w) {
          const float2 ml = ml_of[w];
          const float top = fmaxf(m, ml.x), was = m == top ? 1.f : ex2(m - top), f = ml.x == top ? 1.f : ex2(ml.x - top);
          l = brought(l, m, top) + brought(ml.y, ml.x, top);
#pragma unroll
          for (int c = 0; c < kC; ++c) acc[c] = acc[c] * was + f * reinterpret_cast<const float*>(part[w])[lane * kC + c];
          m = top;
        }
      }
      write_joined<T, kC>(p, b, head, lane, m, l, acc);
    }
    return;
  }
  // ---- weights ----
  const uint32_t gw = (blockIdx.x - (uint32_t)p.join_ctas) * (uint32_t)kWarps + (uint32_t)warp;
  const uint32_t run = gw / (uint32_t)p.a.kv_heads;
  const int kvh = (int)(gw - run * (uint32_t)p.a.kv_heads);
  const Runs mine(total, p.weigh_runs, kWeighKeys >> p.key_shift);
  int64_t left = (int64_t)run < mine.runs ? mine.begin((int64_t)run + 1) - mine.begin(run) : 0;
  Segment c = {};
  if (left > 0) c = segment_at(p, mine.begin(run), left, lane);
  int64_t begin = mine.begin(run) - c.s0;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // (by every CTA: this kernel does not end before the one in front)
  if (left <= 0) return;
  for (;;) {
    const int64_t end = begin + c.blocks;
    const int32_t upto = (int32_t)min((int64_t)c.n, (int64_t)c.s1 << p.key_shift);
    const float* w = p.a.weight != nullptr ? p.a.weight + c.b * p.a.w_seq + (int64_t)kvh * p.a.w_head : nullptr;
    float* wo = p.a.weight_out + c.b * p.a.wo_seq + (int64_t)kvh * p.a.wo_head;
    for (int hb = 0; hb < p.head_blocks; ++hb) {
      const int unit = kvh * p.head_blocks + hb, heads = min(nh, p.group - hb * nh);
      const Parts parts(p, line, begin, end, unit);
      // log2 of the head's sum of exponentials, in the lane of the head's number
      float all = -INFINITY;
      if (parts.n == 1) {
        if (lane < heads) all = p.lse2[c.b * p.a.q_heads + (int64_t)kvh * p.group + hb * nh + lane];
      } else {
        float m = -INFINITY, l = 0.f;  // (lanes of a head take its parts in turn)
        for (int i = lane / nh; i < parts.n; i += 4 * (32 / nh)) {
          float2 ml[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int at = i + u * (32 / nh);
            ml[u] = at < parts.n ? p.ml[parts[at] * nh + lane % nh] : make_float2(-INFINITY, 0.f);
          }
          const float top = fmaxf(fmaxf(m, fmaxf(ml[0].x, ml[1].x)), fmaxf(ml[2].x, ml[3].x));
          l = brought(l, m, top);
          m = top;
#pragma unroll
          for (int u = 0; u < 4; ++u) l += brought(ml[u].y, ml[u].x, m);
        }
        for (int i = nh; i < 32; i *= 2) {
          const float m2 = __shfl_xor_sync(kAll, m, i), l2 = __shfl_xor_sync(kAll, l, i), top = fmaxf(m, m2);
          l = brought(l, m, top) + brought(l2, m2, top);
          m = top;
        }
        all = l == 0.f ? -INFINITY : m + log2f(l);
      }
      for (int h8 = 0; h8 < heads; h8 += 8) {
        float all8[8];  // (without keys: everything counts nothing against infinity)
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          const float a = __shfl_sync(kAll, all, (h8 + n) & 31);
          all8[n] = a != -INFINITY ? a : INFINITY;
        }
        const float* s = p.scores + (c.b * p.units + unit) * p.line * nh + h8;
        const bool first = hb == 0 && h8 == 0;
        constexpr int kAhead = 4;
        for (int64_t j0 = ((int64_t)c.s0 << p.key_shift) + lane; j0 - lane < upto; j0 += 32 * kAhead) {
          float4 x[kAhead][2];
          float y[kAhead];
#pragma unroll
          for (int u = 0; u < kAhead; ++u) {
            const int64_t j = j0 + 32 * u;
            y[u] = 0.f;
            if (j < upto && j < p.a.weight_cols) {
              x[u][0] = *reinterpret_cast<const float4*>(s + j * nh);
              x[u][1] = *reinterpret_cast<const float4*>(s + j * nh + 4);
              if (!first)
                y[u] = wo[j];
              else if (w != nullptr)
                y[u] = w[j];
            }
          }
#pragma unroll
          for (int u = 0; u < kAhead; ++u) {
            const int64_t j = j0 + 32 * u;
            if (j < upto && j < p.a.weight_cols) {
              const float e[8] = {x[u][0].x, x[u][0].y, x[u][0].z, x[u][0].w, x[u][1].x, x[u][1].y, x[u][1].z, x[u][1].w};
              float sum = 0.f;
#pragma unroll
              for (int n = 0; n < 8; ++n) sum += h8 + n < heads ? ex2(e[n] - all8[n]) : 0.f;
              wo[j] = y[u] + sum;  // (rounded once for every eight heads)
            } else if (j < upto && p.status) {
              atomicOr(p.status, (uint32_t)FFTOPK_ST_BAD_INDEX);
            }
          }
        }
      }
    }
    left -= c.s1 - c.s0;
    begin = end;
    if (left <= 0 || !next_segment(p, c, left)) break;
  }
}

DeviceOnce g_paged_once[kMaxDevices];
struct PagedLimits {
  int sms = 0;
  int eights[2][2][2] = {};  // clusters of eight CTAs the device holds at once: [e4m3][heads of 128][sixteens of query heads]
};
PagedLimits g_paged_limits[kMaxDevices];

template <typename T, bool kFp8, int D, int kNT>
int setup_one() {
  cudaError_t e =
      cudaFuncSetAttribute(paged_kernel<T, kFp8, D, kNT, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)paged_smem<kFp8, D>());
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(paged_kernel<T, kFp8, D, kNT, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)paged_smem<kFp8, D>());
  return e == cudaSuccess ? 0 : cuda_fail(e);
}
template <typename T, bool kFp8>
int setup_two() {
  int r = setup_one<T, kFp8, 64, 1>();
  if (!r) r = setup_one<T, kFp8, 64, 2>();
  if (!r) r = setup_one<T, kFp8, 128, 1>();
  if (!r) r = setup_one<T, kFp8, 128, 2>();
  return r;
}
template <bool kFp8, int D>
int eights_of(PagedLimits& limits) {
  int r = clusters_of(limits.eights[kFp8][D == 128][0], paged_kernel<__nv_bfloat16, kFp8, D, 1, true>, kThreads, paged_smem<kFp8, D>());
  if (!r) r = clusters_of(limits.eights[kFp8][D == 128][1], paged_kernel<__nv_bfloat16, kFp8, D, 2, true>, kThreads, paged_smem<kFp8, D>());
  return r;
}
int paged_setup(PagedLimits& limits) {
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e);
  if (dev < 0 || dev >= kMaxDevices) return FFTOPK_EDEVICE;
  const int rc = g_paged_once[dev].run([&] {
    const cudaError_t e2 = cudaDeviceGetAttribute(&g_paged_limits[dev].sms, cudaDevAttrMultiProcessorCount, dev);
    if (e2 != cudaSuccess) return cuda_fail(e2);
    int r = setup_two<__nv_bfloat16, false>();
    if (!r) r = setup_two<__nv_bfloat16, true>();
    if (!r) r = setup_two<__half, false>();
    if (!r) r = setup_two<__half, true>();
    if (!r) r = eights_of<false, 64>(g_paged_limits[dev]);
    if (!r) r = eights_of<false, 128>(g_paged_limits[dev]);
    if (!r) r = eights_of<true, 64>(g_paged_limits[dev]);
    if (!r) r = eights_of<true, 128>(g_paged_limits[dev]);
    return r;
  });
  limits = g_paged_limits[dev];
  return rc;
}

template <typename... A>
cudaError_t launch(void (*kernel)(A...), int64_t grid, int threads, size_t smem, int cluster, bool dependent, cudaStream_t stream, const PagedParams& p) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid, 1, 1);
  cfg.blockDim = dim3((unsigned)threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  if (cluster > 1) {
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)cluster;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
  } else {
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
  }
  cfg.attrs = at;
  cfg.numAttrs = cluster > 1 || dependent ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

bool on(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(bytes - 1)) == 0; }
// rows of 16-byte pieces whatever their sequence (slot) and head; the stride of a lone one says nothing
bool on16(const void* p, int64_t n, int64_t a, int64_t heads, int64_t b, int bytes) {
  return on(p, 16) && (n <= 1 || a * bytes % 16 == 0) && (heads <= 1 || b * bytes % 16 == 0);
}

// Keys of a block and CTAs per SM of the kernel that a call goes to
struct Form {
  int keys, ctas;
};
template <bool kFp8, int D>
Form form_of(int nt) {
  return nt == 1 ? Form{block_keys<kFp8, D>(), paged_ctas<kFp8, D, 1>()} : Form{block_keys<kFp8, D>(), paged_ctas<kFp8, D, 2>()};
}
Form form_of(bool fp8, int D, int nt) {
  if (D == 64) return fp8 ? form_of<true, 64>(nt) : form_of<false, 64>(nt);
  return fp8 ? form_of<true, 128>(nt) : form_of<false, 128>(nt);
}

// Sizes of the call, checked; what the workspace holds in turn: lse2, ml, o, scores
struct Plan {
  int nt = 1, nh = 8;
  int64_t ctas = 0, finish_ctas = 0, bytes[4] = {}, total = 0;
};
int64_t up256(int64_t n) { return (n + 255) & ~(int64_t)255; }
int make_plan(const fftopk_paged* a, const PagedLimits& limits, PagedParams& p, Plan& plan) {
  const int sms = limits.sms;
  memset(&p, 0, sizeof(p));
  p.a = *a;
  p.group = a->q_heads / a->kv_heads;
  plan.nt = p.group > 8 ? 2 : 1;
  plan.nh = 8 * plan.nt;
  p.head_blocks = (p.group + plan.nh - 1) / plan.nh;
  const int64_t units = (int64_t)a->kv_heads * p.head_blocks;
  const int64_t bound = (int64_t)a->pages * a->page_size;
  if (units > 0x1000000 || a->seqs > 0x7fffffff / a->q_heads || bound > 0x7ffffff0) return FFTOPK_ERANGE;
  p.units = (int32_t)units;
  p.bound = (int32_t)bound;
  p.weigh = a->weight_out != nullptr;
  const Form form = form_of(a->k_scale != nullptr, a->D, plan.nt);
  const int keys = form.keys;
  p.key_shift = keys == 32 ? 5 : 4;
  const int64_t blocks = a->seqs * ((bound + keys - 1) / keys);
  const int64_t ctas = (int64_t)sms * form.ctas;
  int64_t runs = ctas / units < blocks / (kMinKeys / keys) ? ctas / units : blocks / (kMinKeys / keys);
  if (runs < 1) runs = 1;
  // Short tables: a sequence and key head is a piece of work, taken by a cluster - of as many CTAs as fit the device at once and have 128 positions each - that joins
  // it by itself. What it saves - the search for runs, the second kernel - is worth more than what unequal lengths cost while a CTA reads 200 KB at most, or
  // 800 KB where there are CTAs for four fifths of the device (in clusters and in equal runs: one sequence of 1,000 8.0 us and 9.3, of 4,096 10.7 and 9.8, of
  // 16,000 27 and 16; 8 of up to 1,000 8.6 and 13; 37 with 3 key heads of 64 of up to 2,999 16 and 20; 64 of up to 300 15 and 23; 32 of up to 1,500 30 and 39; 40 of
  // up to 2,500, which are 1.3 MB, 66 and 60)
  const double bytes = (double)bound * a->D * (a->k_scale != nullptr ? 1 : 2) * 2;
  const int64_t pieces = a->seqs * units, eights = limits.eights[a->k_scale != nullptr][a->D == 128][plan.nt - 1];
  int apart = 1;
  while (apart < kMaxApart && pieces * apart * 2 <= ctas && bound / (apart * 2) >= kMinKeys && (apart * 2 < 8 || pieces <= eights)) apart *= 2;
  if (bytes <= 200e3 * apart || (bytes <= 800e3 * apart && pieces * apart * 5 >= (int64_t)sms * 4)) p.apart = apart, runs = a->seqs;
  p.runs = (int32_t)runs;
  plan.ctas = runs * units * (p.apart > 1 ? p.apart : 1);
  p.line = (bound + keys - 1) / keys * keys;
  if (runs > 1 && !p.apart) {
    plan.bytes[1] = up256(runs * units * 2 * plan.nh * 8);
    plan.bytes[2] = up256(runs * units * 2 * plan.nh * a->D * 4);
    // a warp a pair where a CTA each would take more than the device holds at once, and several where that would
    const int64_t pairs = a->seqs * a->q_heads, room = (int64_t)sms * 64;
    p.join_each = pairs * kWarps <= room ? 0 : (int32_t)((pairs + room - 1) / room);
    plan.finish_ctas = p.join_ctas = (int32_t)(p.join_each == 0 ? pairs : ((pairs + p.join_each - 1) / p.join_each + kWarps - 1) / kWarps);
  }
  if (p.weigh) {
    plan.bytes[0] = up256(a->seqs * a->q_heads * 4);
    // (below 2^31 sequences * heads, times 2^31 positions, times 64 bytes: in question where it would wrap)
    if (p.line > 0 && a->seqs * units > ((int64_t)1 << 50) / (p.line * plan.nh)) return FFTOPK_ERANGE;
    plan.bytes[3] = up256(a->seqs * units * p.line * plan.nh * 4);
  }
  p.weigh_here = p.weigh && p.apart && p.head_blocks == 1;
  if (p.weigh && !p.weigh_here) {
    int64_t each = (int64_t)sms * 8 * kWarps / a->kv_heads;
    if (each > blocks) each = blocks;
    if (each < 1) each = 1;
    p.weigh_runs = (int32_t)each;
    plan.finish_ctas += (each * a->kv_heads + kWarps - 1) / kWarps;
  }
  for (int64_t n : plan.bytes) plan.total += n;
  return 0;
}

int check(const fftopk_paged* a) {
  if (a == nullptr) return FFTOPK_EINVAL;
  if (a->seqs < 0 || a->kv_heads < 0 || a->q_heads < 0 || a->slots < 0 || a->pages < 0 || a->page_size < 1 || a->weight_cols < 0) return FFTOPK_EINVAL;
  if (a->dtype != FFTOPK_DTYPE_FP16 && a->dtype != FFTOPK_DTYPE_BF16) return FFTOPK_EINVAL;
  if (a->D != 64 && a->D != 128) return FFTOPK_ERANGE;
  if (a->seqs == 0 || a->q_heads == 0) return FFTOPK_OK;
  if (a->kv_heads == 0 || a->q_heads % a->kv_heads != 0) return FFTOPK_EINVAL;
  const bool fp8 = a->k_scale != nullptr;
  if (fp8 != (a->v_scale != nullptr)) return FFTOPK_EINVAL;
  if (!a->q || !a->out || !a->lengths || (a->pages > 0 && !a->page_table) || (a->pages > 0 && a->slots > 0 && (!a->k || !a->v))) return FFTOPK_EINVAL;
  if (a->weight != nullptr && a->weight_out == nullptr) return FFTOPK_EINVAL;
  const int ce = fp8 ? 1 : 2;
  if (!on16(a->q, a->seqs, a->q_seq, a->q_heads, a->q_head, 2) || !on16(a->k, a->slots, a->k_slot, a->kv_heads, a->k_head, ce) ||
      !on16(a->v, a->slots, a->v_slot, a->kv_heads, a->v_head, ce))
    return FFTOPK_EINVAL;
  if (!on(a->out, 2) || !on(a->page_table, 4) || !on(a->lengths, 4) || !on(a->lse, 4) || !on(a->k_scale, 4) || !on(a->v_scale, 4) ||
      !on(a->weight, 4) || !on(a->weight_out, 4))
    return FFTOPK_EINVAL;
  if (a->slots > 0x7fffffff || a->seqs > 0x7fffffff) return FFTOPK_ERANGE;
  // (the kernel multiplies slots by 32-bit strides; a lone slot's says nothing)
  if (a->slots > 1 && (a->k_slot < 0 || a->v_slot < 0 || a->k_slot > 0xffffffffll / ce || a->v_slot > 0xffffffffll / ce)) return FFTOPK_ERANGE;
  return FFTOPK_OK;
}

template <typename T, bool kFp8, int D, int kNT>
cudaError_t launch_paged(const PagedParams& p, const Plan& plan, cudaStream_t stream) {
  const bool whole = p.a.page_size % block_keys<kFp8, D>() == 0;
  return launch(whole ? paged_kernel<T, kFp8, D, kNT, true> : paged_kernel<T, kFp8, D, kNT, false>, plan.ctas, kThreads, paged_smem<kFp8, D>(), p.apart, false, stream, p);
}
template <typename T, bool kFp8, int D>
cudaError_t launch_paged(const PagedParams& p, const Plan& plan, cudaStream_t stream) {
  return plan.nt == 1 ? launch_paged<T, kFp8, D, 1>(p, plan, stream) : launch_paged<T, kFp8, D, 2>(p, plan, stream);
}
template <typename T>
cudaError_t launch_paged(const PagedParams& p, const Plan& plan, cudaStream_t stream) {
  const bool fp8 = p.a.k_scale != nullptr;
  const bool d64 = p.a.D == 64;
  cudaError_t e = fp8 ? (d64 ? launch_paged<T, true, 64>(p, plan, stream) : launch_paged<T, true, 128>(p, plan, stream))
                      : d64 ? launch_paged<T, false, 64>(p, plan, stream) : launch_paged<T, false, 128>(p, plan, stream);
  if (e == cudaSuccess && plan.finish_ctas > 0)
    e = launch(d64 ? paged_finish_kernel<T, 64> : paged_finish_kernel<T, 128>, plan.finish_ctas, kThreads, 0, 1, true, stream, p);
  return e;
}

}  // namespace
}  // namespace fftopk

using namespace fftopk;

extern "C" {

int fftopk_paged_workspace_bytes(const fftopk_paged* a, size_t* bytes) {
  if (bytes == nullptr) return FFTOPK_EINVAL;
  *bytes = 0;
  int rc = check(a);
  if (rc || a->seqs == 0 || a->q_heads == 0) return rc;
  PagedLimits limits;
  rc = paged_setup(limits);
  if (rc) return rc;
  PagedParams p;
  Plan plan;
  rc = make_plan(a, limits, p, plan);
  if (rc == 0) *bytes = (size_t)plan.total;
  return rc;
}

int fftopk_paged_attention(const fftopk_paged* a, void* workspace, size_t workspace_bytes, uint32_t* status, void* cuda_stream) {
  int rc = check(a);
  if (rc || a->seqs == 0 || a->q_heads == 0) return rc;
  // (rows written twice would hold whichever came last)
  if (!rows_apart(a->seqs, a->out_seq, a->q_heads, a->out_head, a->D)) return FFTOPK_EINVAL;
  if (a->weight_out != nullptr && !rows_apart(a->seqs, a->wo_seq, a->kv_heads, a->wo_head, a->weight_cols)) return FFTOPK_EINVAL;
  // (q is read by several CTAs, at different times; weights by other threads than those that write what is elsewhere)
  if (rows_meet(a->q, a->q_seq, a->q_head, a->out, a->out_seq, a->out_head, a->seqs, a->q_heads, a->D, 2)) return FFTOPK_EINVAL;
  const bool in_place = a->weight == a->weight_out && (a->seqs == 1 || a->w_seq == a->wo_seq) && (a->kv_heads == 1 || a->w_head == a->wo_head);
  if (a->weight != nullptr && !in_place &&
      rows_meet(a->weight, a->w_seq, a->w_head, a->weight_out, a->wo_seq, a->wo_head, a->seqs, a->kv_heads, a->weight_cols, 4))
    return FFTOPK_EINVAL;
  PagedLimits limits;
  rc = paged_setup(limits);
  if (rc) return rc;
  PagedParams p;
  Plan plan;
  rc = make_plan(a, limits, p, plan);
  if (rc) return rc;
  if (plan.total > 0 && (workspace == nullptr || !on(workspace, 256) || workspace_bytes < (size_t)plan.total)) return FFTOPK_EINVAL;
  if (a->slots <= 1) p.a.k_slot = p.a.v_slot = 0;
  if (a->slots == 0) p.a.k = p.a.v = a->q;  // (an empty cache has no address, and rows that are left out are copies of no bytes: from somewhere)
  p.page = FastDiv((uint32_t)a->page_size);
  p.scale_log2 = a->softmax_scale * 1.44269504088896340736f;
  const int es = a->k_scale != nullptr ? 1 : 2;
  p.stream = (double)a->seqs * p.bound * a->kv_heads * a->D * es * 2 > 128e6;
  p.out_vec = on(a->out, 8) && (a->seqs <= 1 || a->out_seq % 4 == 0) && (a->q_heads <= 1 || a->out_head % 4 == 0);
  p.status = status;
  char* at = static_cast<char*>(workspace);
  p.lse2 = reinterpret_cast<float*>(at), at += plan.bytes[0];
  p.ml = reinterpret_cast<float2*>(at), at += plan.bytes[1];
  p.o = reinterpret_cast<float*>(at), at += plan.bytes[2];
  p.scores = reinterpret_cast<float*>(at);
  cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  const cudaError_t e = a->dtype == FFTOPK_DTYPE_BF16 ? launch_paged<__nv_bfloat16>(p, plan, stream) : launch_paged<__half>(p, plan, stream);
  return e == cudaSuccess ? FFTOPK_OK : cuda_fail(e);
}

}  // extern "C"
