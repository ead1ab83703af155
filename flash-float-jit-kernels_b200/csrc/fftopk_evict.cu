// Eviction from a paged cache by accumulated attention weight. Of every sequence and key head `budget` rows stay: the first `sinks`, the
// last `recent`, and of those between the ones of the largest weights (equal weights: the lower position). They go, in order, to the
// rows that another page table names; their weights go along. A sequence of up to `budget` rows keeps them all. (The reference ends with
// the selection of indices; attention over a paged cache that adds up the weights is fftopk_paged.cu.)
//
// evict_select_kernel: a CTA or a cluster per sequence and key head finds the smallest weight that stays, by radix rounds over the order-preserving keys
// of the weights (11, 11 and 10 bits, histograms in shared memory, summed over the cluster), and lists what stays in order. The first round
// counts weights as they come in; behind it every 32 positions are a word of bits - above the threshold's bin, in it - and what
// follows looks at the few that are in it. Places in the list are prefix sums over the words. A weight is read once and stays in
// shared memory (positions beyond its room are read again).
// evict_move_kernel: a warp takes 32 rows of a key head that lie next to each other where they go; a lane finds where one of them comes from, and
// the warp copies k and v. Reading and writing the rows bounds it.
#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

#include "../../include/fftopk.h"
#include "fftopk_attend.cuh"
#include "fftopk_extent.h"
#include "fftopk_host.h"
#include "fftopk_internal.h"
#include "fftopk_key.h"
#include "fftopk_rows.cuh"
#include "fftopk_tcgen05.cuh"

namespace fftopk {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kBins = 2048, kRounds = 3;
constexpr int kMaxCluster = 8;
constexpr int kMaxKeys = 16 * 1024;       // of a CTA in shared memory: two CTAs per SM
constexpr int kMaxSpan = 256 * 1024;      // positions of a CTA
constexpr int kMoveThreads = 128;

struct EvictParams {
  fftopk_evict a;
  int32_t bound;  // positions that the table and the weights reach
  int32_t words;  // of 32 positions of a CTA
  int32_t moves;  // evict_move_kernel follows
  FastDiv page;
  uint32_t* status;
};

__device__ __forceinline__ int digit_shift(int round) { return round == 0 ? 21 : round == 1 ? 10 : 0; }

// fftopk_key_from_bits of a weight: the sum turns -0 into 0
__device__ __forceinline__ uint32_t key_of(float w) {
  const uint32_t bits = __float_as_uint(w + 0.f), key = bits ^ ((uint32_t)((int32_t)bits >> 31) | 0x80000000u);
  return w != w ? 0xffffffffu : key;
}

struct alignas(16) Word {  // 32 positions: those that stay for certain, those in question, and how many of either lie in front of them
  uint32_t sure, tie, sure_before, tie_before;
};
struct SelectSmem {
  uint32_t hist[kRounds][kBins];
  alignas(16) uint32_t warp_total[kWarps];
  alignas(16) uint64_t warp_stay[kWarps];
  uint32_t found[4];  // bin, count above it, count in it
  uint64_t stay;      // of this CTA: rows that stay for certain, and, in the upper half, rows of the smallest weight that stays
};

__device__ __forceinline__ uint64_t scan64(uint64_t x, int lane) {
#pragma unroll
  for (int i = 1; i < 32; i <<= 1) {
    const uint64_t y = __shfl_up_sync(kAll, x, i);
    if (lane >= i) x += y;
  }
  return x;
}
// Where the count from the top of the round's histogram - summed over the cluster - reaches `need`: the bin, the count above it, the count in it
__device__ __forceinline__ void pick(SelectSmem& sm, cg::cluster_group& cluster, int ctas, int round, uint32_t need) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int kPer = kBins / kThreads;  // bins a thread, the highest first
  static_assert(kPer == 4, "a thread's bins are one load");
  const int bin0 = kBins - kPer - kPer * tid;
  uint32_t v[kPer];
  if (ctas > 1) {
    cluster.sync();
    uint4 x[kMaxCluster];  // (every CTA's bins are asked for before any are used)
    const uint32_t at = smem_u32(&sm.hist[round][bin0]);
#pragma unroll
    for (int c = 0; c < kMaxCluster; ++c) {
      x[c] = make_uint4(0u, 0u, 0u, 0u);
      if (c < ctas) {
        const float4 r = lds_cluster4(shared_of(at, c));
        x[c] = make_uint4(__float_as_uint(r.x), __float_as_uint(r.y), __float_as_uint(r.z), __float_as_uint(r.w));
      }
    }
    v[0] = v[1] = v[2] = v[3] = 0u;
#pragma unroll
    for (int c = 0; c < kMaxCluster; ++c) v[0] += x[c].w, v[1] += x[c].z, v[2] += x[c].y, v[3] += x[c].x;
  } else {
    __syncthreads();
    const uint4 x = *reinterpret_cast<const uint4*>(&sm.hist[round][bin0]);
    v[0] = x.w, v[1] = x.z, v[2] = x.y, v[3] = x.x;
  }
  uint32_t s = 0;
#pragma unroll
  for (int e = 0; e < kPer; ++e) s += v[e];
  uint32_t upto = s;
#pragma unroll
  for (int i = 1; i < 32; i <<= 1) {
    const uint32_t y = __shfl_up_sync(kAll, upto, i);
    if (lane >= i) upto += y;
  }
  if (lane == 31) sm.warp_total[warp] = upto;
  __syncthreads();
  uint32_t above = upto - s;
#pragma unroll
  for (int i = 0; i < kWarps; i += 4) {
    const uint4 x = *reinterpret_cast<const uint4*>(&sm.warp_total[i]);
    above += (i < warp ? x.x : 0u) + (i + 1 < warp ? x.y : 0u) + (i + 2 < warp ? x.z : 0u) + (i + 3 < warp ? x.w : 0u);
  }
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    if (above < need && above + v[e] >= need) sm.found[0] = (uint32_t)(bin0 + kPer - 1 - e), sm.found[1] = above, sm.found[2] = v[e];
    above += v[e];
  }
  __syncthreads();
}

// What bounds it, beside a dozen waits for the slowest thread, is integer instructions: some 20 cycles of an SM for 32 positions in each of three passes. Its
// loops are not unrolled (17 positions a thread in registers, unrolled: 16 us for 8 units of 4,608 positions where this takes 9.6).
// kHeld: shared memory has room for the keys of all of a CTA's positions
template <bool kHeld>
__global__ void __launch_bounds__(kThreads) evict_select_kernel(const __grid_constant__ EvictParams p) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  SelectSmem& sm = *reinterpret_cast<SelectSmem*>(smem_raw);
  Word* const words = reinterpret_cast<Word*>(smem_raw + sizeof(SelectSmem));
  uint32_t* const held = reinterpret_cast<uint32_t*>(words + p.words);  // kHeld: the CTA's weights, as bits
  // (only where a kernel of this call follows, which waits: another one's inputs may be this one's results)
  if (p.moves) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t unit = blockIdx.x / (uint32_t)ctas;
  const int64_t b = unit / (uint32_t)p.a.heads;
  const int h = (int)(unit - (uint32_t)b * (uint32_t)p.a.heads);
  const int32_t length = p.a.lengths[b], budget = p.a.budget;
#pragma unroll 1
  for (int i = tid; i < kRounds * kBins / 4; i += kThreads) reinterpret_cast<uint4*>(&sm.hist[0][0])[i] = make_uint4(0u, 0u, 0u, 0u);
  const int32_t n = min(max(length, 0), p.bound), left = min(n, budget);
  if (rank == 0 && h == 0 && tid == 0) {
    p.a.new_lengths[b] = left;
    if (length > p.bound && p.status) atomicOr(p.status, (uint32_t)FFTOPK_ST_BAD_INDEX);
  }
  const float* w = p.a.weight + b * p.a.w_seq + (int64_t)h * p.a.w_head;
  float* const wo = p.a.weight_out + b * p.a.wo_seq + (int64_t)h * p.a.wo_head;
  int32_t* const kept = p.a.kept + ((int64_t)b * p.a.heads + h) * budget;
  const bool evicts = n > budget;
  const int32_t first = p.a.sinks, last = n - p.a.recent;  // (where rows are dropped: sinks + recent <= budget < n)
  const int32_t each = ((n + ctas - 1) / ctas + 31) & ~31;
  const int32_t from = min(n, rank * each), span = min(n - from, each);
  const int32_t lo = first - from, hi = min(last - from, span);  // the rows between, counted from the CTA's first
  w += from;
  if (kHeld && evicts) {
    const int32_t fours = (reinterpret_cast<uintptr_t>(w) & 15u) == 0 ? span / 4 : 0;
#pragma unroll 1
    for (int32_t i = tid; i < fours; i += kThreads) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(held + 4 * i)), "l"(w + 4 * i) : "memory");
#pragma unroll 1
    for (int32_t i = 4 * fours + tid; i < span; i += kThreads) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(held + i)), "l"(w + i) : "memory");
  }
  // behind what stays: no rows, and weights that start at zero
  const int all = ctas * kThreads, me = rank * kThreads + tid;
#pragma unroll 1
  for (int64_t j = (int64_t)left + me; j < budget; j += all) kept[j] = -1;
  // (by fours where they begin on 16 bytes)
  const int64_t odd = min(p.a.weight_cols - left, (int64_t)((0u - (uint32_t)(reinterpret_cast<uintptr_t>(wo + left) >> 2)) & 3u));
  const int64_t fours = (p.a.weight_cols - left - odd) / 4;
#pragma unroll 1
  for (int64_t j = me; j < fours; j += all) reinterpret_cast<float4*>(wo + left + odd)[j] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int64_t j = me; j < p.a.weight_cols - left - 4 * fours; j += all) wo[j < odd ? left + j : left + 4 * fours + j] = 0.f;
  if (!evicts) {
#pragma unroll 1
    for (int32_t i = tid; i < span; i += kThreads) kept[from + i] = from + i, wo[from + i] = w[i];
    return;  // (the whole cluster)
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  auto key_at = [&](int32_t i) { return key_of(kHeld ? __uint_as_float(held[i]) : w[i]); };
  // the bits of word `word` that are positions a .. z - 1
  auto bits_of = [](int32_t word, int32_t a, int32_t z) {
    a = min(max(a - word * 32, 0), 32), z = min(max(z - word * 32, 0), 32);
    return a < z ? (0xffffffffu >> (32 - (z - a))) << a : 0u;
  };
  // of the rows between those stay whose key, as far as `mask`, is above `edge`, and the first `ties` of those at it
  uint32_t need = (uint32_t)(budget - first - p.a.recent);  // of the rows between
  uint32_t edge = 0, mask = 0, ties = 0;
  if (need == 0) edge = mask = 0xffffffffu;  // (none)
  const int32_t n_words = (span + 31) / 32;
#pragma unroll 1
  for (int round = 0;; ++round) {
    const int shift = digit_shift(round);
    const uint32_t top = round < 2 ? 0x7ffu : 0x3ffu;
    if (round == 0) {
#pragma unroll 1
      for (int32_t i0 = warp * 32; i0 < span; i0 += kThreads) {
        const int32_t i = i0 + lane;
        if (i0 >= lo && i0 + 32 <= hi) {
          const uint32_t digit = key_at(i) >> 21;
          if (__reduce_min_sync(kAll, digit) != __reduce_max_sync(kAll, digit))
            atomicAdd(&sm.hist[0][digit], 1u);
          else if (lane == 0)  // (copies of one weight: one addition for the warp)
            atomicAdd(&sm.hist[0][digit], 32u);
        } else if (i >= lo && i < hi) {
          atomicAdd(&sm.hist[0][key_at(i) >> 21], 1u);
        }
      }
    }
    if (need > 0) {
      if (round > 0) {  // the other rounds look at what is in question only, a thread a word
#pragma unroll 1
        for (int32_t word = tid; word < n_words; word += kThreads) {
          uint32_t t = words[word].tie, digit = 0, count = 0;  // (runs of one digit are added at once)
#pragma unroll 1
          while (t != 0u) {
            const uint32_t key = key_at(word * 32 + __ffs((int)t) - 1);
            t &= t - 1u;
            if ((key & mask) != edge) continue;
            const uint32_t d = key >> shift & top;
            if (d != digit && count > 0) atomicAdd(&sm.hist[round][digit], count), count = 0;
            digit = d, ++count;
          }
          if (count > 0) atomicAdd(&sm.hist[round][digit], count);
        }
      }
      pick(sm, cluster, ctas, round, need);
      edge |= sm.found[0] << shift;
      mask |= top << shift;
      need -= sm.found[1];
      ties = need;
    }
    const bool done = need == 0 || sm.found[2] == need || round + 1 == kRounds;  // (the bin stays whole, or is one weight)
    if (round == 0) {
#pragma unroll 4
      for (int32_t word = warp; word < n_words; word += kWarps) {
        const int32_t i = word * 32 + lane;
        const uint32_t key = (i < span ? key_at(i) : 0u) & mask;
        uint32_t above = __ballot_sync(kAll, key > edge), at = __ballot_sync(kAll, key == edge);
        if (word * 32 < lo || word * 32 + 32 > hi) {
          const uint32_t between = bits_of(word, lo, hi);
          above = bits_of(word, 0, span) & (above | ~between), at &= between;
        }
        if (lane == 0) *reinterpret_cast<uint2*>(&words[word]) = make_uint2(above, at);
      }
      __syncthreads();
    }
    if (done) break;
  }
  // what was in question is settled, and counted over words, warps and CTAs
  uint64_t before = 0;
#pragma unroll 1
  for (int32_t w0 = 0; w0 < n_words; w0 += kThreads) {
    const int32_t word = w0 + tid;
    uint32_t s = 0, t = 0;
    if (word < n_words) {
      s = words[word].sure;
#pragma unroll 1
      for (uint32_t q = words[word].tie; q != 0u; q &= q - 1u) {
        const uint32_t key = key_at(word * 32 + __ffs((int)q) - 1) & mask;
        if (key > edge) s |= q & -q;
        if (key == edge) t |= q & -q;
      }
    }
    const uint64_t mine = (uint64_t)__popc(t) << 32 | (uint32_t)__popc(s), upto = scan64(mine, lane);
    if (lane == 31) sm.warp_stay[warp] = upto;
    __syncthreads();
    uint64_t sum = before + upto - mine;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      const uint64_t x = sm.warp_stay[i];
      sum += i < warp ? x : 0;
      before += x;
    }
    if (word < n_words) *reinterpret_cast<uint4*>(&words[word]) = make_uint4(s, t, (uint32_t)sum, (uint32_t)(sum >> 32));
    __syncthreads();
  }
  uint32_t sures = 0, tied = 0;  // in front of this CTA
  if (ctas > 1) {
    if (tid == 0) sm.stay = before;
    cluster.sync();
#pragma unroll 1
    for (int c = 0; c < rank; ++c) {
      const uint64_t x = *cluster.map_shared_rank(&sm.stay, c);
      sures += (uint32_t)x, tied += (uint32_t)(x >> 32);
    }
  }
#pragma unroll 2
  for (int32_t word = warp; word < n_words; word += kWarps) {
    const uint4 q = *reinterpret_cast<const uint4*>(&words[word]);  // (a Word)
    bool stays = (q.x & 1u << lane) != 0u;
    const uint32_t below = (1u << lane) - 1u;
    uint32_t at = sures + q.z + (uint32_t)__popc(q.x & below), tie_rank = tied + q.w;
    if (q.y != 0u) {
      tie_rank += (uint32_t)__popc(q.y & below);
      stays = stays || ((q.y & 1u << lane) != 0u && tie_rank < ties);
    }
    at += min(tie_rank, ties);
    if (stays && at < (uint32_t)left) {
      const int32_t i = word * 32 + lane;
      kept[at] = from + i;
      wo[at] = kHeld ? __uint_as_float(held[i]) : w[i];
    }
  }
  if (ctas > 1) cluster.sync();  // (nobody leaves while its memory is read)
}

// P: what a piece of a row is copied as. Two rows of k and of v a lane on their way at a time: warps beside each other keep memory busier than
// rows in front of one another (524,288 rows of e4m3, eviction as a whole: 70 us; four and eight rows 78 and 80).
template <typename P>
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const __grid_constant__ EvictParams p, int pieces, int lanes, int groups, int rows) {
  constexpr int kAhead = 2;
  const int lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * (kMoveThreads / 32) + (threadIdx.x >> 5);
  // (`rows` rows, up to 32, of a key head; the key heads of the same places are neighbours)
  const int64_t rest = item / p.a.heads;
  const int h = (int)(item - rest * p.a.heads);
  const int64_t b = rest / groups;
  const int32_t j0 = (int32_t)(rest - b * groups) * rows, j = j0 + lane;
  // where they go is known before the kernel in front is through
  const int32_t left = b < p.a.seqs ? min(min(max(p.a.lengths[b], 0), p.bound), p.a.budget) : 0;
  const bool mine = lane < rows && j < left;
  int64_t dst = -1;
  if (mine) {
    const uint32_t m = p.page.div((uint32_t)j);
    const int32_t to = p.a.to_table[b * p.a.to_row + m];
    if (to >= 0) dst = (int64_t)to * p.page.d + ((uint32_t)j - m * p.page.d);
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");  // (by every CTA: this kernel does not end before the one in front)
  if (j0 >= left) return;
  int src_row = -1, dst_row = -1;
  if (mine) {
    const uint32_t pos = (uint32_t)p.a.kept[(b * p.a.heads + h) * p.a.budget + j], n = p.page.div(pos);
    const int32_t from = p.a.page_table[b * p.a.table_row + n];
    const int64_t src = (int64_t)from * p.page.d + (pos - n * p.page.d);
    if (from < 0 || src >= p.a.slots || dst < 0 || dst >= p.a.slots) {
      if (p.status) atomicOr(p.status, (uint32_t)FFTOPK_ST_BAD_INDEX);
    } else {
      src_row = (int)src, dst_row = (int)dst;
    }
  }
  if (p.a.k_scale != nullptr && dst_row >= 0) {
    const float* ks = p.a.k_scale + (int64_t)h * p.a.ks_head;
    const float* vs = p.a.v_scale + (int64_t)h * p.a.vs_head;
    const float x = ks[src_row * p.a.ks_slot], y = vs[src_row * p.a.vs_slot];
    p.a.k_scale[dst_row * p.a.ks_slot + (int64_t)h * p.a.ks_head] = x;
    p.a.v_scale[dst_row * p.a.vs_slot + (int64_t)h * p.a.vs_head] = y;
  }
  const int es = p.a.elem_bytes, sub = lane / lanes, piece = lane - sub * lanes, once = 32 / lanes;
  char* const k = static_cast<char*>(p.a.k) + (int64_t)h * p.a.k_head * es;
  char* const v = static_cast<char*>(p.a.v) + (int64_t)h * p.a.v_head * es;
  const uint32_t kstep = (uint32_t)(p.a.k_slot * es), vstep = (uint32_t)(p.a.v_slot * es);
  for (int at = 0; at < rows; at += once * kAhead) {
    int from[kAhead], to[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int row = at + i * once + sub;
      from[i] = __shfl_sync(kAll, src_row, row & 31);
      to[i] = __shfl_sync(kAll, dst_row, row & 31);
      if (row >= rows) to[i] = -1;
    }
    for (int c = piece; c < pieces; c += lanes) {
      const uint32_t off = (uint32_t)c * (uint32_t)sizeof(P);
      P x[kAhead], y[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (to[i] >= 0) {
          x[i] = *reinterpret_cast<const P*>(k + (uint64_t)(uint32_t)from[i] * kstep + off);
          y[i] = *reinterpret_cast<const P*>(v + (uint64_t)(uint32_t)from[i] * vstep + off);
        }
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (to[i] >= 0) {
          *reinterpret_cast<P*>(k + (uint64_t)(uint32_t)to[i] * kstep + off) = x[i];
          *reinterpret_cast<P*>(v + (uint64_t)(uint32_t)to[i] * vstep + off) = y[i];
        }
      }
    }
  }
}

DeviceOnce g_evict_once[kMaxDevices];
int g_evict_sms[kMaxDevices];
int evict_setup(int& sms) {
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e);
  if (dev < 0 || dev >= kMaxDevices) return FFTOPK_EDEVICE;
  const int rc = g_evict_once[dev].run([&] {
    cudaError_t e2 = cudaDeviceGetAttribute(&g_evict_sms[dev], cudaDevAttrMultiProcessorCount, dev);
    const int words = (int)(sizeof(SelectSmem) + kMaxSpan / 32 * sizeof(Word));
    if (e2 == cudaSuccess) e2 = cudaFuncSetAttribute(evict_select_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, words);
    const int held = (int)(sizeof(SelectSmem) + kMaxKeys / 32 * sizeof(Word) + kMaxKeys * 4);
    if (e2 == cudaSuccess) e2 = cudaFuncSetAttribute(evict_select_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, held);
    return e2 == cudaSuccess ? 0 : cuda_fail(e2);
  });
  sms = g_evict_sms[dev];
  return rc;
}

bool on(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(bytes - 1)) == 0; }
// rows of pieces of `piece` bytes, whatever their slot and head; the stride of a lone one says nothing
bool rows_on(const void* p, int64_t slots, int64_t slot, int64_t heads, int64_t head, int es, int piece) {
  return on(p, piece) && (slots <= 1 || slot * es % piece == 0) && (heads <= 1 || head * es % piece == 0);
}

template <typename P>
cudaError_t launch_move(const EvictParams& p, int row_bytes, int sms, cudaStream_t stream) {
  const int pieces = row_bytes / (int)sizeof(P);
  int rows = 32, groups = 0;
  // fewer rows a warp where 32 leave warps without any (32,768 rows: 12.5 us with 8 a warp, the call, and 13.5 with 32; 524,288 rows: 78 and 70)
  while (rows > 8 && p.a.seqs * p.a.heads * ((p.a.budget + rows - 1) / rows) < (int64_t)sms * 32) rows /= 2;
  groups = (p.a.budget + rows - 1) / rows;
  int lanes = 1;
  while (lanes < 32 && lanes < pieces) lanes *= 2;
  const int64_t warps = p.a.seqs * p.a.heads * groups;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((warps + kMoveThreads / 32 - 1) / (kMoveThreads / 32)), 1, 1);
  cfg.blockDim = dim3(kMoveThreads, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, evict_move_kernel<P>, p, pieces, lanes, groups, rows);
}

}  // namespace
}  // namespace fftopk

using namespace fftopk;

extern "C" int fftopk_cache_evict(const fftopk_evict* a, uint32_t* status, void* cuda_stream) {
  if (a == nullptr) return FFTOPK_EINVAL;
  if (a->seqs < 0 || a->heads < 0 || a->slots < 0 || a->pages < 0 || a->to_pages < 0 || a->page_size < 1 || a->budget < 0 || a->recent < 0 ||
      a->sinks < 0 || a->weight_cols < 0)
    return FFTOPK_EINVAL;
  if ((int64_t)a->sinks + a->recent > a->budget) return FFTOPK_EINVAL;
  if (a->elem_bytes != 1 && a->elem_bytes != 2) return FFTOPK_EINVAL;
  if (a->D < 8 || a->D > 256 || (a->D & 7) != 0) return FFTOPK_ERANGE;
  if (a->seqs == 0 || a->heads == 0) return FFTOPK_OK;
  if ((a->k_scale != nullptr) != (a->v_scale != nullptr)) return FFTOPK_EINVAL;
  if (!a->lengths || !a->new_lengths || (a->pages > 0 && !a->page_table) || (a->budget > 0 && (!a->to_table || !a->kept))) return FFTOPK_EINVAL;
  if (a->weight_cols > 0 && (!a->weight || !a->weight_out)) return FFTOPK_EINVAL;
  if (a->slots > 0 && (!a->k || !a->v)) return FFTOPK_EINVAL;
  if (!on(a->k, a->elem_bytes) || !on(a->v, a->elem_bytes) || !on(a->k_scale, 4) || !on(a->v_scale, 4) || !on(a->weight, 4) || !on(a->weight_out, 4) ||
      !on(a->page_table, 4) || !on(a->to_table, 4) || !on(a->lengths, 4) || !on(a->new_lengths, 4) || !on(a->kept, 4))
    return FFTOPK_EINVAL;
  const int64_t bound = (int64_t)a->pages * a->page_size < a->weight_cols ? (int64_t)a->pages * a->page_size : a->weight_cols;
  if (a->slots > 0x7fffffff || a->seqs > 0x7fffffff / a->heads || bound > kMaxCluster * kMaxSpan || (int64_t)a->to_pages * a->page_size < a->budget ||
      a->budget > 0x7ffff000)
    return FFTOPK_ERANGE;
  // (rows are found by the product of two 32-bit numbers; a lone slot's stride says nothing)
  if (a->slots > 1 && (a->k_slot < 0 || a->v_slot < 0 || a->k_slot > 0xffffffffll / a->elem_bytes || a->v_slot > 0xffffffffll / a->elem_bytes))
    return FFTOPK_ERANGE;
  const int64_t units = a->seqs * a->heads;
  if (units * ((a->budget + 7) / 8) > 0x7fffffff) return FFTOPK_ERANGE;
  // (rows written twice would hold whichever came last; lengths are read while new_lengths are written)
  if (!rows_apart(a->seqs, a->wo_seq, a->heads, a->wo_head, a->weight_cols) || !rows_apart(a->slots, a->k_slot, a->heads, a->k_head, a->D) ||
      !rows_apart(a->slots, a->v_slot, a->heads, a->v_head, a->D) || a->lengths == a->new_lengths)
    return FFTOPK_EINVAL;
  if (a->k_scale != nullptr && (!rows_apart(a->slots, a->ks_slot, a->heads, a->ks_head, 1) || !rows_apart(a->slots, a->vs_slot, a->heads, a->vs_head, 1)))
    return FFTOPK_EINVAL;
  // (a unit's weights are read while another one's are written)
  if (rows_meet(a->weight, a->w_seq, a->w_head, a->weight_out, a->wo_seq, a->wo_head, a->seqs, a->heads, a->weight_cols, 4)) return FFTOPK_EINVAL;
  int sms = 0;
  const int rc = evict_setup(sms);
  if (rc) return rc;
  EvictParams p;
  memset(&p, 0, sizeof(p));
  p.a = *a;
  p.bound = (int32_t)bound;
  p.moves = a->budget > 0 && bound > 0;
  p.page = FastDiv((uint32_t)a->page_size);
  p.status = status;
  // CTAs a unit: as many as fit the device at once, of 4,096 positions at least; and enough for what a CTA can hold
  int ctas = 1;
  while (ctas < kMaxCluster && ((units * ctas * 2 <= 2 * (int64_t)sms && bound / ctas > 8192) || bound > (int64_t)ctas * kMaxSpan)) ctas *= 2;
  if (units * ctas > 0x7fffffff) return FFTOPK_ERANGE;
  const int64_t each = ((bound + ctas - 1) / ctas + 31) & ~(int64_t)31;
  const bool held = each <= kMaxKeys;
  p.words = (int32_t)(each / 32);
  cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(units * ctas), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = sizeof(SelectSmem) + (size_t)p.words * sizeof(Word) + (held ? (size_t)each * 4 : 0);
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)ctas;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const auto select = held ? evict_select_kernel<true> : evict_select_kernel<false>;
  cudaError_t e = cudaLaunchKernelEx(&cfg, select, p);
  if (e == cudaSuccess && p.moves) {
    const int bytes = a->D * a->elem_bytes;
    int piece = 16;
    while (piece > a->elem_bytes && (bytes % piece != 0 || !rows_on(a->k, a->slots, a->k_slot, a->heads, a->k_head, a->elem_bytes, piece) ||
                                     !rows_on(a->v, a->slots, a->v_slot, a->heads, a->v_head, a->elem_bytes, piece)))
      piece /= 2;
    e = piece == 16  ? launch_move<uint4>(p, bytes, sms, stream)
        : piece == 8 ? launch_move<uint2>(p, bytes, sms, stream)
        : piece == 4 ? launch_move<uint32_t>(p, bytes, sms, stream)
        : piece == 2 ? launch_move<uint16_t>(p, bytes, sms, stream)
                     : launch_move<uint8_t>(p, bytes, sms, stream);
  }
  return e == cudaSuccess ? FFTOPK_OK : cuda_fail(e);
}
