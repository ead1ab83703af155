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
#include <stdlib.h>

#include "../../include/fftopk.h"
#include "fftopk_host.h"
#include "fftopk_internal.h"
#include "fftopk_key.h"
#include "fftopk_rows.cuh"

namespace fftopk {
namespace {

namespace cg = cooperative_groups;

constexpr unsigned kAll = 0xffffffffu;
constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kBins = 2048, kRounds = 3;
constexpr int kMaxCluster = 8;
constexpr int kBatch = 8;  // weights a thread has on their way
constexpr int kMaxKeys = 16 * 1024;       // of a CTA in shared memory: two CTAs per SM
constexpr int kMaxSpan = 256 * 1024;      // positions of a CTA
constexpr int kMoveThreads = 128;

struct EvictParams {
  fftopk_evict a;
  int32_t bound;  // positions that the table and the weights reach
  int32_t keys;   // of a CTA that shared memory has room for
  int32_t words;  // of 32 positions of a CTA
  int32_t moves;  // evict_move_kernel follows
  FastDiv page;
  uint32_t* status;
};

__device__ __forceinline__ int digit_shift(int round) { return round == 0 ? 21 : round == 1 ? 10 : 0; }

struct Word {  // 32 positions: those that stay for certain, those in question, and how many of either lie in front of them
  uint32_t sure, tie, sure_before, tie_before;
};
struct SelectSmem {
  uint32_t hist[kRounds][kBins];
  uint32_t warp_total[kWarps];
  uint32_t found[3];  // bin, count above it, count in it
  uint64_t warp_stay[kWarps];
  uint64_t stay;      // of this CTA: rows that stay for certain, and, in the upper half, rows of the smallest weight that stays
};

// Where the count from the top of the round's histogram - summed over the cluster - reaches `need`: the bin, the count above it, the count in it
__device__ __forceinline__ void pick(SelectSmem& sm, cg::cluster_group& cluster, int ctas, int round, uint32_t need) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (ctas > 1)
    cluster.sync();
  else
    __syncthreads();
  uint32_t v[4] = {0u, 0u, 0u, 0u};  // four bins a thread, the highest first
  const int bin0 = kBins - 4 - 4 * tid;
  for (int c = 0; c < ctas; ++c) {
    const uint4 x = *reinterpret_cast<const uint4*>(cluster.map_shared_rank(&sm.hist[round][bin0], c));
    v[0] += x.w, v[1] += x.z, v[2] += x.y, v[3] += x.x;
  }
  const uint32_t s = v[0] + v[1] + v[2] + v[3];
  uint32_t upto = s;
#pragma unroll
  for (int i = 1; i < 32; i <<= 1) {
    const uint32_t y = __shfl_up_sync(kAll, upto, i);
    if (lane >= i) upto += y;
  }
  if (lane == 31) sm.warp_total[warp] = upto;
  __syncthreads();
  uint32_t above = upto - s;
  for (int i = 0; i < warp; ++i) above += sm.warp_total[i];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (above < need && above + v[e] >= need) sm.found[0] = (uint32_t)(bin0 + 3 - e), sm.found[1] = above, sm.found[2] = v[e];
    above += v[e];
  }
  __syncthreads();
}

__global__ void __launch_bounds__(kThreads) evict_select_kernel(const __grid_constant__ EvictParams p) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  SelectSmem& sm = *reinterpret_cast<SelectSmem*>(smem_raw);
  Word* const words = reinterpret_cast<Word*>(smem_raw + sizeof(SelectSmem));
  uint32_t* const held = reinterpret_cast<uint32_t*>(words + p.words);  // the CTA's weights, as bits
  // (only where a kernel of this call follows, which waits: another one's inputs may be this one's results)
  if (p.moves) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t unit = blockIdx.x / (uint32_t)ctas;
  const int64_t b = unit / (uint32_t)p.a.heads;
  const int h = (int)(unit - (uint32_t)b * (uint32_t)p.a.heads);
  const int32_t length = p.a.lengths[b], n = min(max(length, 0), p.bound), budget = p.a.budget;
  const int32_t left = min(n, budget);
  if (rank == 0 && h == 0 && tid == 0) {
    p.a.new_lengths[b] = left;
    if (length > p.bound && p.status) atomicOr(p.status, (uint32_t)FFTOPK_ST_BAD_INDEX);
  }
  const float* w = p.a.weight + b * p.a.w_seq + (int64_t)h * p.a.w_head;
  float* wo = p.a.weight_out + b * p.a.wo_seq + (int64_t)h * p.a.wo_head;
  int32_t* kept = p.a.kept + ((int64_t)b * p.a.heads + h) * budget;
  // behind what stays: no rows, and weights that start at zero
  const int all = ctas * kThreads, me = rank * kThreads + tid;
  for (int64_t j = (int64_t)left + me; j < budget; j += all) kept[j] = -1;
  for (int64_t j = (int64_t)left + me; j < p.a.weight_cols; j += all) wo[j] = 0.f;
  if (n <= budget) {
    for (int32_t j = me; j < n; j += all) kept[j] = j, wo[j] = w[j];
    return;  // (the whole cluster)
  }
  const int32_t first = p.a.sinks, last = n - p.a.recent;  // (sinks + recent <= budget < n)
  uint32_t need = (uint32_t)(budget - first - p.a.recent);  // of the rows between
  const int32_t each = ((n + ctas - 1) / ctas + 31) & ~31;
  const int32_t from = min(n, rank * each), span = min(n - from, each), there = min(span, p.keys);
  const int32_t lo = first - from, hi = last - from;  // the rows between, counted from the CTA's first
  w += from;
  auto bits_at = [&](int32_t i) { return i < there ? held[i] : __float_as_uint(w[i]); };
  auto key_at = [&](int32_t i) { return fftopk_key_from_bits(bits_at(i)); };

  for (int i = tid; i < kRounds * kBins / 4; i += kThreads) reinterpret_cast<uint4*>(&sm.hist[0][0])[i] = make_uint4(0u, 0u, 0u, 0u);
  __syncthreads();
  // round 0 as the weights come in
  for (int32_t i0 = tid; i0 - lane < span; i0 += kThreads * kBatch) {
    float x[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) x[u] = i0 + u * kThreads < span ? w[i0 + u * kThreads] : 0.f;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int32_t i = i0 + u * kThreads;
      const uint32_t bits = __float_as_uint(x[u]);
      if (i < there) held[i] = bits;
      const bool counts = i < span && i >= lo && i < hi;
      const uint32_t digit = fftopk_key_from_bits(bits) >> 21;
      const unsigned who = __ballot_sync(kAll, counts);
      if (who == 0u) continue;
      const uint32_t lead = __shfl_sync(kAll, digit, __ffs((int)who) - 1);
      if (__all_sync(kAll, !counts || digit == lead)) {  // (copies of one weight: one addition for the warp)
        if (lane == 0) atomicAdd(&sm.hist[0][lead], (uint32_t)__popc(who));
      } else if (counts) {
        atomicAdd(&sm.hist[0][digit], 1u);
      }
    }
  }
  // of the rows between those stay whose key, as far as `mask`, is above `edge`, and the first `ties` of those at it
  uint32_t edge = 0xffffffffu, mask = 0xffffffffu, ties = 0;  // (none)
  bool whole = true;  // the bin stays whole, or is one weight
  if (need > 0) {
    pick(sm, cluster, ctas, 0, need);
    edge = sm.found[0] << 21, mask = 0x7ffu << 21;
    need -= sm.found[1];
    ties = need;
    whole = sm.found[2] == need;
  }
  const int32_t n_words = (span + 31) / 32;
  for (int32_t word = warp; word < n_words; word += kWarps) {
    const int32_t i = word * 32 + lane;
    const bool in = i < span, between = in && i >= lo && i < hi;
    const uint32_t key = between ? key_at(i) & mask : 0u;
    const unsigned s = __ballot_sync(kAll, in && (!between || key > edge)), t = __ballot_sync(kAll, between && key == edge);
    if (lane == 0) words[word].sure = s, words[word].tie = t;
  }
  __syncthreads();
  // the other rounds look at what is in question only, a thread a word
  for (int round = 1; round < kRounds && !whole; ++round) {
    const int shift = digit_shift(round);
    const uint32_t top = round == 1 ? 0x7ffu : 0x3ffu;
    for (int32_t word = tid; word < n_words; word += kThreads) {
      uint32_t t = words[word].tie, digit = 0, count = 0;  // (runs of one digit are added at once)
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
    pick(sm, cluster, ctas, round, need);
    edge |= sm.found[0] << shift;
    mask |= top << shift;
    need -= sm.found[1];
    ties = need;
    whole = sm.found[2] == need;
  }
  // what was in question is settled, and counted over words, warps and CTAs
  uint64_t before = 0;
  for (int32_t w0 = 0; w0 < n_words; w0 += kThreads) {
    const int32_t word = w0 + tid;
    uint32_t s = 0, t = 0;
    if (word < n_words) {
      s = words[word].sure;
      for (uint32_t q = words[word].tie; q != 0u; q &= q - 1u) {
        const uint32_t key = key_at(word * 32 + __ffs((int)q) - 1) & mask;
        if (key > edge) s |= q & -q;
        if (key == edge) t |= q & -q;
      }
    }
    const uint64_t mine = (uint64_t)__popc(t) << 32 | (uint32_t)__popc(s);
    uint64_t upto = mine;
#pragma unroll
    for (int i = 1; i < 32; i <<= 1) {
      const uint64_t y = __shfl_up_sync(kAll, upto, i);
      if (lane >= i) upto += y;
    }
    if (lane == 31) sm.warp_stay[warp] = upto;
    __syncthreads();
    uint64_t sum = before, total = before;
    for (int i = 0; i < kWarps; ++i) {
      if (i < warp) sum += sm.warp_stay[i];
      total += sm.warp_stay[i];
    }
    sum += upto - mine;
    if (word < n_words) words[word] = Word{s, t, (uint32_t)sum, (uint32_t)(sum >> 32)};
    before = total;
    __syncthreads();
  }
  uint32_t sures = 0, tied = 0;  // in front of this CTA
  if (ctas > 1) {
    if (tid == 0) sm.stay = before;
    cluster.sync();
    for (int c = 0; c < rank; ++c) {
      const uint64_t x = *cluster.map_shared_rank(&sm.stay, c);
      sures += (uint32_t)x, tied += (uint32_t)(x >> 32);
    }
  }
  for (int32_t word = warp; word < n_words; word += kWarps) {
    const Word q = words[word];
    const uint32_t below = (1u << lane) - 1u, tie_rank = tied + q.tie_before + (uint32_t)__popc(q.tie & below);
    if ((q.sure >> lane & 1u) || ((q.tie >> lane & 1u) && tie_rank < ties)) {
      const uint32_t at = sures + q.sure_before + (uint32_t)__popc(q.sure & below) + min(tie_rank, ties);
      const int32_t i = word * 32 + lane;
      if (at < (uint32_t)left) kept[at] = from + i, wo[at] = __uint_as_float(bits_at(i));
    }
  }
  if (ctas > 1) cluster.sync();  // (nobody leaves while its memory is read)
}

// P: what a piece of a row is copied as
template <typename P>
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const __grid_constant__ EvictParams p, int pieces, int lanes, int groups, int rows) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * (kMoveThreads / 32) + (threadIdx.x >> 5);
  // (`rows` rows, up to 32, of a key head; the key heads of the same places are neighbours)
  const int64_t rest = item / p.a.heads;
  const int h = (int)(item - rest * p.a.heads);
  const int64_t b = rest / groups;
  const int32_t j0 = (int32_t)(rest - b * groups) * rows;
  if (b >= p.a.seqs) return;
  const int32_t left = p.a.new_lengths[b];
  if (j0 >= left) return;
  int64_t src = -1, dst = -1;
  const int32_t j = j0 + lane;
  if (lane < rows && j < left) {
    const uint32_t pos = (uint32_t)p.a.kept[(b * p.a.heads + h) * p.a.budget + j];
    const uint32_t n = p.page.div(pos), m = p.page.div((uint32_t)j);
    const int32_t from = p.a.page_table[b * p.a.table_row + n], to = p.a.to_table[b * p.a.to_row + m];
    src = (int64_t)from * p.page.d + (pos - n * p.page.d);
    dst = (int64_t)to * p.page.d + ((uint32_t)j - m * p.page.d);
    if (from < 0 || to < 0 || src >= p.a.slots || dst >= p.a.slots) {
      src = dst = -1;
      if (p.status) atomicOr(p.status, (uint32_t)FFTOPK_ST_BAD_INDEX);
    } else if (p.a.k_scale != nullptr) {
      p.a.k_scale[dst * p.a.ks_slot + (int64_t)h * p.a.ks_head] = p.a.k_scale[src * p.a.ks_slot + (int64_t)h * p.a.ks_head];
      p.a.v_scale[dst * p.a.vs_slot + (int64_t)h * p.a.vs_head] = p.a.v_scale[src * p.a.vs_slot + (int64_t)h * p.a.vs_head];
    }
  }
  const int es = p.a.elem_bytes;
  char* const k = static_cast<char*>(p.a.k) + (int64_t)h * p.a.k_head * es;
  char* const v = static_cast<char*>(p.a.v) + (int64_t)h * p.a.v_head * es;
  const int sub = lane / lanes, piece = lane - sub * lanes, once = 32 / lanes;
  constexpr int kAhead = 4;
  for (int at = 0; at < rows; at += once * kAhead) {
    int64_t from[kAhead], to[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int row = at + i * once + sub;
      from[i] = __shfl_sync(kAll, src, row & 31);
      to[i] = __shfl_sync(kAll, dst, row & 31);
      if (row >= 32) to[i] = -1;
    }
    for (int c = piece; c < pieces; c += lanes) {
      P x[kAhead], y[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (to[i] >= 0) {
          x[i] = *reinterpret_cast<const P*>(k + from[i] * p.a.k_slot * es + (int64_t)c * sizeof(P));
          y[i] = *reinterpret_cast<const P*>(v + from[i] * p.a.v_slot * es + (int64_t)c * sizeof(P));
        }
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (to[i] >= 0) {
          *reinterpret_cast<P*>(k + to[i] * p.a.k_slot * es + (int64_t)c * sizeof(P)) = x[i];
          *reinterpret_cast<P*>(v + to[i] * p.a.v_slot * es + (int64_t)c * sizeof(P)) = y[i];
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
    if (e2 == cudaSuccess)
      e2 = cudaFuncSetAttribute(evict_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(sizeof(SelectSmem) + kMaxSpan / 32 * sizeof(Word) + kMaxKeys * 4));
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

int move_rows(const EvictParams& p) { const char* e = getenv("MOVE_ROWS"); return e ? atoi(e) : 32; }
template <typename P>
cudaError_t launch_move(const EvictParams& p, int row_bytes, cudaStream_t stream) {
  const int pieces = row_bytes / (int)sizeof(P), rows = move_rows(p), groups = (p.a.budget + rows - 1) / rows;
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
  if (a->weight_cols > 0 && (!a->weight || !a->weight_out || a->weight == a->weight_out)) return FFTOPK_EINVAL;
  if (a->slots > 0 && (!a->k || !a->v)) return FFTOPK_EINVAL;
  if (!on(a->k, a->elem_bytes) || !on(a->v, a->elem_bytes) || !on(a->k_scale, 4) || !on(a->v_scale, 4) || !on(a->weight, 4) || !on(a->weight_out, 4) ||
      !on(a->page_table, 4) || !on(a->to_table, 4) || !on(a->lengths, 4) || !on(a->new_lengths, 4) || !on(a->kept, 4))
    return FFTOPK_EINVAL;
  const int64_t bound = (int64_t)a->pages * a->page_size < a->weight_cols ? (int64_t)a->pages * a->page_size : a->weight_cols;
  if (a->slots > 0x7fffffff || a->seqs > 0x7fffffff / a->heads || bound > kMaxCluster * kMaxSpan || (int64_t)a->to_pages * a->page_size < a->budget ||
      a->budget > 0x7ffff000)
    return FFTOPK_ERANGE;
  const int64_t units = a->seqs * a->heads;
  if (units * ((a->budget + 7) / 8) > 0x7fffffff) return FFTOPK_ERANGE;
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
  p.keys = (int32_t)(each < kMaxKeys ? each : kMaxKeys);
  p.words = (int32_t)(each / 32);
  cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(units * ctas), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = sizeof(SelectSmem) + (size_t)p.words * sizeof(Word) + (size_t)p.keys * 4;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)ctas;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, evict_select_kernel, p);
  if (e == cudaSuccess && p.moves) {
    const int bytes = a->D * a->elem_bytes;
    int piece = 16;
    while (piece > a->elem_bytes && (bytes % piece != 0 || !rows_on(a->k, a->slots, a->k_slot, a->heads, a->k_head, a->elem_bytes, piece) ||
                                     !rows_on(a->v, a->slots, a->v_slot, a->heads, a->v_head, a->elem_bytes, piece)))
      piece /= 2;
    e = piece == 16  ? launch_move<uint4>(p, bytes, stream)
        : piece == 8 ? launch_move<uint2>(p, bytes, stream)
        : piece == 4 ? launch_move<uint32_t>(p, bytes, stream)
        : piece == 2 ? launch_move<uint16_t>(p, bytes, stream)
                     : launch_move<uint8_t>(p, bytes, stream);
  }
  return e == cudaSuccess ? FFTOPK_OK : cuda_fail(e);
}
