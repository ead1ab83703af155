// Eviction from a paged cache by accumulated attention weight. Of every sequence and key head `budget` rows stay: the first `sinks`, the
// last `recent`, and of those between the ones of the largest weights (equal weights: the lower position). They go, in order, to the
// rows that another page table names; their weights go along. A sequence of up to `budget` rows keeps them all. (The reference ends with
// the selection of indices; attention over a paged cache that adds up the weights is fftopk_paged.cu.)
//
// evict_select_kernel: a cluster per sequence and key head finds the smallest weight that stays, by radix rounds over the order-preserving
// keys of the weights (11, 11 and 10 bits, histograms in shared memory, summed over the cluster), and lists what stays in order: every CTA has
// a stretch of the positions, every warp a stretch of those, so that places are prefix sums. A weight is read once, its key stays in
// shared memory (positions beyond its room are read again).
// evict_move_kernel: a warp takes 32 rows of a key head that lie next to each other where they go; a lane finds where one of them comes from, and
// the warp copies k and v. Reading and writing the rows bounds it.
#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

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
constexpr int kMaxKeys = 20 * 1024;  // of a CTA in shared memory: two CTAs per SM
constexpr int kMoveThreads = 128;

struct EvictParams {
  fftopk_evict a;
  int32_t bound;  // positions that the table and the weights reach
  int32_t keys;   // of a CTA that shared memory has room for
  int32_t moves;  // evict_move_kernel follows
  FastDiv page;
  uint32_t* status;
};

__device__ __forceinline__ int digit_shift(int round) { return round == 0 ? 21 : round == 1 ? 10 : 0; }

struct SelectSmem {
  uint32_t hist[kRounds][kBins];
  uint32_t warp_total[kWarps];
  uint32_t found[3];       // bin, count above it, count in it
  uint32_t stay[2];        // of this CTA: rows that stay for certain, rows of the smallest weight that stays
  uint32_t warp_stay[2][kWarps];
};

__global__ void __launch_bounds__(kThreads) evict_select_kernel(const __grid_constant__ EvictParams p) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  SelectSmem& sm = *reinterpret_cast<SelectSmem*>(smem_raw);
  uint32_t* const keys = reinterpret_cast<uint32_t*>(smem_raw + sizeof(SelectSmem));
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
  const int32_t from = min(n, rank * each), to = min(n, from + each);
  const int32_t lo = max(from, first), hi = min(to, last);  // of the CTA's stretch, between

  for (int i = tid; i < kRounds * kBins; i += kThreads) (&sm.hist[0][0])[i] = 0u;
  __syncthreads();
  auto key_at = [&](int32_t j) { return j - from < p.keys ? keys[j - from] : fftopk_key_from_bits(__float_as_uint(w[j])); };
  // the key of the smallest weight that stays, and how many of that weight do (0 of 0xffffffff + 1: none is in question)
  uint32_t edge = 0, mask = 0, ties = need;
  for (int round = 0; round < kRounds; ++round) {
    const int shift = digit_shift(round);
    const uint32_t top = round == 0 ? 0x7ffu : round == 1 ? 0x7ffu : 0x3ffu;
    for (int32_t base = lo; base < hi; base += kThreads) {
      const int32_t j = base + tid;
      const bool in = j < hi;
      uint32_t key = 0;
      if (in) {
        if (round == 0) {
          key = fftopk_key_from_bits(__float_as_uint(w[j]));
          if (j - from < p.keys) keys[j - from] = key;
        } else {
          key = key_at(j);
        }
      }
      const bool counts = in && (key & mask) == edge;
      const uint32_t digit = key >> shift & top;
      const unsigned who = __ballot_sync(kAll, counts);
      if (who == 0u) continue;
      const uint32_t lead = __shfl_sync(kAll, digit, __ffs((int)who) - 1);
      if (__all_sync(kAll, !counts || digit == lead)) {  // (copies of one weight: one addition for the warp)
        if (lane == 0) atomicAdd(&sm.hist[round][lead], (uint32_t)__popc(who));
      } else if (counts) {
        atomicAdd(&sm.hist[round][digit], 1u);
      }
    }
    if (ctas > 1)
      cluster.sync();
    else
      __syncthreads();
    // four bins a thread, from the top: where the count from above reaches `need`
    uint32_t v[4], s = 0;
    const int bin0 = kBins - 4 - 4 * tid;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = 0;
    for (int c = 0; c < ctas; ++c) {
      const uint4 x = *reinterpret_cast<const uint4*>(cluster.map_shared_rank(&sm.hist[round][bin0], c));
      v[0] += x.w, v[1] += x.z, v[2] += x.y, v[3] += x.x;  // highest bin first
    }
    s = v[0] + v[1] + v[2] + v[3];
    uint32_t upto = s;
#pragma unroll
    for (int i = 1; i < 32; i <<= 1) {
      const uint32_t y = __shfl_up_sync(kAll, upto, i);
      if (lane >= i) upto += y;
    }
    if (lane == 31) sm.warp_total[warp] = upto;
    if (tid == 0) sm.found[0] = 0xffffffffu;
    __syncthreads();
    uint32_t above = upto - s;
    for (int i = 0; i < warp; ++i) above += sm.warp_total[i];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (above < need && above + v[e] >= need) sm.found[0] = (uint32_t)(bin0 + 3 - e), sm.found[1] = above, sm.found[2] = v[e];
      above += v[e];
    }
    __syncthreads();
    const uint32_t bin = sm.found[0], over = sm.found[1], in_bin = sm.found[2];
    if (bin == 0xffffffffu) {  // (need = 0: none of the rows between stays)
      edge = 0xffffffffu, mask = 0xffffffffu, ties = 0;
      break;
    }
    edge |= bin << shift;
    mask |= top << shift;
    need -= over;
    ties = need;
    if (in_bin == need) break;  // the whole bin stays
  }
  // Rows above the bin stay; of the bin's, where it is one weight (mask all ones) or stays whole, the first `ties`.
  // count, sum over warps and CTAs, write
  const int32_t part = ((to - from + kWarps - 1) / kWarps + 31) & ~31;
  const int32_t w0 = min(to, from + warp * part), w1 = min(to, w0 + part);
  auto sort_of = [&](int32_t j, bool& sure, bool& tie) {
    sure = j < first || j >= last;
    tie = false;
    if (!sure) {
      const uint32_t k = key_at(j) & mask;
      sure = k > edge;
      tie = k == edge;
    }
  };
  uint32_t sures = 0, tied = 0;
  for (int32_t base = w0; base < w1; base += 32) {
    bool sure = false, tie = false;
    if (base + lane < w1) sort_of(base + lane, sure, tie);
    sures += (uint32_t)__popc(__ballot_sync(kAll, sure));
    tied += (uint32_t)__popc(__ballot_sync(kAll, tie));
  }
  if (lane == 0) sm.warp_stay[0][warp] = sures, sm.warp_stay[1][warp] = tied;
  __syncthreads();
  if (tid < 2) {
    uint32_t s = 0;
    for (int i = 0; i < kWarps; ++i) s += sm.warp_stay[tid][i];
    sm.stay[tid] = s;
  }
  if (ctas > 1)
    cluster.sync();
  else
    __syncthreads();
  uint32_t sures_before = 0, tied_before = 0;
  for (int c = 0; c < rank; ++c) {
    const uint32_t* s = cluster.map_shared_rank(&sm.stay[0], c);
    sures_before += s[0], tied_before += s[1];
  }
  for (int i = 0; i < warp; ++i) sures_before += sm.warp_stay[0][i], tied_before += sm.warp_stay[1][i];
  for (int32_t base = w0; base < w1; base += 32) {
    const int32_t j = base + lane;
    bool sure = false, tie = false;
    if (j < w1) sort_of(j, sure, tie);
    const unsigned s = __ballot_sync(kAll, sure), t = __ballot_sync(kAll, tie), below = (1u << lane) - 1u;
    const uint32_t tie_rank = tied_before + (uint32_t)__popc(t & below);
    if (sure || (tie && tie_rank < ties)) {
      const uint32_t at = sures_before + (uint32_t)__popc(s & below) + min(tie_rank, ties);
      if (at < (uint32_t)left) kept[at] = j, wo[at] = w[j];
    }
    sures_before += (uint32_t)__popc(s), tied_before += (uint32_t)__popc(t);
  }
  if (ctas > 1) cluster.sync();  // (nobody leaves while its memory is read)
}

// P: what a piece of a row is copied as
template <typename P>
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const __grid_constant__ EvictParams p, int pieces, int lanes, int groups) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * (kMoveThreads / 32) + (threadIdx.x >> 5);
  // (32 rows of a key head; the key heads of the same places are neighbours)
  const int64_t rest = item / p.a.heads;
  const int h = (int)(item - rest * p.a.heads);
  const int64_t b = rest / groups;
  const int32_t j0 = (int32_t)(rest - b * groups) * 32;
  if (b >= p.a.seqs) return;
  const int32_t left = p.a.new_lengths[b];
  if (j0 >= left) return;
  int64_t src = -1, dst = -1;
  const int32_t j = j0 + lane;
  if (j < left) {
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
  for (int at = 0; at < 32; at += once * kAhead) {
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
      e2 = cudaFuncSetAttribute(evict_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(sizeof(SelectSmem) + kMaxKeys * 4));
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
cudaError_t launch_move(const EvictParams& p, int row_bytes, cudaStream_t stream) {
  const int pieces = row_bytes / (int)sizeof(P), groups = (p.a.budget + 31) / 32;
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
  return cudaLaunchKernelEx(&cfg, evict_move_kernel<P>, p, pieces, lanes, groups);
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
  if (a->slots > 0x7fffffff || a->seqs > 0x7fffffff / a->heads || bound > 0x7ffff000 || (int64_t)a->to_pages * a->page_size < a->budget ||
      a->budget > 0x7ffff000)
    return FFTOPK_ERANGE;
  const int64_t units = a->seqs * a->heads;
  if (units * ((a->budget + 31) / 32) > 0x7fffffff) return FFTOPK_ERANGE;
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
  // CTAs a unit: as many as fit the device at once, of 4,096 positions at least
  int ctas = 1;
  while (ctas < kMaxCluster && units * ctas * 2 <= 2 * (int64_t)sms && bound / ctas > 8192) ctas *= 2;
  if (units * ctas > 0x7fffffff) return FFTOPK_ERANGE;
  const int64_t each = ((bound + ctas - 1) / ctas + 31) & ~(int64_t)31;
  p.keys = (int32_t)(each < kMaxKeys ? each : kMaxKeys);
  cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(units * ctas), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = sizeof(SelectSmem) + (size_t)p.keys * 4;
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
