// Eviction from the paged cache by accumulated weight.
//
// Of a sequence's slots each key head keeps the `budget` of largest rank: the
// weight, or +inf for tokens numbered recent_from[seq] or later; NaN ranks
// below everything, equal ranks by the lower slot.  What is kept does not
// move but for kept slots at or past the new length ("movers"), which fill
// the slots below it whose tokens are evicted ("holes"): the n-th hole takes
// the n-th mover.  Attention does not depend on the order of cached tokens,
// so this moves the fewest rows, and sources and destinations never overlap:
// all rows move at once.
//
// One launch.  A cluster of CTAs serves a sequence and head (8 CTAs for long
// rows, else one): each takes a contiguous share of the slots, reads their
// weights once into shared memory as monotone 32-bit keys and
//  * finds the smallest kept key by a radix selection of 8 bits a pass, the
//    CTAs' histograms added up over distributed shared memory;
//  * counts ties, holes and movers by one scan each, continued over the CTAs,
//    so that every hole and mover knows its number, and writes the lists;
//  * copies weights and numbers (out of place), then moves the rows, all CTAs
//    of the cluster taking their share of the list, 16 bytes a lane.
// What bounds it: one frame out of 32 in 16 heads (21.6 MB) takes 34 us, a chain
// of four passes of 2 us each, two scans and the moves' dependent loads.  16
// prompts cut from 16,383 to 4,096 tokens (379 MB moved in rows of 256 bytes)
// take 101 us, 3.8 TB/s: 512 threads a CTA, so that the passes of some CTAs run
// beside the moves of others, and the moves' addresses resolved a round ahead of
// the rows (with every row's look-ups before its copy: 162 us).  Four CTAs to an
// SM leave a thread 32 registers, and spill 44 bytes of them (60 with one CTA a
// row).
#include <cooperative_groups.h>

#include "kernels.h"
#include "paged.cuh"

namespace vggt {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kCopies = 8;  // of the histogram: lanes of equal digits meet less often
// keys that a CTA holds in shared memory; longer shares are read again
constexpr int kCachedKeys = 24 * 1024;

struct EvictParams {
  EvictArgs a;
  int64_t slots, most_moves;
  int cached;   // keys that the launch has shared memory for
  int* holes;   // [seqs * heads][most_moves]
  int* movers;
};

__device__ __forceinline__ uint32_t rank_key(float w, int32_t id, int32_t recent) {
  if (id >= recent) return 0xff800000u;  // that of +inf
  return w != w ? 0u : score_key(w);
}

// Exclusive sum over the CTA's threads of two counts in one word; `total` gets
// the sum of all.
__device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t* warp_sums, uint64_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint64_t s = v;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const uint64_t up = __shfl_up_sync(0xffffffffu, s, off);
    if (lane >= off) s += up;
  }
  if (lane == 31) warp_sums[warp] = s;
  __syncthreads();
  uint64_t w = lane < kThreads / 32 ? warp_sums[lane] : 0;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const uint64_t up = __shfl_up_sync(0xffffffffu, w, off);
    if (lane >= off) w += up;
  }
  total = __shfl_sync(0xffffffffu, w, 31);
  const uint64_t before = __shfl_sync(0xffffffffu, w, warp > 0 ? warp - 1 : 0);
  __syncthreads();
  return s - v + (warp > 0 ? before : 0);
}

__device__ __forceinline__ int64_t row_of(const EvictArgs& a, int64_t seq, int head, int slot) {
  const int page = checked_page(a.t, a.pool, seq, slot >> a.pool.page_shift);
  if (page < 0) return -1;
  return page * a.pool.page_stride + head * a.pool.head_stride +
         (slot & (a.pool.page - 1)) * a.pool.row_stride;
}

template <int C, int D>
__global__ void __launch_bounds__(kThreads, 4) evict_kernel(const EvictParams p) {
  extern __shared__ uint32_t keys[];
  __shared__ __align__(16) int copies[256 * kCopies];
  __shared__ int hist[2][256], sums[256];
  __shared__ uint64_t warp_sums[32];
  __shared__ uint64_t share[2];  // this CTA's ties; its holes and movers
  __shared__ uint32_t s_digit;
  __shared__ int s_left, s_equal;
  const EvictArgs& a = p.a;
  const int tid = threadIdx.x, lane = tid & 31;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = C > 1 ? (int)cluster.block_rank() : 0;
  auto sync = [&] {
    if constexpr (C > 1)
      cluster.sync();
    else
      __syncthreads();
  };
  auto remote = [&](auto* at, int r) {
    if constexpr (C > 1)
      return cluster.map_shared_rank(at, r);
    else
      return at;
  };
  const int64_t item = blockIdx.x / C, seq = item / a.pool.kv_heads;
  const int head = (int)(item % a.pool.kv_heads);
  const int n = (int)checked_length(a.t, a.pool, seq);
  const int keep = (int)(n < a.budget ? n : a.budget);
  const bool numbered = a.recent_from != nullptr;
  const int32_t recent = numbered ? a.recent_from[seq] : 0x7fffffff;
  const float* w = a.weights + item * p.slots;
  const int32_t* ids = a.ids + item * p.slots;
  float* w2 = a.new_weights + item * p.slots;
  int32_t* ids2 = a.new_ids + item * p.slots;
  if (tid == 0 && rank == 0 && head == 0) a.new_lengths[seq] = keep;
  // past the new length: 0 and -1
  for (int64_t s = keep + rank * kThreads + tid; s < p.slots; s += C * kThreads) {
    w2[s] = 0.f;
    ids2[s] = -1;
  }
  if (keep == n || keep == 0) {  // the same for the whole cluster: nothing is evicted, or all is
    for (int s = rank * kThreads + tid; s < keep; s += C * kThreads) {
      w2[s] = w[s];
      ids2[s] = ids[s];
    }
    return;
  }
  const int per = (n + C - 1) / C;
  const int first = rank * per < n ? rank * per : n;
  const int count = n - first < per ? n - first : per;
  const bool cached = per <= p.cached;
  auto fresh_key = [&](int s) { return rank_key(w[s], numbered ? ids[s] : 0, recent); };
  auto key_of = [&](int s) { return cached ? keys[s - first] : fresh_key(s); };

  // ---- the keep-th largest key `bound`; `left` of its `equal` equals are kept ----
  uint32_t bound = 0;
  int left = keep, equal = 0;
#pragma unroll 1
  for (int pass = 0; pass < 4; ++pass) {
    const int shift = 24 - 8 * pass;
    int* h = hist[pass & 1];
    for (int i = tid; i < 256 * kCopies; i += kThreads) copies[i] = 0;
    __syncthreads();
    auto add = [&](uint32_t k) {
      atomicAdd(&copies[((k >> shift) & 255u) * kCopies + (tid & (kCopies - 1))], 1);
    };
    if (pass == 0) {
      // four loads in flight; what lies below the new length is copied on the
      // way (holes are overwritten at the end)
      for (int i0 = tid; i0 < count; i0 += 4 * kThreads) {
        float v[4];
        int32_t id[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int i = i0 + j * kThreads;
          v[j] = i < count ? w[first + i] : 0.f;
          id[j] = i < count ? ids[first + i] : 0;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int i = i0 + j * kThreads;
          if (i < count) {
            const uint32_t k = rank_key(v[j], numbered ? id[j] : 0, recent);
            if (cached) keys[i] = k;
            add(k);
            if (first + i < keep) {
              w2[first + i] = v[j];
              ids2[first + i] = id[j];
            }
          }
        }
      }
    } else {
#pragma unroll 4
      for (int i = tid; i < count; i += kThreads) {
        const uint32_t k = cached ? keys[i] : fresh_key(first + i);
        if ((k >> (shift + 8)) == bound) add(k);
      }
    }
    __syncthreads();
    if (tid < 256) {
      int sum = 0;
#pragma unroll
      for (int c = 0; c < kCopies; ++c) sum += copies[tid * kCopies + ((c + tid) & (kCopies - 1))];
      h[tid] = sum;
    }
    sync();
    // from the largest digit down
    int sum = 0;
    if (tid < 256) {
#pragma unroll
      for (int r = 0; r < C; ++r) sum += remote(h, r)[255 - tid];
      int run = sum;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, run, off);
        if (lane >= off) run += up;
      }
      sums[tid] = run;
    }
    __syncthreads();
    if (tid < 256) {
      int above = 0;
      for (int q = 0; q < tid / 32; ++q) above += sums[q * 32 + 31];
      const int upto = above + sums[tid];
      if (upto >= left && upto - sum < left) {
        s_digit = 255 - tid;
        s_left = left - (upto - sum);
        s_equal = sum;
      }
    }
    __syncthreads();
    bound = (bound << 8) | s_digit;
    left = s_left;
    equal = s_equal;
    if (equal == left) {  // all keys with these leading bits are kept
      bound <<= shift;
      break;
    }
  }

  // ---- a thread's slots lie side by side: number its ties, holes, movers ----
  const int each = (count + kThreads - 1) / kThreads;
  const int from = first + (tid * each < count ? tid * each : count);
  const int to = first + ((tid + 1) * each < count ? (tid + 1) * each : count);
  int tie_at = 0;  // number of this thread's first tie
  if (equal != left) {
    uint64_t ties = 0, total;
    for (int s = from; s < to; ++s) ties += key_of(s) == bound;
    tie_at = (int)block_scan(ties, warp_sums, total);
    if (tid == 0) share[0] = total;
    sync();
    for (int r = 0; r < rank; ++r) tie_at += (int)*remote(&share[0], r);
  }
  auto walk = [&](auto&& visit) {
    int tie = tie_at;
    for (int s = from; s < to; ++s) {
      const uint32_t k = key_of(s);
      visit(s, k > bound || (k == bound && (equal == left || tie++ < left)));
    }
  };
  uint64_t mine = 0, total;  // holes below 2^32, movers above
  walk([&](int s, bool kept) { mine += s < keep ? (uint64_t)!kept : (uint64_t)kept << 32; });
  uint64_t at = block_scan(mine, warp_sums, total);
  if (tid == 0) share[1] = total;
  sync();
  int moves = 0;
  for (int r = 0; r < C; ++r) {
    const uint64_t v = *remote(&share[1], r);
    if (r < rank) at += v;
    moves += (int)(uint32_t)v;
  }
  int hole = (int)(uint32_t)at, mover = (int)(at >> 32);
  int* holes = p.holes + item * p.most_moves;
  int* movers = p.movers + item * p.most_moves;
  walk([&](int s, bool kept) {
    if (s >= keep) {
      if (kept) movers[mover++] = s;
    } else if (!kept) {
      holes[hole++] = s;
    }
  });
  sync();  // the lists are complete

  // ---- the moves: addresses first, a pair a thread, then the rows, D / 8 lanes
  // to a row of K and as many to its row of V ----
  static_assert(sizeof(copies) >= 2 * kThreads * sizeof(int64_t), "room for a round's pairs");
  int64_t* src_at = reinterpret_cast<int64_t*>(copies);
  int64_t* dst_at = src_at + kThreads;
  constexpr int kLanes = D / 4, kBatch = 4, kStep = kThreads / kLanes;
  uint4* pages = reinterpret_cast<uint4*>(tid % kLanes < kLanes / 2 ? a.k_pages : a.v_pages);
  const int chunk = tid % (kLanes / 2);
  // (a round is 512 neighbours, even where that leaves CTAs without: the same
  // pairs dealt evenly over the cluster took 114 us for the 16 prompts, not 101)
  for (int base = rank * kThreads; base < moves; base += C * kThreads) {
    const int here = moves - base < kThreads ? moves - base : kThreads;
    __syncthreads();
    if (tid < here) {
      const int src = movers[base + tid], dst = holes[base + tid];
      const int64_t from_row = row_of(a, seq, head, src), to_row = row_of(a, seq, head, dst);
      src_at[tid] = from_row / 8;
      dst_at[tid] = from_row < 0 || to_row < 0 ? -1 : to_row / 8;
      w2[dst] = w[src];
      ids2[dst] = ids[src];
    }
    __syncthreads();
    for (int i0 = tid / kLanes; i0 < here; i0 += kBatch * kStep) {
      uint4 row[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int i = i0 + j * kStep;
        if (i < here && dst_at[i] >= 0) row[j] = pages[src_at[i] + chunk];
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int i = i0 + j * kStep;
        if (i < here && dst_at[i] >= 0) pages[dst_at[i] + chunk] = row[j];
      }
    }
  }
}

template <int C, int D>
cudaError_t launch_evict(const EvictParams& p, int64_t items, cudaStream_t st) {
  auto kernel = evict_kernel<C, D>;
  const size_t smem = (size_t)p.cached * 4;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       kCachedKeys * 4);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(items * C));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = C;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

// Moves of one sequence and head at most: every mover is past the budget,
// every hole below it.
int64_t most_moves(int64_t slots, int64_t budget) {
  const int64_t past = slots - budget;
  const int64_t m = budget < past ? budget : past;
  return m > 0 ? m : 0;
}

size_t evict_bytes(int64_t items, int64_t moves) { return (size_t)items * moves * 2 * 4; }

}  // namespace
}  // namespace vggt

using namespace vggt;

extern "C" size_t vggt_paged_evict_workspace_size(int64_t seqs, int kv_heads, int64_t slots,
                                                  int64_t budget) {
  if (seqs <= 0 || kv_heads < 1 || slots < 0 || budget < 0) return 0;
  return evict_bytes(seqs * kv_heads, most_moves(slots, budget));
}

extern "C" int vggt_paged_evict(const float* weights, const int32_t* ids, int dtype, void* k_pages,
                                void* v_pages, int64_t n_pages, int kv_heads, int page, int dim,
                                int64_t page_stride, int64_t head_stride, int64_t row_stride,
                                const int32_t* table, int64_t table_width, int64_t seqs,
                                const int32_t* lengths, int64_t budget, const int32_t* recent_from,
                                int64_t max_len, float* new_weights, int32_t* new_ids,
                                int32_t* new_lengths, int32_t* status, void* workspace,
                                size_t workspace_bytes, void* stream) {
  EvictParams p{};
  EvictArgs& a = p.a;
  if (int rc = check_pool(dtype, n_pages, kv_heads, page, dim, page_stride, head_stride,
                          row_stride, table_width, seqs, 0, &a.pool))
    return rc;
  if (budget < 0 || max_len < 0) return api_fail("budget and max_len must not be negative");
  const int64_t items = seqs * kv_heads;
  if (items > 65535) return api_fail("seqs * kv_heads = %lld exceeds 65535", (long long)items);
  if (seqs == 0) return api_fail(nullptr);
  if (!lengths || !new_lengths) return api_fail("lengths and new_lengths must be non-NULL");
  p.slots = table_width * page;
  if (p.slots > 0 &&
      (!weights || !ids || !new_weights || !new_ids || !table || !k_pages || !v_pages))
    return api_fail("weights, ids, their outputs, the table and the pools must be non-NULL");
  if (lengths == new_lengths || (p.slots > 0 && (weights == new_weights || ids == new_ids)))
    return api_fail("the outputs must not be the inputs");
  if ((reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages)) & 15u)
    return api_fail("the pools must be 16-byte aligned");
  p.most_moves = most_moves(p.slots, budget);
  const size_t need = evict_bytes(items, p.most_moves);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return api_fail("workspace of %zu bytes, %zu needed", workspace_bytes, need);
  a.weights = weights;
  a.ids = ids;
  a.k_pages = k_pages;
  a.v_pages = v_pages;
  a.t = {table, lengths, nullptr, table_width, seqs, 0, status};
  a.budget = budget;
  a.recent_from = recent_from;
  a.new_weights = new_weights;
  a.new_ids = new_ids;
  a.new_lengths = new_lengths;
  p.holes = static_cast<int*>(workspace);
  p.movers = p.holes + items * p.most_moves;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // A cluster of 8 CTAs where a row has more than 2,048 slots (16 heads of one
  // sequence, one CTA against eight: 1,500 slots 13.0 / 16.7 us, 3,000 slots
  // 26.0 / 14.4 us, 6,000 slots 36.1 / 20.4 us).
  const int64_t longest = max_len < p.slots ? max_len : p.slots;
  const bool wide = longest > 2048;
  const int64_t share = wide ? (longest + 7) / 8 : longest;
  p.cached = (int)(share < kCachedKeys ? (share + 31) / 32 * 32 : kCachedKeys);
  if (dim == 64)
    return api_cuda(wide ? launch_evict<8, 64>(p, items, st) : launch_evict<1, 64>(p, items, st));
  return api_cuda(wide ? launch_evict<8, 128>(p, items, st) : launch_evict<1, 128>(p, items, st));
}
