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
// First launch: one CTA per sequence and head finds the smallest kept rank
// by a radix selection, marks what is kept, pairs holes with movers and
// writes the new weights and numbers (out of place).  Second launch: the
// rows.
#include "kernels.h"
#include "paged.cuh"

namespace vggt {
namespace {

constexpr int kThreads = 1024;

struct EvictParams {
  EvictArgs a;
  int64_t slots, most_moves;
  int* counts;  // [seqs * heads]
  int* holes;   // [seqs * heads][most_moves]
  int* movers;
};

__device__ __forceinline__ uint32_t rank_key(float w, int32_t id, int32_t recent) {
  if (id >= recent) return 0xff800000u;  // that of +inf
  return w != w ? 0u : score_key(w);
}

// Exclusive sum over the CTA's threads; `total` gets the sum of all.
__device__ __forceinline__ int block_scan(int v, int* warp_sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int s = v;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, s, off);
    if (lane >= off) s += up;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = s;
  __syncthreads();
  if (warp == 0) {
    int w = lane < kThreads / 32 ? warp_sums[lane] : 0;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, w, off);
      if (lane >= off) w += up;
    }
    warp_sums[lane] = w;
  }
  __syncthreads();
  total = warp_sums[kThreads / 32 - 1];
  return s - v + (warp > 0 ? warp_sums[warp - 1] : 0);
}

__global__ void __launch_bounds__(kThreads) evict_select_kernel(const EvictParams p) {
  __shared__ int hist[256];
  __shared__ int warp_sums[32];
  __shared__ uint32_t s_prefix;
  __shared__ int s_need;
  const EvictArgs& a = p.a;
  const int64_t item = blockIdx.x, seq = item / a.pool.kv_heads;
  const int n = (int)checked_length(a.t, a.pool, seq);
  const int keep = (int)(n < a.budget ? n : a.budget);
  const int32_t recent = a.recent_from != nullptr ? a.recent_from[seq] : 0x7fffffff;
  const float* w = a.weights + item * p.slots;
  const int32_t* ids = a.ids + item * p.slots;
  float* w2 = a.new_weights + item * p.slots;
  int32_t* ids2 = a.new_ids + item * p.slots;
  const int tid = threadIdx.x;
  if (tid == 0 && item % a.pool.kv_heads == 0) a.new_lengths[seq] = keep;
  auto key_of = [&](int s) {
    return rank_key(w[s], a.recent_from != nullptr ? ids[s] : 0, recent);
  };
  // ---- the keep-th largest key `bound`, and how many of its equals are kept ----
  uint32_t bound = 0;
  int need = 0;
  if (keep < n && keep > 0) {
    if (tid == 0) {
      s_prefix = 0;
      s_need = keep;
    }
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      const uint32_t prefix = s_prefix;
      for (int s = tid; s < n; s += kThreads) {
        const uint32_t k = key_of(s);
        if (shift == 24 || (k >> (shift + 8)) == prefix) atomicAdd(&hist[(k >> shift) & 255], 1);
      }
      __syncthreads();
      if (tid == 0) {
        int left = s_need, d = 255;
        for (; d > 0 && hist[d] < left; --d) left -= hist[d];
        s_need = left;
        s_prefix = (prefix << 8) | (uint32_t)d;
      }
      __syncthreads();
    }
    bound = s_prefix;
    need = s_need;
  }
  // ---- kept or not, in the order of the slots ----
  int ties = 0, holes = 0, movers = 0;
  int* hole_at = p.holes + item * p.most_moves;
  int* mover_at = p.movers + item * p.most_moves;
  for (int s0 = 0; s0 < n; s0 += kThreads) {
    const int s = s0 + tid;
    const uint32_t k = s < n ? key_of(s) : 0u;
    bool kept = s < n && keep > 0;
    if (keep < n && keep > 0) {
      const bool tie = s < n && k == bound;
      int total;
      const int before = block_scan(tie ? 1 : 0, warp_sums, total);
      kept = s < n && (k > bound || (tie && ties + before < need));
      ties += total;
    }
    const bool hole = s < keep && !kept, mover = s < n && s >= keep && kept;
    int total;
    const int packed = block_scan((hole ? 1 : 0) | (mover ? 1 << 16 : 0), warp_sums, total);
    if (hole) hole_at[holes + (packed & 0xffff)] = s;
    if (mover) mover_at[movers + (packed >> 16)] = s;
    holes += total & 0xffff;
    movers += total >> 16;
    if (s < keep && kept) {
      w2[s] = w[s];
      ids2[s] = ids[s];
    }
  }
  __syncthreads();
  for (int i = tid; i < holes; i += kThreads) {
    const int from = mover_at[i], to = hole_at[i];
    w2[to] = w[from];
    ids2[to] = ids[from];
  }
  for (int64_t s = keep + tid; s < p.slots; s += kThreads) {
    w2[s] = 0.f;
    ids2[s] = -1;
  }
  if (tid == 0) p.counts[item] = holes;
}

__device__ __forceinline__ int64_t row_of(const EvictArgs& a, int64_t seq, int head, int slot) {
  const int page = checked_page(a.t, a.pool, seq, slot >> a.pool.page_shift);
  if (page < 0) return -1;
  return page * a.pool.page_stride + head * a.pool.head_stride +
         (slot & (a.pool.page - 1)) * a.pool.row_stride;
}

// D / 8 lanes to a row of K and as many to its row of V.
template <int D>
__global__ void __launch_bounds__(256) evict_move_kernel(const EvictParams p) {
  constexpr int kLanes = D / 4;
  const EvictArgs& a = p.a;
  const int64_t item = blockIdx.y;
  const int64_t seq = item / a.pool.kv_heads;
  const int head = (int)(item % a.pool.kv_heads);
  const int moves = p.counts[item];
  const int lane = threadIdx.x % kLanes;
  uint4* pages = reinterpret_cast<uint4*>(lane < kLanes / 2 ? a.k_pages : a.v_pages);
  const int c = lane % (kLanes / 2);
  const int step = gridDim.x * (256 / kLanes);
  for (int i = blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes; i < moves; i += step) {
    const int64_t from = row_of(a, seq, head, p.movers[item * p.most_moves + i]);
    const int64_t to = row_of(a, seq, head, p.holes[item * p.most_moves + i]);
    if (from >= 0 && to >= 0) pages[to / 8 + c] = pages[from / 8 + c];
  }
}

// Moves of one sequence and head at most: every mover is past the budget,
// every hole below it.
int64_t most_moves(int64_t slots, int64_t budget) {
  const int64_t past = slots - budget;
  const int64_t m = budget < past ? budget : past;
  return m > 0 ? m : 0;
}

size_t evict_bytes(int64_t items, int64_t moves) {
  return (((size_t)items * 4 + 255) & ~(size_t)255) + (size_t)items * moves * 2 * 4;
}

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
  if (!workspace || workspace_bytes < need)
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
  p.counts = static_cast<int*>(workspace);
  p.holes = reinterpret_cast<int*>(static_cast<char*>(workspace) +
                                   (((size_t)items * 4 + 255) & ~(size_t)255));
  p.movers = p.holes + items * p.most_moves;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  evict_select_kernel<<<(unsigned)items, kThreads, 0, st>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || p.most_moves == 0) return api_cuda(e);
  // CTAs of 8 to 16 rows: enough for the expected moves, eight per SM at most
  const int64_t expect = most_moves(max_len > budget ? max_len : budget, budget);
  int64_t gx = (expect * (dim / 4) + 255) / 256;
  const int64_t fill = (8 * 148 + items - 1) / items;
  gx = gx < 1 ? 1 : (gx > fill ? fill : gx);
  const dim3 grid((unsigned)gx, (unsigned)items);
  if (dim == 64)
    evict_move_kernel<64><<<grid, 256, 0, st>>>(p);
  else
    evict_move_kernel<128><<<grid, 256, 0, st>>>(p);
  return api_cuda(cudaGetLastError());
}
