// What the paged-cache kernels share: the pools, the page table, the packed
// new tokens and their checks on the device.
#pragma once

#include <cuda.h>

#include "common.cuh"
#include "vggt_cache.h"

namespace vggt {

// K and V pools [n_pages][kv_heads][page][dim] with common strides (elements).
struct Pool {
  int64_t n_pages, page_stride, head_stride, row_stride;
  int kv_heads, page, page_shift, dim;
};

struct PageTable {
  const int32_t* table;    // [seqs][width]
  const int32_t* lengths;  // [seqs]
  const int32_t* starts;   // [seqs + 1]
  int64_t width, seqs, total;
  int32_t* status;
};

__device__ __forceinline__ void raise_status(int32_t* status, int bit) {
  if (status != nullptr) atomicOr(status, bit);
}

// A page number that may be used as an address, or -1.
__device__ __forceinline__ int checked_page(const PageTable& t, const Pool& pool, int64_t seq,
                                            int64_t index) {
  const int32_t p = __ldg(t.table + seq * t.width + index);
  if (p >= 0 && p < pool.n_pages) return p;
  raise_status(t.status, VGGT_STATUS_BAD_PAGE);
  return -1;
}

// Cached tokens of a sequence, clamped to what its table row can hold.
__device__ __forceinline__ int64_t checked_length(const PageTable& t, const Pool& pool,
                                                  int64_t seq) {
  const int64_t slots = t.width << pool.page_shift;
  const int64_t n = __ldg(t.lengths + seq);
  if (n >= 0 && n <= slots) return n;
  raise_status(t.status, VGGT_STATUS_BAD_LENGTH);
  return n < 0 ? 0 : slots;
}

// First packed row of a sequence and the number of its new tokens, clamped to
// [0, total].
__device__ __forceinline__ int64_t checked_rows(const PageTable& t, int64_t seq, int64_t& first) {
  const int64_t a = __ldg(t.starts + seq), b = __ldg(t.starts + seq + 1);
  if (a >= 0 && b >= a && b <= t.total) {
    first = a;
    return b - a;
  }
  raise_status(t.status, VGGT_STATUS_BAD_LENGTH);
  first = a < 0 ? 0 : (a > t.total ? t.total : a);
  const int64_t e = b > t.total ? t.total : b;
  return e > first ? e - first : 0;
}

// The sequence that packed row `row` belongs to (the last one whose start is
// not above it), or -1 when the row lies before the first or behind the last.
__device__ __forceinline__ int64_t sequence_of_row(const int32_t* starts, int64_t seqs,
                                                   int64_t row) {
  int64_t lo = 0, hi = seqs;
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (__ldg(starts + mid + 1) <= row)
      lo = mid + 1;
    else
      hi = mid;
  }
  return lo < seqs && __ldg(starts + lo) <= row ? lo : -1;
}

// The queries of a sequence and a key head are the rows r = token * group + g,
// g the query head within the head's group, cut into tiles of `tile` rows.
// (The entry points keep total * group below 2^31, so row numbers fit an int.)
struct RowTile {
  int64_t seq, first, len;  // len: cached tokens
  int n_new, row0, rows;  // rows: of the sequence, over all its tiles
};

// Finds the `index`-th row tile over all sequences; false past the last one.
// Called by full warps, every lane gets the answer.
__device__ __forceinline__ bool locate_tile(const PageTable& t, const Pool& pool, int group,
                                            int tile, int64_t index, RowTile& out) {
  const int lane = threadIdx.x & 31;
  int64_t base = 0;
  for (int64_t s0 = 0; s0 < t.seqs; s0 += 32) {
    const int64_t b = s0 + lane;
    int64_t first = 0, n = 0, len = 0;
    if (b < t.seqs) {
      len = checked_length(t, pool, b);  // beside the starts: one latency for both
      n = checked_rows(t, b, first);
    }
    const int64_t tiles = (n * group + tile - 1) / tile;
    int64_t sum = tiles;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int64_t up = __shfl_up_sync(0xffffffffu, sum, off);
      if (lane >= off) sum += up;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, base + sum > index);
    if (hit) {
      const int src = __ffs(hit) - 1;
      out.seq = s0 + src;
      out.first = __shfl_sync(0xffffffffu, first, src);
      out.len = __shfl_sync(0xffffffffu, len, src);
      out.n_new = (int)__shfl_sync(0xffffffffu, n, src);
      out.row0 = (int)(index - base - __shfl_sync(0xffffffffu, sum - tiles, src)) * tile;
      out.rows = out.n_new * group;
      return true;
    }
    base += __shfl_sync(0xffffffffu, sum, 31);
  }
  return false;
}

// Upper bound of the number of row tiles.
inline int64_t most_tiles(int64_t total, int64_t seqs, int group, int tile) {
  return (total * group + seqs * (tile - 1)) / tile;
}

// Tensor map over a pool: boxes of 64 elements x `rows` slots of one page and
// head, 128-byte swizzle; pages outside the pool read as zeros.
bool encode_pool_tmap(CUtensorMap* map, const void* pages, int dtype, const Pool& pool,
                      uint32_t rows);

// Arguments of attention over the paged cache.
struct PagedAttnArgs {
  const void* q;
  int64_t q_token, q_head;
  const void *k_pages, *v_pages;
  Pool pool;
  PageTable t;
  int group, causal, dtype;
  float scale;
  void* out;
  int64_t o_token, o_head;
  float* lse;       // [total][q_heads] or null
  void* workspace;  // counters (zero before and after), then partial results
  uint64_t wait_ns;
  // self-test of the failure detection: one warp waits on a barrier that
  // nothing completes and takes the CTA through the abort path
  int wait_selftest;
};

// Zeros and -inf for the packed rows that belong to no sequence, those before
// the first start and behind the last.  Every CTA calls it once, by one of its
// warps, and takes its share of them.
template <typename T, int D>
__device__ __forceinline__ void fill_rows_of_no_sequence(const PagedAttnArgs& a) {
  const int64_t total = a.t.total;
  int64_t lo = __ldg(a.t.starts), hi = __ldg(a.t.starts + a.t.seqs);
  lo = lo < 0 ? 0 : (lo < total ? lo : total);
  hi = hi < lo ? lo : (hi < total ? hi : total);
  const int64_t rows = lo + total - hi;
  if (rows == 0) return;
  const int lane = threadIdx.x & 31;
  if (blockIdx.x == 0 && lane == 0) raise_status(a.t.status, VGGT_STATUS_BAD_LENGTH);
  const int heads = a.pool.kv_heads * a.group;
#pragma unroll 1
  for (int64_t i = blockIdx.x; i < rows; i += gridDim.x) {
    const int64_t row = i < lo ? i : hi + i - lo;
#pragma unroll 1
    for (int j = lane; j < heads * (D / 8); j += 32)
      reinterpret_cast<uint4*>(static_cast<T*>(a.out) + row * a.o_token +
                               j / (D / 8) * a.o_head)[j % (D / 8)] = make_uint4(0u, 0u, 0u, 0u);
    if (a.lse != nullptr)
#pragma unroll 1
      for (int j = lane; j < heads; j += 32) a.lse[row * heads + j] = -INFINITY;
  }
}

struct WeighArgs {
  const void* q;
  int64_t q_token, q_head;
  const float* lse;  // [total][kv_heads * group]
  const void* k_pages;
  Pool pool;
  PageTable t;
  int group, causal, dtype;
  float scale, decay;
  float* weights;  // [seqs][kv_heads][slots]
  int64_t max_new, max_len;
  uint64_t wait_ns;
  int wait_selftest;
};

struct EvictArgs {
  const float* weights;
  const int32_t* ids;
  void *k_pages, *v_pages;
  Pool pool;
  PageTable t;  // no starts
  int64_t budget;
  const int32_t* recent_from;  // [seqs] or null
  float* new_weights;
  int32_t *new_ids, *new_lengths;
};

cudaError_t launch_paged_weigh_rows(const WeighArgs& a, cudaStream_t st);
cudaError_t launch_paged_weigh_tc05(const WeighArgs& a, cudaStream_t st);

// Counters of unfinished items at the front of a workspace: zero before the
// first call and after every call, in a place that no call uses otherwise.
constexpr int64_t kMaxCounters = VGGT_PAGED_WORKSPACE_ZERO_BYTES / 4;

// A key's weight after a call.  +inf, which keeps a token from eviction, stays
// whatever the decay (0 times it would be NaN, the lowest rank) and the sum.
__device__ __forceinline__ float new_weight(float old, float decay, float sum) {
  return old == INFINITY ? old : fmaf(old, decay, sum);
}

// The expected most new tokens and greatest length, cut down to what can be, so
// that the plans' arithmetic holds for any.
inline void clamp_expected(int64_t total, int64_t& max_new, int64_t& max_len) {
  if (max_new > total) max_new = total > 0 ? total : 1;
  if (max_len > 0x7fffffffLL) max_len = 0x7fffffffLL;
}

// How a launch cuts its work.
struct PagedPlan {
  int rows;               // query rows per CTA
  int64_t tiles;          // row tiles, an upper bound
  int64_t chunk, splits;  // key tiles per CTA, CTAs per row tile and head at most
  size_t partial_bytes;
};

PagedPlan paged_rows_plan(int64_t total, int64_t seqs, int kv_heads, int group, int dim,
                          int64_t max_len);
cudaError_t launch_paged_rows(const PagedAttnArgs& a, const PagedPlan& plan, cudaStream_t st);
PagedPlan paged_tc05_plan(int64_t total, int64_t seqs, int kv_heads, int group, int dim,
                          int64_t max_len);
cudaError_t launch_paged_tc05(const PagedAttnArgs& a, const PagedPlan& plan, cudaStream_t st);

// Host: checks the sizes that every paged entry point takes and fills `pool`.
int check_pool(int dtype, int64_t n_pages, int kv_heads, int page, int dim, int64_t page_stride,
               int64_t head_stride, int64_t row_stride, int64_t table_width, int64_t seqs,
               int64_t total, Pool* pool);

}  // namespace vggt
