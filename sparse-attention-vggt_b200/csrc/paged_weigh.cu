// Accumulated attention weight: for every cached key j of a key head
//   w_j = decay * w_j + sum_i exp(s_ij - lse_i)
// over the new tokens i and query heads of its group that see it, the
// probabilities recomputed from the log-sum-exp that the attention left.
// Every key is owned by one CTA, which walks over all rows, so the sums have
// a fixed order and need no atomics.
//
// Few rows (decode): bound by reading K once.  The CTA keeps the rows in
// shared memory and streams 64-key tiles through a ring as the attention
// kernel does; a warp owns 16 keys of a tile and adds its rows' probabilities
// in registers.
#include <cuda.h>

#include <cmath>

#include "kernels.h"
#include "mma.cuh"
#include "paged.cuh"
#include "paged_producer.cuh"
#include "tc05.cuh"

namespace vggt {
namespace {

constexpr int kTile = 64, kRowsMax = 64, kThreads = 160;

// short rings, and so three or four CTAs to an SM: a tile's chain of wait,
// products, exponentials and sums takes longer than its copy
template <int D>
constexpr int kStagesOf = D == 64 ? 5 : 3;
template <int D>
constexpr int kCtas = D == 64 ? 4 : 3;

struct WeighParams {
  WeighArgs a;
  float scale_log2;
  int64_t splits, chunk;  // CTAs per sequence and head, key tiles per CTA (least)
};

// Whether `ok` holds in all of the four compute warps.
__device__ __forceinline__ bool all_of_128(bool ok) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 q, %1, 0;\n\t"
      "barrier.cta.red.and.pred p, 1, 128, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)ok)
      : "memory");
  return r != 0;
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, kCtas<D>)
    weigh_rows_kernel(const __grid_constant__ CUtensorMap tm_k, const WeighParams p) {
  constexpr int kHalves = D / 64, kSteps = D / 16;
  constexpr uint32_t kStage = kTile * D * 2;
  constexpr int kStages = kStagesOf<D>;
  extern __shared__ unsigned char raw[];
  unsigned char* ring = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
  const uint32_t ring_addr = smem_u32(ring);
  const uint32_t q_addr = ring_addr + kStages * kStage;  // [half][64 rows][128 B], swizzled
  __shared__ uint64_t bars[2 * kStages + 1];  // the last: nothing arrives (wait self-test)
  __shared__ float lse2[kRowsMax];
  __shared__ int limit[kRowsMax];
  __shared__ int s_abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const WeighArgs& a = p.a;

  const int64_t split = blockIdx.x % p.splits, item = blockIdx.x / p.splits;
  const int head = (int)(item % a.pool.kv_heads);
  const int64_t seq = item / a.pool.kv_heads;
  const int64_t len = checked_length(a.t, a.pool, seq);
  int64_t first;
  const int n_new = (int)checked_rows(a.t, seq, first);
  const int rows = n_new * a.group;
  const int64_t all_tiles = (len + kTile - 1) / kTile;
  int64_t chunk = (all_tiles + p.splits - 1) / p.splits;
  if (chunk < p.chunk) chunk = p.chunk;
  const int64_t tile0 = split * chunk;
  if (tile0 >= all_tiles) return;
  const int64_t tiles = all_tiles - tile0 < chunk ? all_tiles - tile0 : chunk;

  auto full = [&](int s) { return smem_u32(&bars[s]); };
  auto empty = [&](int s) { return smem_u32(&bars[kStages + s]); };
  volatile int* abort_flag = &s_abort;
  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
      tc::mbar_init(full(s), 1);
      tc::mbar_init(empty(s), 4);
    }
    tc::mbar_init(smem_u32(&bars[2 * kStages]), 1);
    s_abort = 0;
    tc::mbar_fence_init();
  }
  __syncthreads();

  if (warp == 4) {
    // ================= TMA producer =================
    if (!a.wait_selftest || tc::warp_wait(smem_u32(&bars[2 * kStages]), 0, abort_flag, a.wait_ns))
      produce_tiles<kHalves, kStages>(a.t, a.pool, seq, head, tile0 * kTile,
                                      (int)(len - tile0 * kTile), (int)tiles, &tm_k, ring_addr,
                                      full(0), empty(0), abort_flag, a.wait_ns);
  } else {
    const int krow = ((lane >> 4) & 1) * 8 + (lane & 7), kchunk = (lane >> 3) & 1;
    const int qrow = ((lane >> 3) & 1) * 8 + (lane & 7), qchunk = (lane >> 4) & 1;
    // rows c0 .. c0 + 63 into shared memory, filled up to a multiple of 16 with
    // the first one, its limit and lse +inf, which gives nothing (rows of zeros
    // would give NaN against a key with an infinite element, whose scores may
    // all be -inf)
    auto load_rows = [&](int c0) {
      const int here = rows - c0 < kRowsMax ? rows - c0 : kRowsMax;
#pragma unroll
      for (int i = tid; i < kRowsMax * (D / 8); i += 128) {
        const int r = i / (D / 8), c = i % (D / 8);
        if (r >= (here + 15) / 16 * 16) break;
        const int row = c0 + (r < here ? r : 0);
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(
            static_cast<const T*>(a.q) + (first + row / a.group) * a.q_token +
            ((int64_t)head * a.group + row % a.group) * a.q_head + c * 8));
        const uint32_t dst =
            q_addr + (c >> 3) * (kRowsMax * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4);
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(v.x), "r"(v.y),
                     "r"(v.z), "r"(v.w)
                     : "memory");
      }
      if (tid < kRowsMax) {
        const int row = c0 + (tid < here ? tid : 0);
        float l = -INFINITY;
        if (tid < here)
          l = a.lse[(first + row / a.group) * ((int64_t)a.pool.kv_heads * a.group) +
                    (int64_t)head * a.group + row % a.group];
        // a row without keys gives nothing either
        lse2[tid] = l == -INFINITY ? INFINITY : l * 1.4426950408889634f;
        // keys of this CTA's run that the row sees
        const int64_t n = (a.causal ? len - n_new + row / a.group + 1 : len) - tile0 * kTile;
        limit[tid] = (int)(n < 0 ? 0 : (n < tiles * kTile ? n : tiles * kTile));
      }
    };
    auto sync_rows = [] { asm volatile("bar.sync 1, 128;" ::: "memory"); };
    // With 64 rows at most they are loaded once and the warps go their own
    // ways; more rows (the caller expected fewer) are loaded again per tile.
    const bool once = rows <= kRowsMax;
    if (once) {
      load_rows(0);
      sync_rows();
    }
    float* weights =
        a.weights + (seq * a.pool.kv_heads + head) * (a.t.width << a.pool.page_shift);
    // the old weights of this lane's keys in tile t, loaded a tile ahead: their
    // latency is a tile's whole time
    auto load_old = [&](int64_t t, float* v) {
      if (lane >= 4) return;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t key =
            (tile0 + t) * kTile + warp * 16 + (j >> 1) * 8 + lane * 2 + (j & 1);
        v[j] = t < tiles && key < len ? weights[key] : 0.f;
      }
    };
    float next_old[4];
    load_old(0, next_old);
    for (int64_t t = 0; t < tiles; ++t) {
      const int stage = (int)(t % kStages);
      const bool got =
          tc::warp_wait(full(stage), (uint32_t)((t / kStages) & 1), abort_flag, a.wait_ns);
      // sharing barriers below, the warps go on or leave together
      if (once ? !got : !all_of_128(got)) break;
      const int at = (int)t * kTile + warp * 16;  // this warp's first key, in the run
      const int64_t key0 = tile0 * kTile + at;
      const uint32_t kbase = ring_addr + (uint32_t)stage * kStage + warp * 16 * 128;
      float old[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) old[j] = next_old[j];
      load_old(t + 1, next_old);
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
      for (int c0 = 0; c0 < rows; c0 += kRowsMax) {
        if (!once) {
          sync_rows();
          load_rows(c0);
          sync_rows();
        }
        const int here = rows - c0 < kRowsMax ? rows - c0 : kRowsMax;
        const bool masked = at + 16 > limit[0];
        for (int m0 = 0; m0 < here; m0 += 16) {
          float s[2][4];
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[n][j] = 0.f;
#pragma unroll
          for (int k = 0; k < kSteps; ++k) {
            uint32_t q[4], b0, b1, b2, b3;
            const int r = m0 + qrow, cq = (k & 3) * 2 + qchunk, ck = (k & 3) * 2 + kchunk;
            ldsm_x4(q_addr + (k >> 2) * (kRowsMax * 128) + r * 128 + ((cq ^ (r & 7)) << 4), q[0],
                    q[1], q[2], q[3]);
            ldsm_x4(kbase + (k >> 2) * (kTile * 128) + krow * 128 + ((ck ^ (krow & 7)) << 4), b0,
                    b1, b2, b3);
            MmaOp<T>::mma(s[0], q, b0, b1);
            MmaOp<T>::mma(s[1], q, b2, b3);
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int r = m0 + (lane >> 2) + 8 * i;
            const float l = lse2[r];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              float e = fast_exp2(fmaf(s[j >> 1][2 * i + (j & 1)], p.scale_log2, -l));
              if (masked && at + (j >> 1) * 8 + (lane & 3) * 2 + (j & 1) >= limit[r]) e = 0.f;
              sum[j] += e;
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(empty(stage));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 4);
        sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 8);
        sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 16);
      }
      if (lane < 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int64_t key = key0 + (j >> 1) * 8 + lane * 2 + (j & 1);
          if (key < len) weights[key] = new_weight(old[j], a.decay, sum[j]);
        }
      }
    }
  }
  __syncthreads();
  if (tid == 0 && s_abort) raise_status(a.t.status, VGGT_STATUS_TIMEOUT);
}

template <typename T, int D>
cudaError_t launch_weigh_rows(const WeighParams& p, const CUtensorMap& mk, cudaStream_t st) {
  auto kernel = weigh_rows_kernel<T, D>;
  const size_t smem = kStagesOf<D> * kTile * D * 2 + kRowsMax * D * 2 + 1024;
  const cudaError_t e =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  kernel<<<(unsigned)(p.a.t.seqs * p.a.pool.kv_heads * p.splits), kThreads, smem, st>>>(mk, p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_paged_weigh_rows(const WeighArgs& a, cudaStream_t st) {
  WeighParams p;
  p.a = a;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  const int64_t items = a.t.seqs * a.pool.kv_heads;
  const int64_t key_tiles = (a.max_len + kTile - 1) / kTile;
  p.chunk = items * key_tiles / (4 * 3 * 148);
  if (p.chunk < 2) p.chunk = 2;
  p.splits = key_tiles > 0 ? (key_tiles + p.chunk - 1) / p.chunk : 1;
  if (items * p.splits > 0x7fffffffLL) return cudaErrorInvalidValue;
  CUtensorMap mk;
  const uint32_t box = (uint32_t)(a.pool.page < kTile ? a.pool.page : kTile);
  if (!encode_pool_tmap(&mk, a.k_pages, a.dtype, a.pool, box)) return cudaErrorInvalidValue;
  if (a.dtype == VGGT_DTYPE_BF16)
    return a.pool.dim == 64 ? launch_weigh_rows<__nv_bfloat16, 64>(p, mk, st)
                            : launch_weigh_rows<__nv_bfloat16, 128>(p, mk, st);
  return a.pool.dim == 64 ? launch_weigh_rows<__half, 64>(p, mk, st)
                          : launch_weigh_rows<__half, 128>(p, mk, st);
}

}  // namespace vggt

using namespace vggt;

extern "C" int vggt_paged_weights(const void* q, int dtype, int64_t total, int64_t q_token_stride,
                                  int64_t q_head_stride, const float* lse, const void* k_pages,
                                  int64_t n_pages, int kv_heads, int page, int dim,
                                  int64_t page_stride, int64_t head_stride, int64_t row_stride,
                                  const int32_t* table, int64_t table_width, int64_t seqs,
                                  const int32_t* lengths, const int32_t* starts, int group,
                                  int causal, float scale, float decay, int64_t max_new,
                                  int64_t max_len, float* weights, int32_t* status, void* stream) {
  WeighArgs a{};
  if (int rc = check_pool(dtype, n_pages, kv_heads, page, dim, page_stride, head_stride,
                          row_stride, table_width, seqs, total, &a.pool))
    return rc;
  if (group < 1 || (int64_t)kv_heads * group > 65535 || total * group > 0x7fffffffLL)
    return api_fail("group %d: kv_heads * group must lie in [1, 65535], tokens * group below 2^31",
                    group);
  if (!std::isfinite(scale) || scale <= 0.f) return api_fail("scale must be positive and finite");
  if (!std::isfinite(decay)) return api_fail("decay must be finite");
  if (max_new < 1 || max_len < 0) return api_fail("max_new must be positive, max_len not negative");
  if (seqs == 0 || table_width == 0) return api_fail(nullptr);
  if (!lengths || !starts || !table || !weights || (total > 0 && (!q || !lse)))
    return api_fail("q, lse, lengths, starts, table and weights must be non-NULL");
  if (!k_pages || n_pages < 1) return api_fail("the pool is empty");
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_pages)) & 15u)
    return api_fail("q and the pool must be 16-byte aligned");
  if (q_token_stride % 8 || q_head_stride % 8)
    return api_fail("strides of q must be multiples of 8 elements");
  a.q = q;
  a.q_token = q_token_stride;
  a.q_head = q_head_stride;
  a.lse = lse;
  a.k_pages = k_pages;
  a.t = {table, lengths, starts, table_width, seqs, total, status};
  a.group = group;
  a.causal = causal != 0;
  a.dtype = dtype;
  a.scale = scale;
  a.decay = decay;
  a.weights = weights;
  clamp_expected(total, max_new, max_len);
  a.max_new = max_new;
  a.max_len = max_len;
  a.wait_ns = api_wait_ns();
  a.wait_selftest = api_wait_selftest();
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // Up to 40 rows per sequence and key head (and groups wider than a tile) go to
  // the warp-level kernel: 32 sequences over 32,768 keys of 128, in us,
  // warp-level against tcgen05: 20 rows 356 / 442, 32 rows 395 / 441, 64 rows
  // 594 / 451.
  const bool rows = max_new * group <= 40 || group > 128 || total == 0;
  return api_cuda(rows ? launch_paged_weigh_rows(a, st) : launch_paged_weigh_tc05(a, st));
}
