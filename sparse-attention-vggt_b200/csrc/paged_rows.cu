// Attention of a few new tokens (decode steps) over the paged cache.
//
// For a sequence and a key head the query rows (tokens x the head's group)
// are few, and every key and value is used by all of them: the pass is bound
// by reading K and V once.  So a CTA takes one tile of 16 rows and one
// run of key tiles, and what matters is that loads never pause:
//  * warp 4 streams 64-key K and V tiles by TMA (boxes of one page, 128-byte
//    swizzle) into a ring; page numbers are read 32 boxes ahead.  (Its 64-bit
//    counters cost what paged_producer.cuh says; long caches are at the memory's
//    rate all the same.)
//  * warps 0-3 share a tile's keys, 16 each; each keeps its own running
//    maximum, sum and output rows in registers (mma.sync m16n8k16, fp32), so no
//    warp waits for another before the end.  tcgen05 would spend M = 128 rows
//    on 16; it is as fast from 20 rows on (see paged_attn.cu).
//  * a long cache is cut into runs of `chunk` tiles, one CTA each; the CTA
//    that finishes last (a counter per item) joins the runs' results in their
//    order and leaves the counter at zero, so there is one launch and the
//    result does not depend on the order in which CTAs finish.
//
// P is rounded to the tensors' type for the product with V; maxima, sums and
// outputs are fp32, and the sums take P before it is rounded.  In fp16 the
// exponents are shifted up by 15, so that P <= 2^15 and probabilities down to
// 2^-29 of the row's largest keep all of the type's bits (with P <= 1 those of
// 2^-25 and less were lost to the product, though not to the sum); bf16 has the
// exponents of fp32.  So P's error is that of the output's own rounding.
#include <cuda.h>

#include <type_traits>

#include "kernels.h"
#include "mma.cuh"
#include "paged.cuh"
#include "paged_slow.cuh"
#include "tc05.cuh"

namespace vggt {
namespace {

constexpr int kTile = 64;  // keys per ring stage
constexpr int kThreads = 160;
constexpr int kRows = 16;
constexpr int kGroups = 4;              // warps that share a tile's keys
constexpr int kKeys = kTile / kGroups;  // keys of a warp in a tile
constexpr int kN = kKeys / 8;           // n-tiles of S

template <int D>
struct Ring {
  static constexpr int kHalves = D / 64;
  static constexpr uint32_t kMatrix = kTile * D * 2;  // bytes of one K or V tile
  static constexpr uint32_t kStage = 2 * kMatrix;
  static constexpr int kStages = D == 64 ? 6 : 3;  // 96 KB: two CTAs to an SM
  static constexpr uint32_t kBytes = kStages * kStage;
};

struct RowsParams {
  PagedAttnArgs a;
  float scale_log2;
  int64_t tiles, heads, splits;  // row tiles (upper bound), key heads, runs per item (most)
  int64_t chunk;                 // key tiles per run
  int* counters;                 // [tiles * heads], zero between calls
  float* partial;                // [tiles * heads][splits][rows * (D + 2)]
};

struct Shared {
  uint64_t full[8], empty[8], never;  // never: nothing arrives (wait self-test)
  int abort, last, odd;
  float m[4][kRows], l[4][kRows];  // per warp, then per row
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 2)
    paged_rows_kernel(const __grid_constant__ CUtensorMap tm_k,
                      const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ RowsParams p) {
  using R = Ring<D>;
  constexpr int kSteps = D / 16;
  constexpr float kShift = std::is_same<T, __half>::value ? 15.f : 0.f;
  extern __shared__ unsigned char raw[];
  unsigned char* ring = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
  const uint32_t ring_addr = smem_u32(ring);
  __shared__ Shared sh;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  // ---- which rows and which keys ----
  const int64_t split = blockIdx.x % p.splits, item = blockIdx.x / p.splits;
  const int head = (int)(item % p.heads);
  const PagedAttnArgs& a = p.a;
  RowTile rt;
  if (!locate_tile(a.t, a.pool, a.group, kRows, item / p.heads, rt)) {
    if (warp == 0) fill_rows_of_no_sequence<T, D>(a);
    return;
  }
  const int64_t len = rt.len;
  const int rows = rt.rows - rt.row0 < kRows ? rt.rows - rt.row0 : kRows;
  // keys that row r of the tile sees
  auto limit_of = [&](int r) -> int64_t {
    if (!a.causal) return len;
    const int64_t n = len - rt.n_new + (rt.row0 + r) / a.group + 1;
    return n < 0 ? 0 : (n < len ? n : len);
  };
  const int64_t most = limit_of(rows - 1), least = limit_of(0);
  const int64_t all_tiles = (most + kTile - 1) / kTile;
  int64_t chunk = (all_tiles + p.splits - 1) / p.splits;
  if (chunk < p.chunk) chunk = p.chunk;
  const int64_t runs = all_tiles > 0 ? (all_tiles + chunk - 1) / chunk : 1;
  if (split >= runs) {
    if (warp == 0) fill_rows_of_no_sequence<T, D>(a);
    return;
  }
  const int64_t tile0 = split * chunk;
  const int64_t tiles = all_tiles - tile0 < chunk ? all_tiles - tile0 : chunk;

  auto full = [&](int s) { return smem_u32(&sh.full[s]); };
  auto empty = [&](int s) { return smem_u32(&sh.empty[s]); };
  volatile int* abort_flag = &sh.abort;
  if (tid == 0) {
    for (int s = 0; s < R::kStages; ++s) {
      tc::mbar_init(full(s), 1);
      tc::mbar_init(empty(s), 4);
    }
    tc::mbar_init(smem_u32(&sh.never), 1);
    sh.abort = 0;
    sh.odd = 0;
    tc::mbar_fence_init();
  }
  __syncthreads();

  float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};
  float o[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) o[i][j] = 0.f;

  if (warp == 4) {
    // ================= TMA producer =================
    const int box = a.pool.page < kTile ? a.pool.page : kTile;  // slots per box
    const int boxes = kTile / box;                              // per tile: 1, 2 or 4
    const int ahead = 32 / boxes;                               // tiles per read of the table
    int page = -1;
    int64_t issued = 0;
    const bool go = !a.wait_selftest ||
                    __all_sync(0xffffffffu, tc::mbar_wait(smem_u32(&sh.never), 0, abort_flag, a.wait_ns));
    for (int64_t t = 0; go && t < tiles; ++t) {
      const int64_t key0 = (tile0 + t) * kTile;
      if (t % ahead == 0) {
        const int64_t slot = key0 + (int64_t)lane * box;
        page = (int)a.pool.n_pages;  // past the pool: reads as zeros
        if (slot < most && slot < (tile0 + tiles) * kTile) {
          const int got = checked_page(a.t, a.pool, rt.seq, slot >> a.pool.page_shift);
          if (got >= 0) page = got;
        }
      }
      const int stage = (int)(t % R::kStages);
      bool ok = true;
      if (t >= R::kStages)
        ok = tc::mbar_wait(empty(stage), (uint32_t)((t / R::kStages - 1) & 1), abort_flag,
                           a.wait_ns);
      if (!__all_sync(0xffffffffu, ok)) break;
      const int need = (int)((most - key0 + box - 1) / box);
      const int live = need < boxes ? need : boxes;
      const uint32_t dst = ring_addr + (uint32_t)stage * R::kStage;
      if (lane == 0)
        tc::mbar_expect_tx(full(stage), (uint32_t)(live * box) * D * 4u);
      __syncwarp();
      const int mine = __shfl_sync(0xffffffffu, page, (int)(t % ahead) * boxes + (lane & (boxes - 1)));
      // lane = box + boxes * (half + halves * matrix)
      if (lane < boxes * R::kHalves * 2 && (lane & (boxes - 1)) < live) {
        const int b = lane & (boxes - 1), rest = lane / boxes;
        const int half = rest % R::kHalves, matrix = rest / R::kHalves;
        const int row = (int)((key0 + b * box) & (a.pool.page - 1));
        tc::tma_load_4d(dst + matrix * R::kMatrix + half * (kTile * 128) + b * box * 128,
                        matrix ? &tm_v : &tm_k, full(stage), half * 64, row, head, mine);
      }
      ++issued;
    }
    // no copy may be in flight when the CTA leaves
    const int64_t from = issued > R::kStages ? issued - R::kStages : 0;
    for (int64_t t = from; t < issued; ++t)
      tc::mbar_wait_drain(full((int)(t % R::kStages)), (uint32_t)((t / R::kStages) & 1),
                          1000000000ull);
    fill_rows_of_no_sequence<T, D>(a);  // while the others finish
  } else {
    // ================= S, softmax, O =================
    const int kg = warp;
    const int r0 = lane >> 2;  // this thread's rows: r0, r0 + 8
    int64_t lim[2];
    uint32_t qf[kSteps][4];
    {
      const T* src[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = r0 + 8 * i;
        const int row = rt.row0 + (r < rows ? r : 0);
        // rows past the last one repeat the first: they mask nothing new
        lim[i] = limit_of(r < rows ? r : 0);
        src[i] = static_cast<const T*>(a.q) + (rt.first + row / a.group) * a.q_token +
                 ((int64_t)head * a.group + row % a.group) * a.q_head;
      }
#pragma unroll
      for (int k = 0; k < kSteps; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          qf[k][j] = __ldg(reinterpret_cast<const uint32_t*>(
              src[j & 1] + k * 16 + (j >> 1) * 8 + (lane & 3) * 2));
    }
    const int krow = ((lane >> 4) & 1) * 8 + (lane & 7), kchunk = (lane >> 3) & 1;
    const int vrow = ((lane >> 3) & 1) * 8 + (lane & 7), vchunk = (lane >> 4) & 1;
    for (int64_t t = 0; t < tiles; ++t) {
      const int stage = (int)(t % R::kStages);
      if (!__all_sync(0xffffffffu, tc::mbar_wait(full(stage), (uint32_t)((t / R::kStages) & 1),
                                                 abort_flag, a.wait_ns)))
        break;
      const uint32_t kbase = ring_addr + (uint32_t)stage * R::kStage + kg * kKeys * 128;
      const uint32_t vbase = kbase + R::kMatrix;
      float s[kN][4];
#pragma unroll
      for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[n][j] = 0.f;
#pragma unroll
      for (int n = 0; n < kN; n += 2) {
        const int key = n * 8 + krow;
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
          uint32_t b0, b1, b2, b3;
          const int c = (k & 3) * 2 + kchunk;
          ldsm_x4(kbase + (k >> 2) * (kTile * 128) + key * 128 + ((c ^ (key & 7)) << 4), b0, b1,
                  b2, b3);
          MmaOp<T>::mma(s[n], qf[k], b0, b1);
          MmaOp<T>::mma(s[n + 1], qf[k], b2, b3);
        }
      }
      const int64_t key0 = (tile0 + t) * kTile + kg * kKeys;  // this warp's first key
      const bool masked = key0 + kKeys > least;
      if (masked) {
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (key0 + n * 8 + (lane & 3) * 2 + (j & 1) >= lim[j >> 1]) s[n][j] = -INFINITY;
      }
      float base[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float mx = -INFINITY;
#pragma unroll
        for (int n = 0; n < kN; ++n) mx = fmaxf(mx, fmaxf(s[n][2 * i], s[n][2 * i + 1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        // less the shift, rounded up: no exponent passes the shift, however
        // large the scores are
        mx = fmaxf(m_run[i], __fmaf_ru(mx, p.scale_log2, -kShift));
        // a row that has seen nothing yet keeps a finite base, so that its
        // masked scores give 2^(-inf - 0) = 0
        base[i] = mx == -INFINITY ? 0.f : mx;
        const float f = fast_exp2(m_run[i] - base[i]);
        if (mx != m_run[i]) {
          l_run[i] *= f;
#pragma unroll
          for (int d = 0; d < D / 8; ++d) {
            o[d][2 * i] *= f;
            o[d][2 * i + 1] *= f;
          }
        }
        m_run[i] = mx;
      }
      uint32_t pf[kN / 2][4];
#pragma unroll
      for (int n = 0; n < kN; ++n) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float e0 = fast_exp2(fmaf(s[n][2 * i], p.scale_log2, -base[i]));
          const float e1 = fast_exp2(fmaf(s[n][2 * i + 1], p.scale_log2, -base[i]));
          l_run[i] += e0 + e1;
          pf[n >> 1][(n & 1) * 2 + i] = ElemOps<T>::pack2(e0, e1);
        }
      }
      bool odd = false;
#pragma unroll
      for (int kk = 0; kk < kN / 2; ++kk) {
        const int key = kk * 16 + vrow;
        // of the two keys in a register, those that hold a value of this pass
        uint32_t keep[2] = {0xffffffffu, 0xffffffffu}, part[2] = {0u, 0u};
        if (masked) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int64_t k0 = key0 + kk * 16 + j * 8 + (lane & 3) * 2;
            keep[j] = (k0 < most ? 0xffffu : 0u) | (k0 + 1 < most ? 0xffff0000u : 0u);
            part[j] = keep[j] & ((k0 >= least ? 0xffffu : 0u) | (k0 + 1 >= least ? 0xffff0000u : 0u));
          }
        }
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
          uint32_t b[4];
          const int c = (d & 3) * 2 + vchunk;
          ldsm_x4_t(vbase + (d >> 2) * (kTile * 128) + key * 128 + ((c ^ (key & 7)) << 4), b[0],
                    b[1], b[2], b[3]);
          if (masked) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              odd = odd || has_nonfinite<T>(b[j] & part[j & 1]);
              b[j] &= keep[j & 1];
            }
          }
          MmaOp<T>::mma(o[2 * d], pf[kk], b[0], b[1]);
          MmaOp<T>::mma(o[2 * d + 1], pf[kk], b[2], b[3]);
        }
      }
      if (odd) sh.odd = 1;
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(empty(stage));
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l_run[i] += __shfl_xor_sync(0xffffffffu, l_run[i], 1);
      l_run[i] += __shfl_xor_sync(0xffffffffu, l_run[i], 2);
      if ((lane & 3) == 0) {
        sh.m[kg][r0 + 8 * i] = m_run[i];
        sh.l[kg][r0 + 8 * i] = l_run[i];
      }
    }
  }
  __syncthreads();  // the ring is free now: its space takes the output rows
  float* obuf = reinterpret_cast<float*>(ring);  // [kGroups][kRows][D]
  if (warp < 4) {
    const int kg = warp;
    const int r0 = lane >> 2;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = r0 + 8 * i;
      float mx = sh.m[0][r];
#pragma unroll
      for (int g = 1; g < kGroups; ++g) mx = fmaxf(mx, sh.m[g][r]);
      const float f = fast_exp2(m_run[i] - (mx == -INFINITY ? 0.f : mx));
#pragma unroll
      for (int d = 0; d < D / 8; ++d) {
        float2 v = make_float2(o[d][2 * i] * f, o[d][2 * i + 1] * f);
        *reinterpret_cast<float2*>(obuf + (kg * kRows + r) * D + d * 8 + (lane & 3) * 2) = v;
      }
    }
  }
  __syncthreads();
  float rm = -INFINITY, rl = 0.f;
  if (tid < kRows) {
#pragma unroll
    for (int g = 0; g < kGroups; ++g) rm = fmaxf(rm, sh.m[g][tid]);
#pragma unroll
    for (int g = 0; g < kGroups; ++g)
      rl += sh.l[g][tid] * fast_exp2(sh.m[g][tid] - (rm == -INFINITY ? 0.f : rm));
  }
  __syncthreads();
  if (tid < kRows) {
    sh.m[0][tid] = rm;
    sh.l[0][tid] = rl;
  }
  for (int i = tid; i < kRows * D; i += kThreads) {
    float v = obuf[i];
#pragma unroll
    for (int g = 1; g < kGroups; ++g) v += obuf[g * kRows * D + i];
    obuf[i] = v;
  }
  __syncthreads();
  if (sh.odd) {
    // a value that only some rows see is not finite: zero times it is not
    // zero, so the rows are formed key by key
    for (int r = warp; r < rows; r += kThreads / 32)
      slow_row<T, D>(a, rt, r, head, p.scale_log2, tile0 * kTile, (tile0 + tiles) * kTile,
                     limit_of(r), obuf + r * D, &sh.m[0][r], &sh.l[0][r]);
    __syncthreads();
  }
  if (tid == 0 && sh.abort) raise_status(a.t.status, VGGT_STATUS_TIMEOUT);

  if (runs > 1) {
    float* part = p.partial + (item * p.splits + split) * (int64_t)(kRows * (D + 2));
    for (int i = tid; i < kRows * D / 4; i += kThreads)
      reinterpret_cast<float4*>(part)[i] = reinterpret_cast<const float4*>(obuf)[i];
    if (tid < kRows) {
      part[kRows * D + tid] = sh.m[0][tid];
      part[kRows * (D + 1) + tid] = sh.l[0][tid];
    }
    __threadfence();
    __syncthreads();
    if (tid == 0) {
      const int before = atomicAdd(p.counters + item, 1);
      sh.last = before == (int)runs - 1;
      if (sh.last) p.counters[item] = 0;
    }
    __syncthreads();
    if (!sh.last) return;
    __threadfence();
    // the runs' maxima and sums, then the rows, 4 vectors of 4 runs in flight
    constexpr int64_t kRun = kRows * (D + 2);
    const float* from = p.partial + item * p.splits * kRun;
    float* wgt = obuf + kRows * D;        // [runs][kRows], 64 runs at most
    float* sums = wgt + 64 * kRows;
    for (int i = tid; i < (int)runs * kRows; i += kThreads) {
      const float* ml = from + (i / kRows) * kRun + kRows * D + i % kRows;
      wgt[i] = __ldcg(ml);
      sums[i] = __ldcg(ml + kRows);
    }
    __syncthreads();
    if (tid < kRows) {
      float mx = -INFINITY, l = 0.f;
      for (int s = 0; s < (int)runs; ++s) mx = fmaxf(mx, wgt[s * kRows + tid]);
      for (int s = 0; s < (int)runs; ++s) {
        const float f = fast_exp2(wgt[s * kRows + tid] - (mx == -INFINITY ? 0.f : mx));
        wgt[s * kRows + tid] = f;
        l = fmaf(f, sums[s * kRows + tid], l);
      }
      sh.m[0][tid] = mx;
      sh.l[0][tid] = l;
    }
    __syncthreads();
    constexpr int kBatch = 4;
    for (int i0 = tid; i0 < kRows * D / 4; i0 += kBatch * kThreads) {
      float4 acc[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) acc[j] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int s = 0; s < (int)runs; ++s) {
        const float4* src = reinterpret_cast<const float4*>(from + s * kRun);
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          const int i = i0 + j * kThreads;
          if (i < kRows * D / 4) {
            const float4 v = __ldcg(src + i);
            const float f = wgt[s * kRows + i / (D / 4)];
            acc[j].x = fmaf(f, v.x, acc[j].x);
            acc[j].y = fmaf(f, v.y, acc[j].y);
            acc[j].z = fmaf(f, v.z, acc[j].z);
            acc[j].w = fmaf(f, v.w, acc[j].w);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (i0 + j * kThreads < kRows * D / 4)
          reinterpret_cast<float4*>(obuf)[i0 + j * kThreads] = acc[j];
    }
    __syncthreads();
  }
  // ---- out = O / l, lse = (m + log2 l) ln 2; a row without keys: 0, -inf ----
  for (int i = tid; i < rows * (D / 4); i += kThreads) {
    const int r = i / (D / 4), d = (i % (D / 4)) * 4;
    const int row = rt.row0 + r;
    const float l = sh.l[0][r];
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const float4 v = *reinterpret_cast<const float4*>(obuf + r * D + d);
    T* dst = static_cast<T*>(a.out) + (rt.first + row / a.group) * a.o_token +
             ((int64_t)head * a.group + row % a.group) * a.o_head + d;
    *reinterpret_cast<uint2*>(dst) = make_uint2(ElemOps<T>::pack2(v.x * inv, v.y * inv),
                                                ElemOps<T>::pack2(v.z * inv, v.w * inv));
  }
  if (a.lse != nullptr && tid < rows) {
    const int row = rt.row0 + tid;
    const float l = sh.l[0][tid];
    a.lse[(rt.first + row / a.group) * (p.heads * a.group) + (int64_t)head * a.group +
          row % a.group] =
        l == 0.f ? -INFINITY : (sh.m[0][tid] + log2f(l)) * 0.6931471805599453f;
  }
}

template <typename T, int D>
cudaError_t launch_rows(const RowsParams& p, const CUtensorMap& mk, const CUtensorMap& mv,
                        cudaStream_t st) {
  auto kernel = paged_rows_kernel<T, D>;
  const size_t smem = Ring<D>::kBytes + 1024;
  const cudaError_t e =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  kernel<<<(unsigned)(p.tiles * p.heads * p.splits), kThreads, smem, st>>>(mk, mv, p);
  return cudaGetLastError();
}

}  // namespace

PagedPlan paged_rows_plan(int64_t total, int64_t seqs, int kv_heads, int group, int dim,
                          int64_t max_len) {
  PagedPlan plan{};
  plan.rows = kRows;
  plan.tiles = most_tiles(total, seqs, group, plan.rows);
  const int64_t items = plan.tiles * kv_heads;
  const int64_t key_tiles = (max_len + kTile - 1) / kTile;
  // Runs per row tile, in microseconds as measured: a CTA takes 0.63 a key tile
  // (dim 64), twice that where K and V rows are twice as wide; 5 to start, 3
  // more where two share an SM; joining 3 and 0.1 a run.  Beyond one wave of
  // 296, sequences of different lengths leave half a run idle at the end.  One
  // token over 1,375 keys in 16 heads: 8 runs 11.6 us, 1 run 19.9, 11 runs
  // 15.6; over 43,001 keys: 16 runs 43.5, 8 runs 64.4, 22 runs 69.1.
  const double tile_us = dim == 64 ? 0.63 : 1.26;
  double best = -1;
  plan.splits = 1;
  for (int64_t s = 1; s <= 64 && (s == 1 || (s <= key_tiles && items <= kMaxCounters)); ++s) {
    const int64_t ctas = items * s;
    const double run = (double)((key_tiles + s - 1) / s) * tile_us;
    const double waves = ctas > 296 ? (double)ctas / 296 : 1.0;
    const double cost = waves * (run + (ctas > 148 ? 8 : 5)) + (ctas > 296 ? 0.5 * run : 0) +
                        (s > 1 ? 3 + 0.1 * s : 0);
    if (best < 0 || cost < best) {
      best = cost;
      plan.splits = s;
    }
  }
  plan.chunk = key_tiles > 0 ? (key_tiles + plan.splits - 1) / plan.splits : 1;
  plan.partial_bytes =
      plan.splits > 1 ? (size_t)items * plan.splits * kRows * (dim + 2) * 4 : 0;
  return plan;
}

cudaError_t launch_paged_rows(const PagedAttnArgs& a, const PagedPlan& plan, cudaStream_t st) {
  RowsParams p;
  p.a = a;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.tiles = plan.tiles;
  p.heads = a.pool.kv_heads;
  p.splits = plan.splits;
  p.chunk = plan.chunk;
  p.counters = static_cast<int*>(a.workspace);
  p.partial = reinterpret_cast<float*>(static_cast<char*>(a.workspace) + kMaxCounters * 4);
  if (plan.tiles == 0) return cudaSuccess;
  if (p.tiles * p.heads * p.splits > 0x7fffffffLL) return cudaErrorInvalidValue;
  CUtensorMap mk, mv;
  const uint32_t box = (uint32_t)(a.pool.page < kTile ? a.pool.page : kTile);
  if (!encode_pool_tmap(&mk, a.k_pages, a.dtype, a.pool, box) ||
      !encode_pool_tmap(&mv, a.v_pages, a.dtype, a.pool, box))
    return cudaErrorInvalidValue;
  if (a.dtype == VGGT_DTYPE_BF16)
    return a.pool.dim == 64 ? launch_rows<__nv_bfloat16, 64>(p, mk, mv, st)
                            : launch_rows<__nv_bfloat16, 128>(p, mk, mv, st);
  return a.pool.dim == 64 ? launch_rows<__half, 64>(p, mk, mv, st)
                          : launch_rows<__half, 128>(p, mk, mv, st);
}

}  // namespace vggt
