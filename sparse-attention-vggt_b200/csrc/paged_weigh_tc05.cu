// Accumulated attention weight of a chunk of new tokens on the 5th-generation
// tensor cores: w_j = decay * w_j + sum_i exp(s_ij - lse_i) for every cached
// key j of a key head, over the rows i (new tokens x the head's group) that
// see it.
//
// The product is turned over, S^T = K Q^T: a tile has 128 keys in TMEM's lanes
// and up to 128 rows in its columns.  A thread then owns one key and adds its
// probabilities up in registers, in a fixed order, with no maximum, no
// reduction between threads and no product after it.
//   warp 0     streams Q tiles (TMA: whole tokens, the group's heads side by
//              side), the rows' log-sum-exps, and K tiles (a box per page)
//   warp 1     issues S^T (both operands in shared memory, N = 128; double-
//              buffered in TMEM)
//   warps 2-5  exponentials, one key per thread
// A CTA walks through a run of key tiles of one sequence and head, all row
// tiles for each; two CTAs share an SM.
//
// What bounds it: 128 x 128 exponentials cost the multi-function unit 1,024
// clocks, the MMAs 256 (dim 64) or 512; so two column pairs of eight take a
// polynomial (error 2.7e-6) on the FMA pipe.  One frame of 1,374 tokens over
// 43,968 keys in 16 heads: 297 us (303 at three pairs of eight, 331 at four).
// Two exponential warps share an SM's quarter; 32 columns take the two some 520
// clocks, where the unit needs 384: they wait for one another's results.  That
// is a third of the time: without the exponentials the frame takes 202 us, and
// without the arithmetic on S 181, which are the tile's own chain of loads from
// TMEM and waits (a Q tile is loaded again for every 128 keys, 1.3 GB of tiles in
// all, but L2 is at 16 % of its rate).  Eight exponential warps instead of four
// were slower (356 us against 341 then).
#include <cuda.h>

#include <type_traits>

#include "exp2.cuh"
#include "kernels.h"
#include "paged.cuh"
#include "tc05.cuh"

namespace vggt {
namespace {

constexpr int kKeys = 128, kCols = 128, kThreads = 192;
constexpr int kLseStages = 4;
constexpr uint32_t kTmemCols = 256;
constexpr uint64_t kDrainNs = 1000000000ull;
// column pairs of every 8 whose exponentials take the polynomial
constexpr unsigned kPolyPairs = 0x11u;

template <int D>
struct Smem {
  static constexpr int kHalves = D / 64;
  static constexpr uint32_t kHalf = 128 * 128;  // 128 rows of 64 elements
  static constexpr uint32_t kTile = kHalves * kHalf;
  // 96 KB in all
  static constexpr int kKStages = D == 64 ? 2 : 1;
  static constexpr int kStages = D == 64 ? 4 : 2;  // of Q
  static constexpr uint32_t kK = 0;
  static constexpr uint32_t kQ = kK + kKStages * kTile;
  static constexpr uint32_t kEnd = kQ + kStages * kTile;
};

struct Bars {
  uint64_t k_full[2], k_empty[2], q_full[4], q_empty[4], lse_empty[kLseStages];
  uint64_t s_full[2], s_empty[2], drain, never;  // never: nothing arrives (wait self-test)
};

struct WeighTcParams {
  WeighArgs a;
  float scale_log2;
  int64_t splits, chunk;  // CTAs per sequence and head, key tiles per CTA (least)
  int tokens;             // per row tile: floor(128 / group)
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 2)
    weigh_tc05_kernel(const __grid_constant__ CUtensorMap tm_k,
                      const __grid_constant__ CUtensorMap tm_q,
                      const __grid_constant__ WeighTcParams p) {
  using L = Smem<D>;
  constexpr int kHalves = L::kHalves, kStages = L::kStages;
  extern __shared__ unsigned char raw[];
  unsigned char* sbase = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
  const uint32_t base = smem_u32(sbase);
  __shared__ Bars bars;
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  __shared__ __align__(16) float s_lse[kLseStages][kCols];  // minus lse, in units of log2
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const WeighArgs& a = p.a;

  const int64_t split = blockIdx.x % p.splits, item = blockIdx.x / p.splits;
  const int head = (int)(item % a.pool.kv_heads);
  const int64_t seq = item / a.pool.kv_heads;
  const int64_t len = checked_length(a.t, a.pool, seq);
  int64_t first;
  const int n_new = (int)checked_rows(a.t, seq, first);
  const int group = a.group, tile_rows = p.tokens * group;
  const int64_t all_tiles = (len + kKeys - 1) / kKeys;
  int64_t chunk = (all_tiles + p.splits - 1) / p.splits;
  if (chunk < p.chunk) chunk = p.chunk;
  const int64_t tile0 = split * chunk;
  if (tile0 >= all_tiles) return;
  const int tiles = (int)(all_tiles - tile0 < chunk ? all_tiles - tile0 : chunk);
  const int row_tiles = (n_new + p.tokens - 1) / p.tokens;
  // key j is seen by the new tokens from number j - past on (causal)
  const int64_t past = len - n_new;
  // the first row tile that sees a key of key tile kt
  auto first_row_tile = [&](int kt) -> int {
    if (!a.causal) return 0;
    const int64_t token = (tile0 + kt) * kKeys - past;
    return token <= 0 ? 0 : (int)(token / p.tokens);  // the last token sees the last key
  };

  volatile int* abort_flag = &s_abort;
  if (tid == 0) {
    for (int s = 0; s < 2; ++s) {
      tc::mbar_init(smem_u32(&bars.k_full[s]), 1);
      tc::mbar_init(smem_u32(&bars.k_empty[s]), 1);
      tc::mbar_init(smem_u32(&bars.s_full[s]), 2);  // the MMAs, and the rows' lse in place
      tc::mbar_init(smem_u32(&bars.s_empty[s]), 4);
    }
    for (int s = 0; s < kStages; ++s) {
      tc::mbar_init(smem_u32(&bars.q_full[s]), 33);  // the copies, and each lane's lse
      tc::mbar_init(smem_u32(&bars.q_empty[s]), 1);
    }
    for (int s = 0; s < kLseStages; ++s) tc::mbar_init(smem_u32(&bars.lse_empty[s]), 4);
    tc::mbar_init(smem_u32(&bars.drain), 1);
    tc::mbar_init(smem_u32(&bars.never), 1);
    s_abort = 0;
    tc::mbar_fence_init();
  }
  // Rows of a Q tile past tile_rows are never loaded.  They hold the last token,
  // which sees every key, with lse +inf: that gives nothing, or NaN where the
  // token itself does.  (Zeros would give NaN against a key with an infinite
  // element, whose scores may all be -inf; to mask the columns in every tile
  // took a frame with groups of three and seven a third longer.)
  if (n_new > 0) {
    const T* last = static_cast<const T*>(a.q) + (first + n_new - 1) * a.q_token +
                    (int64_t)head * group * a.q_head;
    const int pad = kCols - tile_rows;
    for (int i = tid; i < pad * (D / 8); i += kThreads) {
      const int r = tile_rows + i / (D / 8), c = i % (D / 8);
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(last) + c);
      for (int s = 0; s < kStages; ++s)
        *reinterpret_cast<uint4*>(sbase + L::kQ + s * L::kTile + (c >> 3) * L::kHalf + r * 128 +
                                  (((c & 7) ^ (r & 7)) << 4)) = v;
    }
  }
  for (int i = tid; i < kLseStages * kCols; i += kThreads) s_lse[i / kCols][i % kCols] = -INFINITY;
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  if (warp == 1) {
    tc::tmem_alloc(smem_u32(&s_tmem), kTmemCols);
    tc::tmem_relinquish();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = s_tmem;
  auto wait = [&](uint32_t bar, uint32_t parity) {
    return tc::warp_wait(bar, parity, abort_flag, a.wait_ns);
  };
  const uint32_t kfull0 = smem_u32(&bars.k_full[0]), kempty0 = smem_u32(&bars.k_empty[0]);
  const uint32_t qfull0 = smem_u32(&bars.q_full[0]), qempty0 = smem_u32(&bars.q_empty[0]);
  const uint32_t lempty0 = smem_u32(&bars.lse_empty[0]);
  const uint32_t sfull0 = smem_u32(&bars.s_full[0]), sempty0 = smem_u32(&bars.s_empty[0]);

  if (warp == 0) {
    // ================= producer =================
    const int64_t first_slot = tile0 * kKeys;
    const int keys = (int)(len - first_slot);
    const int32_t* table = a.t.table + seq * a.t.width;
    const int page_mask = a.pool.page - 1;
    const int64_t q_heads = (int64_t)a.pool.kv_heads * group;
    const float* lse = a.lse + first * q_heads + (int64_t)head * group;
    // minus the log-sum-exps of this lane's rows of a row tile, in units of
    // log2; -inf for rows without keys and rows that are not there
    int64_t lse_at[kCols / 32];
#pragma unroll
    for (int i = 0; i < kCols / 32; ++i) {
      const int r = lane + 32 * i;
      lse_at[i] = (r / group) * q_heads + r % group;
    }
    auto load_lse = [&](int rt, float* v) {
      const float* at = lse + (int64_t)rt * p.tokens * q_heads;
      const int rows = (n_new - rt * p.tokens) * group;
#pragma unroll
      for (int i = 0; i < kCols / 32; ++i) {
        const int r = lane + 32 * i;
        const float x = r < rows && r < tile_rows ? __ldg(at + lse_at[i]) : -INFINITY;
        v[i] = x == -INFINITY ? x : -1.4426950408889634f * x;
      }
    };
    int n_k = 0, n_q = 0;  // tiles loaded
    bool ok = true;
    for (int kt = 0; ok && kt < tiles && row_tiles > 0; ++kt) {
      const int rt0 = first_row_tile(kt);
      {
        // ---- the K tile: 8 boxes of 16 slots at most ----
        const int stage = n_k % L::kKStages, key0 = kt * kKeys;
        const int box = a.pool.page < kKeys ? a.pool.page : kKeys, boxes = kKeys / box;
        int page = (int)a.pool.n_pages;  // past the pool: reads as zeros
        const int key = key0 + lane * box;
        if (lane < boxes && key < keys) {
          const int got = __ldg(table + ((first_slot + key) >> a.pool.page_shift));
          if (got >= 0 && got < a.pool.n_pages)
            page = got;
          else
            raise_status(a.t.status, VGGT_STATUS_BAD_PAGE);
        }
        if (n_k >= L::kKStages)
          ok = wait(kempty0 + 8u * stage, (uint32_t)(n_k / L::kKStages + 1) & 1u);
        if (!ok) break;
        int live = (keys - key0 + box - 1) / box;
        live = live < boxes ? live : boxes;
        if (lane == 0) tc::mbar_expect_tx(kfull0 + 8u * stage, (uint32_t)(live * box) * D * 2u);
        __syncwarp();
        for (int b = 0; b < live; ++b) {
          const int at = __shfl_sync(0xffffffffu, page, b);
          if (tc::elect_one())
            for (int h = 0; h < kHalves; ++h)
              tc::tma_load_4d(base + L::kK + stage * L::kTile + h * L::kHalf + b * box * 128, &tm_k,
                              kfull0 + 8u * stage, h * 64,
                              (int)((first_slot + key0 + b * box) & page_mask), head, at);
          __syncwarp();
        }
        ++n_k;
      }
      float next[kCols / 32];
      load_lse(rt0, next);
      for (int rt = rt0; rt < row_tiles; ++rt) {
        const int stage = n_q % kStages;
        float mine[kCols / 32];
#pragma unroll
        for (int i = 0; i < kCols / 32; ++i) mine[i] = next[i];
        if (rt + 1 < row_tiles) load_lse(rt + 1, next);  // on their way during the wait
        if (n_q >= kStages) ok = wait(qempty0 + 8u * stage, (uint32_t)(n_q / kStages + 1) & 1u);
        if (!ok) break;
        if (tc::elect_one()) {
          tc::mbar_expect_tx(qfull0 + 8u * stage, (uint32_t)tile_rows * D * 2u);
#pragma unroll
          for (int h = 0; h < kHalves; ++h)
            tc::tma_load_3d(base + L::kQ + stage * L::kTile + h * L::kHalf, &tm_q,
                            qfull0 + 8u * stage, h * 64, head * group,
                            (int)first + rt * p.tokens);
        }
        __syncwarp();
        const int slot = n_q % kLseStages;
        if (n_q >= kLseStages)
          ok = wait(lempty0 + 8u * slot, (uint32_t)(n_q / kLseStages + 1) & 1u);
#pragma unroll
        for (int i = 0; i < kCols / 32; ++i)
          if (lane + 32 * i < tile_rows) s_lse[slot][lane + 32 * i] = mine[i];
        tc::mbar_arrive(qfull0 + 8u * stage);
        ++n_q;
      }
    }
    // no copy may be in flight when the CTA leaves
    for (int t = n_k > L::kKStages ? n_k - L::kKStages : 0; t < n_k; ++t)
      tc::mbar_wait_drain(kfull0 + 8u * (t % L::kKStages), (uint32_t)((t / L::kKStages) & 1),
                          kDrainNs);
    for (int t = n_q > kStages ? n_q - kStages : 0; t < n_q; ++t)
      tc::mbar_wait_drain(qfull0 + 8u * (t % kStages), (uint32_t)((t / kStages) & 1), kDrainNs);
  } else if (warp == 1) {
    // ================= MMA issuer =================
    const uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    const uint32_t id = tc::idesc_f16(fmt, 0u, kKeys, kCols);
    const uint64_t kdesc0 = tc::sw128_desc(base + L::kK, 16);
    const uint64_t qdesc0 = tc::sw128_desc(base + L::kQ, 16);
    int n_k = 0, n = 0;
    bool ok = !a.wait_selftest || wait(smem_u32(&bars.never), 0);
    for (int kt = 0; ok && kt < tiles && row_tiles > 0; ++kt) {
      const int rt0 = first_row_tile(kt);
      const int kstage = n_k % L::kKStages;
      ok = wait(kfull0 + 8u * kstage, (uint32_t)(n_k / L::kKStages) & 1u);
      const uint64_t kdesc = kdesc0 + (uint64_t)(kstage * (L::kTile / 16));
      for (int rt = rt0; ok && rt < row_tiles; ++rt, ++n) {
        const int stage = n % kStages, buf = n & 1;
        ok = (n < 2 || wait(sempty0 + 8u * buf, (uint32_t)((n >> 1) + 1) & 1u)) &&
             wait(qfull0 + 8u * stage, (uint32_t)(n / kStages) & 1u);
        if (!ok) break;
        tc::tc_fence_after();
        if (tc::elect_one()) {
          const uint64_t qdesc = qdesc0 + (uint64_t)(stage * (L::kTile / 16));
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint64_t off = (uint64_t)((kk >> 2) * (L::kHalf / 16) + (kk & 3) * 2);
            tc::mma_ss(tmem + 128u * buf, kdesc + off, qdesc + off, id, kk > 0 ? 1u : 0u);
          }
          tc::mbar_arrive(sfull0 + 8u * buf);  // passes on what q_full said of the lse
          tc::mma_commit(sfull0 + 8u * buf);
          tc::mma_commit(qempty0 + 8u * stage);
          if (rt == row_tiles - 1) tc::mma_commit(kempty0 + 8u * kstage);
        }
        __syncwarp();
      }
      ++n_k;
    }
    if (tc::elect_one()) tc::mma_commit(smem_u32(&bars.drain));
    __syncwarp();
    tc::mbar_wait_drain(smem_u32(&bars.drain), 0, kDrainNs);
  } else {
    // ================= exponentials: one key per thread =================
    const int sub = warp & 3;
    const uint32_t lane_off = (uint32_t)(sub * 32) << 16;
    const float_pair c2 = pack_pair(p.scale_log2, p.scale_log2);
    const Exp2Poly poly;
    float* w = a.weights + (seq * a.pool.kv_heads + head) * (a.t.width << a.pool.page_shift);
    const int64_t key_at = tile0 * kKeys + sub * 32 + lane;
    if (row_tiles == 0) {  // no new tokens
      for (int kt = 0; kt < tiles; ++kt)
        if (key_at + kt * kKeys < len)
          w[key_at + kt * kKeys] = new_weight(w[key_at + kt * kKeys], a.decay, 0.f);
    }
    // The tiles in a row, those of the next key tile behind the last row tile.
    // A part's 32 columns are loaded under the exponentials of the part before,
    // over the tiles' borders too.
    int n = 0, kt = 0, rt = first_row_tile(0), at = -1;
    bool ok = row_tiles == 0 || wait(sfull0, 0);
    uint32_t s[2][32];
    if (ok && row_tiles > 0) {
      tc::tc_fence_after();
      tc::tmem_ld32(tmem + lane_off, s[0]);
    }
    float old = 0.f;
    float_pair sum[2] = {};
    int64_t from = 0;  // rows from this one on see the key
    int plain_rt = 0;  // row tiles from this one to the last but one need no mask
    while (ok && row_tiles > 0 && kt < tiles) {
      const int64_t key = key_at + kt * kKeys;
      if (kt != at) {
        at = kt;
        old = key < len ? w[key] : 0.f;
        sum[0] = sum[1] = pack_pair(0.f, 0.f);
        if (a.causal) {
          from = (key - past) * group;
          const int64_t all = __shfl_sync(0xffffffffu, from, 31);  // see the warp's last key
          plain_rt = all > 0 ? (int)((all + tile_rows - 1) / tile_rows) : 0;
        }
      }
      const int slot = n % kLseStages, buf = n & 1;
      const uint32_t t_s = tmem + lane_off + 128u * buf;
      const uint32_t t_next = tmem + lane_off + 128u * (buf ^ 1);
      int next_kt = kt, next_rt = rt + 1;
      if (next_rt == row_tiles) {
        ++next_kt;
        next_rt = next_kt < tiles ? first_row_tile(next_kt) : 0;
      }
      // Tiles that need no mask take a copy without its branches, so that the
      // compiler orders a part's instructions among one another (a frame: 338
      // us where every part asks, 297).
      auto walk = [&](auto masked) {
        // This thread's key is seen by the columns [lo, left); the warp's keys by
        // none below lo_warp and by all from hi_warp on.
        int lo = 0, lo_warp = 0, hi_warp = 0, left = kCols;
        if (decltype(masked)::value) {
          const int64_t r0 = (int64_t)rt * tile_rows;
          left = (n_new - rt * p.tokens) * group;
          lo = (int)(from - r0 < 0 ? 0 : (from - r0 < kCols ? from - r0 : kCols));
          lo_warp = __shfl_sync(0xffffffffu, lo, 0);
          hi_warp = __shfl_sync(0xffffffffu, lo, 31);
        }
#pragma unroll
        for (int part = 0; part < 4; ++part) {
          const int col0 = 32 * part;
          tc::tmem_wait_ld();
          if (part < 3) {
            tc::tmem_ld32(t_s + 32u * (part + 1), s[(part + 1) & 1]);
          } else {
            // S_t is read
            tc::tc_fence_before();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(sempty0 + 8u * buf);
            if (next_kt < tiles) {
              ok = wait(sfull0 + 8u * (buf ^ 1), (uint32_t)((n + 1) >> 1) & 1u);
              if (!ok) return;
              tc::tc_fence_after();
              tc::tmem_ld32(t_next, s[0]);
            }
          }
          if (decltype(masked)::value && (col0 >= left || col0 + 32 <= lo_warp)) continue;
          uint32_t* sc = s[part & 1];
          if (decltype(masked)::value && (col0 + 32 > left || col0 < hi_warp)) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (col0 + i < lo || col0 + i >= left) sc[i] = __float_as_uint(-INFINITY);
          }
          const float4* minus = reinterpret_cast<const float4*>(&s_lse[slot][col0]);
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            const float4 m = minus[i / 2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const float_pair x = fma_pair(pack_pair(__uint_as_float(sc[2 * (i + j)]),
                                                      __uint_as_float(sc[2 * (i + j) + 1])),
                                            c2, j ? pack_pair(m.z, m.w) : pack_pair(m.x, m.y));
              if ((kPolyPairs >> ((i + j) & 7)) & 1u) {
                float_pair q, scale;
                poly(q, scale, x);
                sum[j] = fma_pair(q, scale, sum[j]);
              } else {
                float ea, eb;
                unpack_pair(ea, eb, x);
                sum[j] = add_pair(sum[j], pack_pair(fast_exp2(ea), fast_exp2(eb)));
              }
            }
          }
        }
      };
      if (rt < plain_rt || rt == row_tiles - 1)
        walk(std::true_type{});
      else
        walk(std::false_type{});
      if (!ok) break;
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(lempty0 + 8u * slot);
      if (next_kt != kt && key < len) {
        float x, y;
        unpack_pair(x, y, add_pair(sum[0], sum[1]));
        w[key] = new_weight(old, a.decay, x + y);
      }
      kt = next_kt;
      rt = next_rt;
      ++n;
    }
    tc::tmem_wait_ld();
  }

  tc::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, kTmemCols);
  }
  if (tid == 0 && s_abort) raise_status(a.t.status, VGGT_STATUS_TIMEOUT);
}

template <typename T, int D>
cudaError_t launch_weigh_tc05(const WeighTcParams& p, const CUtensorMap& mk, const CUtensorMap& mq,
                              cudaStream_t st) {
  auto kernel = weigh_tc05_kernel<T, D>;
  const size_t smem = Smem<D>::kEnd + 1024;
  const cudaError_t e =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  kernel<<<(unsigned)(p.a.t.seqs * p.a.pool.kv_heads * p.splits), kThreads, smem, st>>>(mk, mq, p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_paged_weigh_tc05(const WeighArgs& a, cudaStream_t st) {
  WeighTcParams p;
  p.a = a;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.tokens = kCols / a.group;
  const int64_t items = a.t.seqs * a.pool.kv_heads;
  const int64_t key_tiles = (a.max_len + kKeys - 1) / kKeys;
  const int64_t row_tiles = (a.max_new + p.tokens - 1) / p.tokens;
  // key tiles per CTA: the number that ends the last wave of 2 CTAs per SM
  // soonest, a CTA's start and end counted as six tiles of 128 x 128
  const int64_t slots = 2 * 148;
  p.splits = 1;
  int64_t best = -1;
  for (int64_t s = 1; s <= key_tiles; s += s < 64 ? 1 : s / 32) {
    const int64_t waves = (items * s + slots - 1) / slots;
    const int64_t cost = waves * (((key_tiles + s - 1) / s) * row_tiles + 6);
    if (best < 0 || cost < best) {
      best = cost;
      p.splits = s;
    }
  }
  p.chunk = key_tiles > 0 ? (key_tiles + p.splits - 1) / p.splits : 1;
  if (items * p.splits > 0x7fffffffLL) return cudaErrorInvalidValue;
  CUtensorMap mk, mq;
  const uint32_t box = (uint32_t)(a.pool.page < kKeys ? a.pool.page : kKeys);
  const uint64_t dims[3] = {(uint64_t)a.pool.dim, (uint64_t)a.pool.kv_heads * a.group,
                            (uint64_t)a.t.total};
  const uint64_t strides[2] = {(uint64_t)a.q_head * 2, (uint64_t)a.q_token * 2};
  const uint32_t qbox[3] = {64, (uint32_t)a.group, (uint32_t)p.tokens};
  if (!encode_pool_tmap(&mk, a.k_pages, a.dtype, a.pool, box) ||
      !encode_tmap_sw128(&mq, a.q, a.dtype, 3, dims, strides, qbox))
    return cudaErrorInvalidValue;
  if (a.dtype == VGGT_DTYPE_BF16)
    return a.pool.dim == 64 ? launch_weigh_tc05<__nv_bfloat16, 64>(p, mk, mq, st)
                            : launch_weigh_tc05<__nv_bfloat16, 128>(p, mk, mq, st);
  return a.pool.dim == 64 ? launch_weigh_tc05<__half, 64>(p, mk, mq, st)
                          : launch_weigh_tc05<__half, 128>(p, mk, mq, st);
}

}  // namespace vggt
