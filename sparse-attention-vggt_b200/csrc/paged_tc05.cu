// Attention of a chunk of new tokens over the paged cache on the
// 5th-generation tensor cores.
//
// A CTA takes 128 query rows of a sequence and key head (tokens x the head's
// group, so grouped heads fill the tile) and one run of 64-key tiles:
//   warp 0     streams K and V tiles by TMA, a box per page (or per 64 slots
//              of a larger page), into two rings; page numbers are read 32
//              boxes ahead, one lane issues one box
//   warp 1     one lane issues S_t = Q K_t^T (Q, K in shared memory, S double-
//              buffered in TMEM) and O += P_t V_t (P read from TMEM, where it
//              overwrote S_t; O stays in TMEM for the whole run)
//   warps 2-5  softmax, one query row per thread
// Two CTAs share an SM, so that one's softmax runs under the other's MMAs.
//
// The row's reference maximum moves only when a tile's maximum exceeds it by
// more than 2^8 in the exp2 domain; O is rescaled then.  P is published in
// two halves, so that the first half's product runs under the second half's
// exponentials.  Sums are fp32, of the exponentials before P is rounded: the
// log-sum-exp is good to fp32 and only the product with V sees the rounding.
//
// What bounds it: the multi-function unit gives 16 exponentials per clock and
// SM, so a 128 x 64 tile costs 512 clocks there, against 256 (dim 64) or 512
// (dim 128) of MMA at full rate.  Therefore some column pairs take a
// polynomial on the FMA pipe instead.
//
// Slots past the last key that any row sees are cleared in shared memory
// before their product (their content is not defined).  A key that only later
// rows of the tile see is masked to P = 0; if its value is not finite, the
// tile's rows are formed key by key instead.
#include <cuda.h>

#include <type_traits>

#include "exp2.cuh"
#include "kernels.h"
#include "paged.cuh"
#include "paged_slow.cuh"
#include "tc05.cuh"

namespace vggt {
namespace {

constexpr int kRows = 128, kTile = 64, kThreads = 192;
constexpr uint32_t kTmemCols = 256;  // S0 | S1 | O
constexpr uint64_t kDrainNs = 1000000000ull;

template <int D>
struct Smem {
  static constexpr int kHalves = D / 64;
  static constexpr uint32_t kMatrix = kTile * D * 2;  // one K or V tile
  static constexpr int kStages = D == 64 ? 4 : 2;     // of either ring
  static constexpr uint32_t kQ = 0;                   // [half][128][128 B]
  static constexpr uint32_t kK = kRows * D * 2;
  static constexpr uint32_t kV = kK + kStages * kMatrix;
  static constexpr uint32_t kEnd = kV + kStages * kMatrix;
};

struct Bars {
  uint64_t q_full, k_full[4], k_empty[4], v_full[4], v_empty[4];
  uint64_t s_full[2], p_full[2][2], pv_done, o_full, drain;
};

struct TcParams {
  PagedAttnArgs a;
  float scale_log2;
  int64_t tiles, heads, splits, chunk;
  int* counters;
  float* partial;  // [tiles * heads][splits][128 rows x D, 128 maxima, 128 sums]
};

// column pairs of every 8 whose exponentials take the polynomial
constexpr unsigned kPolyPairs = 0x11u;

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 2)
    paged_tc05_kernel(const __grid_constant__ CUtensorMap tm_k,
                      const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ TcParams p) {
  using L = Smem<D>;
  constexpr int kStages = L::kStages, kHalves = L::kHalves;
  extern __shared__ unsigned char raw[];
  unsigned char* sbase = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
  const uint32_t base = smem_u32(sbase);
  __shared__ Bars bars;
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort, s_odd, s_last;
  __shared__ float s_m[kRows], s_l[kRows];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const PagedAttnArgs& a = p.a;

  // ---- rows and keys of this CTA; the tiles with most keys come first ----
  const int64_t split = blockIdx.x % p.splits;
  const int64_t w = blockIdx.x / p.splits;
  const int head = (int)(w / p.tiles);
  const int64_t tile = p.tiles - 1 - w % p.tiles;
  const int64_t item = head * p.tiles + tile;
  RowTile rt;
  if (!locate_tile(a.t, a.group, kRows, tile, rt)) return;
  const int64_t len = checked_length(a.t, a.pool, rt.seq);
  const int rows = rt.rows - rt.row0 < kRows ? rt.rows - rt.row0 : kRows;
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
  if (split >= runs) return;
  const int64_t tile0 = split * chunk;
  const int tiles = (int)(all_tiles - tile0 < chunk ? all_tiles - tile0 : chunk);

  volatile int* abort_flag = &s_abort;
  if (tid == 0) {
    tc::mbar_init(smem_u32(&bars.q_full), 128);
    for (int s = 0; s < kStages; ++s) {
      tc::mbar_init(smem_u32(&bars.k_full[s]), 1);
      tc::mbar_init(smem_u32(&bars.k_empty[s]), 1);
      tc::mbar_init(smem_u32(&bars.v_full[s]), 1);
      tc::mbar_init(smem_u32(&bars.v_empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      tc::mbar_init(smem_u32(&bars.s_full[b]), 1);
      tc::mbar_init(smem_u32(&bars.p_full[b][0]), 128);
      tc::mbar_init(smem_u32(&bars.p_full[b][1]), 128);
    }
    tc::mbar_init(smem_u32(&bars.pv_done), 1);
    tc::mbar_init(smem_u32(&bars.o_full), 1);
    tc::mbar_init(smem_u32(&bars.drain), 1);
    s_abort = 0;
    s_odd = 0;
    tc::mbar_fence_init();
  }
  if (warp == 1) {
    tc::tmem_alloc(smem_u32(&s_tmem), kTmemCols);
    tc::tmem_relinquish();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = s_tmem;
  const uint32_t t_o = tmem + 128u;

  if (warp == 0) {
    // ================= TMA producer =================
    const int box = a.pool.page < kTile ? a.pool.page : kTile;
    const int boxes = kTile / box, ahead = 32 / boxes;
    // a lane issues box `b` of half `half` of K (matrix 0) or V (matrix 1)
    const int b = lane & (boxes - 1), half = (lane / boxes) % kHalves;
    const int matrix = lane / (boxes * kHalves);
    int page = -1;
    int issued_k = 0, issued_v = 0;
    for (int t = 0; t < tiles; ++t) {
      const int64_t key0 = (tile0 + t) * kTile;
      if (t % ahead == 0) {
        const int64_t slot = key0 + (int64_t)lane * box;
        page = (int)a.pool.n_pages;  // past the pool: reads as zeros
        if (slot < most && slot < (tile0 + tiles) * kTile) {
          const int got = checked_page(a.t, a.pool, rt.seq, slot >> a.pool.page_shift);
          if (got >= 0) page = got;
        }
      }
      const int mine = __shfl_sync(0xffffffffu, page, (t % ahead) * boxes + b);
      const int need = (int)((most - key0 + box - 1) / box);
      const int live = need < boxes ? need : boxes;
      const int row = (int)((key0 + b * box) & (a.pool.page - 1));
      const int stage = t % kStages;
      const uint32_t phase = (uint32_t)((t / kStages - 1) & 1);
      const uint32_t off = stage * L::kMatrix + half * (kTile * 128) + b * box * 128;
      bool ok = t < kStages || tc::mbar_wait(smem_u32(&bars.k_empty[stage]), phase, abort_flag,
                                             a.wait_ns);
      if (!__all_sync(0xffffffffu, ok)) break;
      if (lane == 0)
        tc::mbar_expect_tx(smem_u32(&bars.k_full[stage]), (uint32_t)(live * box) * D * 2u);
      __syncwarp();
      if (matrix == 0 && b < live)
        tc::tma_load_4d(base + L::kK + off, &tm_k, smem_u32(&bars.k_full[stage]), half * 64, row,
                        head, mine);
      ++issued_k;
      ok = t < kStages || tc::mbar_wait(smem_u32(&bars.v_empty[stage]), phase, abort_flag,
                                        a.wait_ns);
      if (!__all_sync(0xffffffffu, ok)) break;
      if (lane == 0)
        tc::mbar_expect_tx(smem_u32(&bars.v_full[stage]), (uint32_t)(live * box) * D * 2u);
      __syncwarp();
      if (matrix == 1 && b < live)
        tc::tma_load_4d(base + L::kV + off, &tm_v, smem_u32(&bars.v_full[stage]), half * 64, row,
                        head, mine);
      ++issued_v;
    }
    // no copy may be in flight when the CTA leaves
    for (int t = issued_k > kStages ? issued_k - kStages : 0; t < issued_k; ++t)
      tc::mbar_wait_drain(smem_u32(&bars.k_full[t % kStages]), (uint32_t)((t / kStages) & 1),
                          kDrainNs);
    for (int t = issued_v > kStages ? issued_v - kStages : 0; t < issued_v; ++t)
      tc::mbar_wait_drain(smem_u32(&bars.v_full[t % kStages]), (uint32_t)((t / kStages) & 1),
                          kDrainNs);
  } else if (warp == 1) {
    // ================= MMA issuer =================
    if (lane == 0) {
      const uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
      const uint32_t id_qk = tc::idesc_f16(fmt, 0u, kRows, kTile);
      const uint32_t id_pv = tc::idesc_f16(fmt, 1u, kRows, D);
      bool ok = tc::mbar_wait(smem_u32(&bars.q_full), 0, abort_flag, a.wait_ns);
      const uint64_t qdesc = tc::sw128_desc(base + L::kQ, 16);
      auto issue_pv = [&](int u) -> bool {
        const int stage = u % kStages, buf = u & 1;
        if (!tc::mbar_wait(smem_u32(&bars.v_full[stage]), (uint32_t)((u / kStages) & 1),
                           abort_flag, a.wait_ns))
          return false;
        // 64-element groups of V's rows lie kTile * 128 bytes apart
        const uint64_t vdesc = tc::sw128_desc(base + L::kV + stage * L::kMatrix, kTile * 128);
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          if (!tc::mbar_wait(smem_u32(&bars.p_full[buf][part]), (uint32_t)((u >> 1) & 1),
                             abort_flag, a.wait_ns))
            return false;
          tc::tc_fence_after();
#pragma unroll
          for (int kk = 2 * part; kk < 2 * part + 2; ++kk)
            tc::mma_ts(t_o, tmem + 64u * buf + 8u * kk, vdesc + (uint64_t)(kk * 128), id_pv,
                       (u > 0 || kk > 0) ? 1u : 0u);
        }
        tc::mma_commit(smem_u32(&bars.pv_done));
        tc::mma_commit(smem_u32(&bars.v_empty[stage]));
        return true;
      };
      for (int t = 0; ok && t < tiles; ++t) {
        const int stage = t % kStages, buf = t & 1;
        ok = tc::mbar_wait(smem_u32(&bars.k_full[stage]), (uint32_t)((t / kStages) & 1),
                           abort_flag, a.wait_ns);
        if (!ok) break;
        tc::tc_fence_after();
        const uint64_t kdesc = tc::sw128_desc(base + L::kK + stage * L::kMatrix, 16);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          tc::mma_ss(tmem + 64u * buf,
                     qdesc + (uint64_t)((kk >> 2) * (kRows * 128 / 16) + (kk & 3) * 2),
                     kdesc + (uint64_t)((kk >> 2) * (kTile * 128 / 16) + (kk & 3) * 2), id_qk,
                     kk > 0 ? 1u : 0u);
        tc::mma_commit(smem_u32(&bars.s_full[buf]));
        tc::mma_commit(smem_u32(&bars.k_empty[stage]));
        if (t >= 1) ok = issue_pv(t - 1);
      }
      if (ok && tiles > 0 && issue_pv(tiles - 1)) tc::mma_commit(smem_u32(&bars.o_full));
      // every issued MMA must finish before the TMEM columns are released
      tc::mma_commit(smem_u32(&bars.drain));
      tc::mbar_wait_drain(smem_u32(&bars.drain), 0, kDrainNs);
    }
  } else {
    // ================= softmax: one query row per thread =================
    const int sub = warp & 3;  // TMEM lane quarter of this warp
    const int row = sub * 32 + lane;
    const uint32_t lane_off = (uint32_t)(sub * 32) << 16;
    const float c = p.scale_log2;
    const int64_t lim = limit_of(row < rows ? row : 0);  // a spare row masks nothing new
    {
      const int r = rt.row0 + (row < rows ? row : 0);
      const uint4* src = reinterpret_cast<const uint4*>(
          static_cast<const T*>(a.q) + (rt.first + r / a.group) * a.q_token +
          ((int64_t)head * a.group + r % a.group) * a.q_head);
#pragma unroll
      for (int k = 0; k < D / 8; ++k) {
        const uint4 v = __ldg(src + k);
        const uint32_t dst = base + L::kQ + (k >> 3) * (kRows * 128) + row * 128 +
                             (((k & 7) ^ (row & 7)) << 4);
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(v.x), "r"(v.y),
                     "r"(v.z), "r"(v.w)
                     : "memory");
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      tc::mbar_arrive(smem_u32(&bars.q_full));
    }
    float m_ref = -INFINITY, l0 = 0.f, l1 = 0.f;
    bool ok = true;
    for (int t = 0; t < tiles; ++t) {
      const int buf = t & 1;
      const int64_t key0 = (tile0 + t) * kTile;
      if (!__all_sync(0xffffffffu, tc::mbar_wait(smem_u32(&bars.s_full[buf]),
                                                 (uint32_t)((t >> 1) & 1), abort_flag,
                                                 a.wait_ns))) {
        ok = false;
        break;
      }
      tc::tc_fence_after();
      uint32_t s[64];
      tc::tmem_ld32(tmem + 64u * buf + lane_off, s);
      tc::tmem_ld32(tmem + 64u * buf + lane_off + 32u, s + 32);
      if (key0 + kTile > least) {  // the same for all four warps
        // V: clear the rows that nobody sees, look at those that only some see
        const int stage = t % kStages;
        if (!__all_sync(0xffffffffu, tc::mbar_wait(smem_u32(&bars.v_full[stage]),
                                                   (uint32_t)((t / kStages) & 1), abort_flag,
                                                   a.wait_ns))) {
          ok = false;
          break;
        }
        const int vrow = row & 63;
        unsigned char* v = sbase + L::kV + stage * L::kMatrix + vrow * 128;
        if (key0 + vrow >= most) {
#pragma unroll
          for (int h = row >> 6; h < 2 * kHalves; h += 2)  // 64 bytes at a time
#pragma unroll
            for (int i = 0; i < 4; ++i)
              *reinterpret_cast<uint4*>(v + (h >> 1) * (kTile * 128) + (h & 1) * 64 + i * 16) =
                  make_uint4(0u, 0u, 0u, 0u);
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        } else if (key0 + vrow >= least) {
          bool odd = false;
          for (int h = row >> 6; h < 2 * kHalves; h += 2)
            for (int i = 0; i < 4; ++i) {
              const uint4 x = *reinterpret_cast<const uint4*>(v + (h >> 1) * (kTile * 128) +
                                                              (h & 1) * 64 + i * 16);
              odd = odd || has_nonfinite<T>(x.x) || has_nonfinite<T>(x.y) ||
                    has_nonfinite<T>(x.z) || has_nonfinite<T>(x.w);
            }
          if (odd) s_odd = 1;
        }
        __syncwarp();
      }
      tc::tmem_wait_ld();
      const bool masked = __any_sync(0xffffffffu, key0 + kTile > lim);
      if (masked) {
        const int n = (int)(lim - key0 < 0 ? 0 : (lim - key0 < kTile ? lim - key0 : kTile));
#pragma unroll
        for (int i = 0; i < kTile; ++i)
          if (i >= n) s[i] = __float_as_uint(-INFINITY);
      }
      float mx[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float* f = reinterpret_cast<const float*>(s) + 8 * j;
        mx[j] = max3_nan(max3_nan(f[0], f[1], f[2]), max3_nan(f[3], f[4], f[5]),
                         max3_nan(f[6], f[7], f[7]));
      }
      const float mloc = max3_nan(max3_nan(mx[0], mx[1], mx[2]), max3_nan(mx[3], mx[4], mx[5]),
                                  max3_nan(mx[6], mx[7], mx[7]));
      // also true where either is NaN or both are -inf (nothing to rescale then)
      const bool grow = !((mloc - m_ref) * c <= 8.f);
      const bool rescale = grow && m_ref != -INFINITY;
      if (__any_sync(0xffffffffu, rescale)) {
        // O must hold the products of all tiles before this one
        if (!__all_sync(0xffffffffu, tc::mbar_wait(smem_u32(&bars.pv_done),
                                                   (uint32_t)((t - 1) & 1), abort_flag,
                                                   a.wait_ns))) {
          ok = false;
          break;
        }
        tc::tc_fence_after();
        const float f = rescale ? fast_exp2((m_ref - mloc) * c) : 1.f;
        l0 *= f;
        l1 *= f;
#pragma unroll
        for (int h = 0; h < D / 32; ++h) {
          uint32_t r[32];
          tc::tmem_ld32(t_o + lane_off + 32u * h, r);
          tc::tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * f);
          tc::tmem_st32(t_o + lane_off + 32u * h, r);
        }
      }
      if (grow) m_ref = mloc;
      // a row that has seen nothing keeps a finite base: its masked scores give 0
      const float mc = m_ref == -INFINITY ? 0.f : m_ref * c;
      uint32_t pk[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        float xa, xb, ea, eb;
        fma_pair(xa, xb, __uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1]), c, -mc);
        if (((kPolyPairs >> (i & 7)) & 1u) && !masked) {
          exp2_poly_pair(ea, eb, xa, xb);
        } else {
          ea = fast_exp2(xa);
          eb = fast_exp2(xb);
        }
        add_pair(l0, l1, ea, eb);
        pk[i] = ElemOps<T>::pack2(ea, eb);
        if (i == 15 || i == 31) {
          const int part = i >> 4;
          tc::tmem_st16(tmem + 64u * buf + lane_off + 16u * part, pk + 16 * part);
          tc::tmem_wait_st();
          tc::tc_fence_before();
          tc::mbar_arrive(smem_u32(&bars.p_full[buf][part]));
        }
      }
    }
    if (ok && tiles > 0)
      ok = __all_sync(0xffffffffu,
                      tc::mbar_wait(smem_u32(&bars.o_full), 0, abort_flag, a.wait_ns));
    tc::tc_fence_after();
    const bool have = ok && tiles > 0;
    const float l = have ? l0 + l1 : 0.f;
    s_m[row] = m_ref * c;
    s_l[row] = l;
    const float inv = runs > 1 ? 1.f : (l == 0.f ? 0.f : 1.f / l);
    float* part = p.partial + (item * p.splits + split) * (int64_t)(kRows * (D + 2)) + row * D;
    T* dst = nullptr;
    if (row < rows) {
      const int r = rt.row0 + row;
      dst = static_cast<T*>(a.out) + (rt.first + r / a.group) * a.o_token +
            ((int64_t)head * a.group + r % a.group) * a.o_head;
    }
#pragma unroll
    for (int h = 0; h < D / 32; ++h) {
      uint32_t r[32];
      if (have) {
        tc::tmem_ld32(t_o + lane_off + 32u * h, r);
        tc::tmem_wait_ld();
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) r[i] = 0u;
      }
      if (row < rows) {
        if (runs > 1) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            reinterpret_cast<uint4*>(part + 32 * h)[i] =
                make_uint4(r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float* f = reinterpret_cast<const float*>(r) + 8 * i;
            reinterpret_cast<uint4*>(dst + 32 * h)[i] =
                make_uint4(ElemOps<T>::pack2(f[0] * inv, f[1] * inv),
                           ElemOps<T>::pack2(f[2] * inv, f[3] * inv),
                           ElemOps<T>::pack2(f[4] * inv, f[5] * inv),
                           ElemOps<T>::pack2(f[6] * inv, f[7] * inv));
          }
        }
      }
    }
  }

  tc::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, kTmemCols);
  }
  if (tid == 0 && s_abort) raise_status(a.t.status, VGGT_STATUS_TIMEOUT);
  float* mine = p.partial + (item * p.splits + split) * (int64_t)(kRows * (D + 2));
  if (s_odd) {
    // a value that only some rows see is not finite: zero times it is not zero
    float* rowbuf = reinterpret_cast<float*>(sbase) + warp * D;  // the rings are free
    for (int r = warp; r < rows; r += kThreads / 32) {
      slow_row<T, D>(a, rt, r, head, p.scale_log2, tile0 * kTile, (tile0 + tiles) * kTile,
                     limit_of(r), rowbuf, &s_m[r], &s_l[r]);
      __syncwarp();
      const float l = s_l[r], inv = l == 0.f ? 0.f : 1.f / l;
      const int q = rt.row0 + r;
      T* dst = static_cast<T*>(a.out) + (rt.first + q / a.group) * a.o_token +
               ((int64_t)head * a.group + q % a.group) * a.o_head;
      for (int d = lane; d < D; d += 32) {
        if (runs > 1)
          mine[r * D + d] = rowbuf[d];
        else
          dst[d] = ElemOps<T>::from_float(rowbuf[d] * inv);
      }
      __syncwarp();
    }
    __syncthreads();
  }
  if (runs > 1) {
    if (tid < rows) {
      mine[kRows * D + tid] = s_m[tid];
      mine[kRows * (D + 1) + tid] = s_l[tid];
    }
    __threadfence();
    __syncthreads();
    if (tid == 0) {
      s_last = atomicAdd(p.counters + item, 1) == (int)runs - 1;
      if (s_last) p.counters[item] = 0;
    }
    __syncthreads();
    if (!s_last) return;
    __threadfence();
    // the CTA that finishes last joins the runs, in their order
    const float* from = p.partial + item * p.splits * (int64_t)(kRows * (D + 2));
    float* wgt = reinterpret_cast<float*>(sbase);  // [runs][128], at most 64 runs
    if (tid < rows) {
      float mx = -INFINITY, l = 0.f;
      for (int64_t s = 0; s < runs; ++s)
        mx = fmaxf(mx, __ldcg(from + s * kRows * (D + 2) + kRows * D + tid));
      const float b = mx == -INFINITY ? 0.f : mx;
      for (int64_t s = 0; s < runs; ++s) {
        const float* ml = from + s * kRows * (D + 2) + kRows * D + tid;
        const float f = fast_exp2(__ldcg(ml) - b);
        wgt[s * kRows + tid] = f;
        l += __ldcg(ml + kRows) * f;
      }
      s_m[tid] = mx;
      s_l[tid] = l;
    }
    __syncthreads();
    for (int i = tid; i < rows * (D / 4); i += kThreads) {
      const int r = i / (D / 4), d = (i % (D / 4)) * 4;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int s = 0; s < (int)runs; ++s) {
        const float f = wgt[s * kRows + r];
        const float4 v = __ldcg(reinterpret_cast<const float4*>(from + (int64_t)s * kRows * (D + 2)) + i);
        acc.x = fmaf(f, v.x, acc.x);
        acc.y = fmaf(f, v.y, acc.y);
        acc.z = fmaf(f, v.z, acc.z);
        acc.w = fmaf(f, v.w, acc.w);
      }
      const float l = s_l[r], inv = l == 0.f ? 0.f : 1.f / l;
      const int q = rt.row0 + r;
      T* dst = static_cast<T*>(a.out) + (rt.first + q / a.group) * a.o_token +
               ((int64_t)head * a.group + q % a.group) * a.o_head + d;
      *reinterpret_cast<uint2*>(dst) = make_uint2(ElemOps<T>::pack2(acc.x * inv, acc.y * inv),
                                                  ElemOps<T>::pack2(acc.z * inv, acc.w * inv));
    }
  }
  if (a.lse != nullptr && tid < rows) {
    const int q = rt.row0 + tid;
    a.lse[(rt.first + q / a.group) * (p.heads * a.group) + (int64_t)head * a.group + q % a.group] =
        s_l[tid] == 0.f ? -INFINITY : (s_m[tid] + log2f(s_l[tid])) * 0.6931471805599453f;
  }
}

template <typename T, int D>
cudaError_t launch_tc05(const TcParams& p, const CUtensorMap& mk, const CUtensorMap& mv,
                        cudaStream_t st) {
  auto kernel = paged_tc05_kernel<T, D>;
  const size_t smem = Smem<D>::kEnd + 1024;
  const cudaError_t e =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  kernel<<<(unsigned)(p.tiles * p.heads * p.splits), kThreads, smem, st>>>(mk, mv, p);
  return cudaGetLastError();
}

}  // namespace

PagedPlan paged_tc05_plan(int64_t total, int64_t seqs, int kv_heads, int group, int dim,
                          int64_t max_len) {
  PagedPlan plan{};
  plan.rows = kRows;
  plan.tiles = most_tiles(total, seqs, group, kRows);
  const int64_t items = plan.tiles * kv_heads, key_tiles = (max_len + kTile - 1) / kTile;
  // Runs per row tile: the number that ends the last wave of 2 CTAs per SM
  // soonest, a CTA's start and end counted as six key tiles.
  plan.splits = 1;
  int64_t best = -1;
  const int64_t slots = 2 * 148;
  for (int64_t s = 1; s <= 64 && (s == 1 || items <= kMaxCounters) && s * 4 <= key_tiles + 4; ++s) {
    const int64_t waves = (items * s + slots - 1) / slots;
    const int64_t cost = waves * ((key_tiles + s - 1) / s + 6);
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

cudaError_t launch_paged_tc05(const PagedAttnArgs& a, const PagedPlan& plan, cudaStream_t st) {
  TcParams p;
  p.a = a;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.tiles = plan.tiles;
  p.heads = a.pool.kv_heads;
  p.splits = plan.splits;
  p.chunk = plan.chunk;
  p.counters = static_cast<int*>(a.workspace);
  p.partial = reinterpret_cast<float*>(static_cast<char*>(a.workspace) + kMaxCounters * 4);
  if (plan.tiles == 0) return cudaSuccess;
  CUtensorMap mk, mv;
  const uint32_t box = (uint32_t)(a.pool.page < kTile ? a.pool.page : kTile);
  if (!encode_pool_tmap(&mk, a.k_pages, a.dtype, a.pool, box) ||
      !encode_pool_tmap(&mv, a.v_pages, a.dtype, a.pool, box))
    return cudaErrorInvalidValue;
  if (a.dtype == VGGT_DTYPE_BF16)
    return a.pool.dim == 64 ? launch_tc05<__nv_bfloat16, 64>(p, mk, mv, st)
                            : launch_tc05<__nv_bfloat16, 128>(p, mk, mv, st);
  return a.pool.dim == 64 ? launch_tc05<__half, 64>(p, mk, mv, st)
                          : launch_tc05<__half, 128>(p, mk, mv, st);
}

}  // namespace vggt
