// Attention of a chunk of new tokens over the paged cache on the
// 5th-generation tensor cores.
//
// A CTA takes 128 query rows of a sequence and key head (tokens x the head's
// group, so grouped heads fill the tile) and one run of 64-key tiles:
//   warp 0     streams K and V tiles by TMA, a box per page (or per 64 slots
//              of a larger page), into two rings; page numbers are read 32
//              boxes ahead
//   warp 1     issues S_t = Q K_t^T (Q, K in shared memory, S double-buffered
//              in TMEM)
//   warp 2     issues O += P_t V_t (P read from TMEM, where it overwrote S_t;
//              O stays in TMEM for the whole run)
//   warps 4-7  softmax, one query row per thread
// Two CTAs share an SM.  The issue is split over two warps, whole warps that
// wait and elect a lane to issue: on this chip a wait on a barrier costs a
// warp some 150 clocks even where it is satisfied, and the issue of four MMAs
// 200 to 300, so that one warp's four steps per tile took longer than the
// tile's softmax (510 us for a frame over 31 cached ones against 375, both
// before the steps below; 335 now).  These and the figures below are of launches
// replayed from a graph; an ordinary call of the frame takes 374 us.
//
// The row's reference maximum moves only when a tile's maximum exceeds it by
// more than 2^8 in the exp2 domain; O is rescaled then.  Sums are fp32, of the
// exponentials before P is rounded: the log-sum-exp is good to fp32 and only
// the product with V sees the rounding.  In fp16 the exponents are shifted up
// by 7 (PRange): P reaches 2^15 at most, and what lies 2^21 under the
// reference still has all of the type's bits.
//
// What bounds it: the multi-function unit gives 16 exponentials per clock and
// SM, so a 128 x 64 tile costs 512 clocks there, against 320 (dim 64) or 640
// (dim 128) of MMA (A from shared memory takes 48 clocks per MMA at N = 64, 32
// from TMEM).  One column pair of eight therefore takes a polynomial on the
// FMA pipe (at two of eight dim 64 gains nothing and dim 128 loses: 462 us for
// its frame against 451).  A tile takes 650 clocks: the softmax warps' own chain
// (wait, load, maximum, exponentials, store) is not fully covered by the other
// CTA's.  A CTA's start and end are 12,000 clocks of latency (sequence look-up,
// set-up, Q, the first product, the last one, the output), which short caches
// feel most: Q is loaded and the output stored with a row's pieces in
// neighbouring lanes, the row arithmetic is in 32 bits, and the output's loop
// is not unrolled, since instructions that run once come from afar (729 tokens
// of 3 sequences, 64 heads of 128: 82 us before, 73 after).
// Tried and slower: 32 keys per thread and 8 softmax warps (404 us),
// 128-key tiles with one S buffer (449 us), the next tile's maximum between
// the exponentials (634 us: its small TMEM loads wait for the stores), no
// maximum but a check of the tile's sum (388 us).
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

constexpr int kRows = 128, kTile = 64;
// Warps 0-3: TMA producer, S issuer, O issuer, and one that only fills rows of no
// sequence; warps 4-7: softmax.
constexpr int kThreads = 256;
// setmaxnreg: the launch gives every thread kLaunchRegs (two CTAs fill the
// register file); warps 0-3 give back down to kControlRegs, the softmax takes
// what that frees.
constexpr int kLaunchRegs = 128, kControlRegs = 64, kSoftRegs = 192;
static_assert(kControlRegs + kSoftRegs == 2 * kLaunchRegs, "register split");
constexpr uint32_t kTmemCols = 256;  // S0 | S1 | O
constexpr uint64_t kDrainNs = 1000000000ull;
constexpr int kMaxRuns = 64;  // per row tile

// How far a row's scores may pass its reference before that moves, and what
// exponents are shifted by, in units of log2.  With P <= 1 at the reference,
// fp16 would drop probabilities of 2^-25 and less from the product with V,
// which their sum still counts: 65,000 keys under one strong one lost 0.2 % of
// the output.  Lag and shift share the 15 steps up to 2^15.  A smaller lag moves
// the reference more often (4 prompts of dim 128 in two runs: 1,430 to 1,480 us;
// 1,560 at 4 and 11, 1,640 at 2 and 13).  bf16 has the exponents of fp32.
template <typename T>
struct PRange {
  static constexpr bool kHalf = std::is_same<T, __half>::value;
  static constexpr float kLag = 8.f, kShift = kHalf ? 7.f : 0.f;
};

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
  uint64_t q_full, full[2][4], empty[2][4];  // of K, of V
  uint64_t s_full[2], s_free[2], p_full[2], o_full, drain[2];
  uint64_t never;  // nothing arrives (wait self-test)
};

struct TcParams {
  PagedAttnArgs a;
  float scale_log2;
  int tiles, heads, splits, chunk;
  float* partial;  // [tiles * heads][splits] of [D / 4][128 rows][4], 128 maxima, 128 sums
};

// The keys that the last of a tile's `rows` rows sees, cut into runs.
struct Runs {
  int tiles, chunk, count;  // key tiles, and those of a run
};
// Keys that row `r` of the tile sees.
__device__ __forceinline__ int keys_of(const PagedAttnArgs& a, const RowTile& rt, int r) {
  const int len = (int)rt.len;
  if (!a.causal) return len;
  const int n = len - rt.n_new + (rt.row0 + r) / a.group + 1;
  return n < 0 ? 0 : (n < len ? n : len);
}
__device__ __forceinline__ Runs runs_of(const TcParams& p, const RowTile& rt, int rows) {
  Runs r;
  r.tiles = (int)(((unsigned)keys_of(p.a, rt, rows - 1) + kTile - 1) / kTile);
  r.chunk = (r.tiles + p.splits - 1) / p.splits;
  if (r.chunk < p.chunk) r.chunk = p.chunk;
  r.count = r.tiles > 0 ? (r.tiles + r.chunk - 1) / r.chunk : 1;
  return r;
}

// column pairs of every 8 whose exponentials take the polynomial
constexpr unsigned kPolyPairs = 0x80u;

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
  __shared__ int s_abort, s_odd;
  __shared__ float s_m[kRows], s_l[kRows];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const PagedAttnArgs& a = p.a;

  // once every CTA is here, the join's may take the places that become free
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // ---- rows and keys of this CTA; the tiles with most keys come first ----
  const int split = (int)(blockIdx.x % (unsigned)p.splits);
  const unsigned w = blockIdx.x / (unsigned)p.splits;
  const int head = (int)(w / (unsigned)p.tiles);
  const int tile = p.tiles - 1 - (int)(w % (unsigned)p.tiles);
  const int64_t item = (int64_t)head * p.tiles + tile;
  RowTile rt;
  if (!locate_tile(a.t, a.pool, a.group, kRows, tile, rt)) {
    if (warp == 0) fill_rows_of_no_sequence<T, D>(a);
    return;
  }
  const int rows = rt.rows - rt.row0 < kRows ? rt.rows - rt.row0 : kRows;
  const Runs cut = runs_of(p, rt, rows);
  const int runs = cut.count;
  if (split >= runs) {
    if (warp == 0) fill_rows_of_no_sequence<T, D>(a);
    return;
  }
  const int first_key = split * cut.chunk * kTile;
  const int tiles = min(cut.tiles - split * cut.chunk, cut.chunk);

  // The softmax warps' rows of Q, a row's 16-byte pieces in neighbouring lanes:
  // on their way while the CTA sets up
  constexpr int kPieces = D / 8, kAtOnce = 32 / kPieces;  // of a row; rows per instruction
  const int row = (warp & 3) * 32 + lane, piece = lane % kPieces;
  uint4 q_in[kPieces];
  if (warp >= 4) {
    const int r = rt.row0 + (row < rows ? row : 0);
    const int64_t mine = (rt.first + r / a.group) * a.q_token +
                         ((int64_t)head * a.group + r % a.group) * a.q_head;
#pragma unroll
    for (int k = 0; k < kPieces; ++k) {
      const int64_t at = __shfl_sync(0xffffffffu, mine, k * kAtOnce + lane / kPieces);
      q_in[k] = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + at) + piece);
    }
  }
  // Where piece c of row r lies: halves of 64 elements, 128-byte swizzle, as
  // the MMA reads Q
  auto piece_at = [&](int r, int c) -> uint32_t {
    return base + L::kQ + (c >> 3) * (kRows * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4);
  };

  volatile int* abort_flag = &s_abort;
  if (tid == 0) {
    tc::mbar_init(smem_u32(&bars.q_full), kRows);
    for (int s = 0; s < kStages; ++s) {
      for (int kv = 0; kv < 2; ++kv) {
        tc::mbar_init(smem_u32(&bars.full[kv][s]), 1);
        tc::mbar_init(smem_u32(&bars.empty[kv][s]), 1);
      }
    }
    for (int b = 0; b < 2; ++b) {
      tc::mbar_init(smem_u32(&bars.s_full[b]), 1);
      tc::mbar_init(smem_u32(&bars.s_free[b]), 1);
      tc::mbar_init(smem_u32(&bars.p_full[b]), kRows);
    }
    tc::mbar_init(smem_u32(&bars.o_full), 1);
    for (int i = 0; i < 2; ++i) tc::mbar_init(smem_u32(&bars.drain[i]), 1);
    tc::mbar_init(smem_u32(&bars.never), 1);
    s_abort = 0;
    s_odd = 0;
    tc::mbar_fence_init();
  }
  if (warp == 4) {
    tc::tmem_alloc(smem_u32(&s_tmem), kTmemCols);
    tc::tmem_relinquish();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = s_tmem;
  const uint32_t t_o = tmem + 128u;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kControlRegs));
    if (warp == 0) {
      // ================= TMA producer =================
      const int keys = keys_of(a, rt, rows - 1) - first_key;  // to the end of the last row's keys
      auto produce = [&](auto boxes_) {
        constexpr int kBoxes = decltype(boxes_)::value;  // boxes per tile
        constexpr int kBox = kTile / kBoxes;             // slots per box
        constexpr int kAhead = 32 / kBoxes;              // tiles per read of the table
        const uint32_t full0 = smem_u32(&bars.full[0][0]), empty0 = smem_u32(&bars.empty[0][0]);
        constexpr uint32_t kToV = sizeof(bars.full[0]);  // from K's barriers to V's
        const int32_t* table = a.t.table + rt.seq * a.t.width;
        const int in_page = first_key & (a.pool.page - 1), page_mask = a.pool.page - 1;
        int page = 0, stage = 0;
        int issued_at[2] = {0, 0};  // of the elected lane
        uint32_t phase = 1;
        for (int t = 0; t < tiles; ++t) {
          const int key0 = t * kTile;
          const int turn = t & (kAhead - 1);
          if (turn == 0) {
            const int key = key0 + lane * kBox;
            page = (int)a.pool.n_pages;  // past the pool: reads as zeros
            if (key < keys && key < tiles * kTile) {
              const int got = __ldg(table + ((first_key + key) >> a.pool.page_shift));
              if (got >= 0 && got < a.pool.n_pages)
                page = got;
              else
                raise_status(a.t.status, VGGT_STATUS_BAD_PAGE);
            }
          }
          int pages[kBoxes];
#pragma unroll
          for (int b = 0; b < kBoxes; ++b)
            pages[b] = __shfl_sync(0xffffffffu, page, turn * kBoxes + b);
          int live = (keys - key0 + kBox - 1) / kBox;
          live = live < kBoxes ? live : kBoxes;
          const int row = (in_page + key0) & page_mask;
          bool ok = true;
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            if (t >= kStages)
              ok = ok &&
                   tc::warp_wait(empty0 + kv * kToV + 8u * stage, phase, abort_flag, a.wait_ns);
            if (ok && tc::elect_one()) {
              const uint32_t bar = full0 + kv * kToV + 8u * stage;
              tc::mbar_expect_tx(bar, (uint32_t)(live * kBox) * D * 2u);
              const uint32_t dst = base + (kv ? L::kV : L::kK) + stage * L::kMatrix;
#pragma unroll
              for (int b = 0; b < kBoxes; ++b)
                if (b < live)
#pragma unroll
                  for (int h = 0; h < kHalves; ++h)
                    tc::tma_load_4d(dst + h * (kTile * 128) + b * kBox * 128, kv ? &tm_v : &tm_k,
                                    bar, h * 64, (row + b * kBox) & page_mask, head, pages[b]);
              issued_at[kv] = t + 1;
            }
            __syncwarp();
          }
          if (!ok) break;
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        // no copy may be in flight when the CTA leaves
        for (int kv = 0; kv < 2; ++kv)
          for (int t = max(issued_at[kv] - kStages, 0); t < issued_at[kv]; ++t)
            tc::mbar_wait_drain(full0 + kv * kToV + 8u * (t % kStages),
                                (uint32_t)((t / kStages) & 1), kDrainNs);
      };
      if (a.pool.page >= 64)
        produce(std::integral_constant<int, 1>{});
      else if (a.pool.page == 32)
        produce(std::integral_constant<int, 2>{});
      else
        produce(std::integral_constant<int, 4>{});
    } else if (warp < 3) {
      // ================= MMA issuers: warp 1 S = Q K^T, warp 2 O += P V ========
      // The whole warp walks through the tiles and waits; one elected lane
      // issues, which keeps the MMA operands in uniform registers.
      const uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
      auto wait = [&](uint32_t bar, uint32_t parity) {
        return tc::warp_wait(bar, parity, abort_flag, a.wait_ns);
      };
      const uint32_t kfull0 = smem_u32(&bars.full[0][0]), kempty0 = smem_u32(&bars.empty[0][0]);
      const uint32_t vfull0 = smem_u32(&bars.full[1][0]), vempty0 = smem_u32(&bars.empty[1][0]);
      const uint32_t sfull0 = smem_u32(&bars.s_full[0]), pfull0 = smem_u32(&bars.p_full[0]);
      const uint32_t sfree0 = smem_u32(&bars.s_free[0]);
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      if (warp == 1) {
        const uint32_t id_qk = tc::idesc_f16(fmt, 0u, kRows, kTile);
        const uint64_t qdesc = tc::sw128_desc(base + L::kQ, 16);
        const uint64_t kdesc0 = tc::sw128_desc(base + L::kK, 16);
        ok = wait(smem_u32(&bars.q_full), 0);
        if (a.wait_selftest) ok = ok && wait(smem_u32(&bars.never), 0);
        for (int t = 0; ok && t < tiles; ++t) {
          const uint32_t buf = t & 1;
          // P of tile t - 2 lay where S_t goes: its product must be done
          ok = (t < 2 || wait(sfree0 + 8u * buf, (uint32_t)((t >> 1) + 1) & 1u)) &&
               wait(kfull0 + 8u * stage, phase);
          if (!ok) break;
          tc::tc_fence_after();
          if (tc::elect_one()) {
            const uint64_t kdesc = kdesc0 + (uint64_t)(stage * (L::kMatrix / 16));
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
              tc::mma_ss(tmem + 64u * buf,
                         qdesc + (uint64_t)((kk >> 2) * (kRows * 128 / 16) + (kk & 3) * 2),
                         kdesc + (uint64_t)((kk >> 2) * (kTile * 128 / 16) + (kk & 3) * 2), id_qk,
                         kk > 0 ? 1u : 0u);
            tc::mma_commit(sfull0 + 8u * buf);
            tc::mma_commit(kempty0 + 8u * stage);
          }
          __syncwarp();
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      } else {
        const uint32_t id_pv = tc::idesc_f16(fmt, 1u, kRows, D);
        // 64-element groups of V's rows lie kTile * 128 bytes apart
        const uint64_t vdesc0 = tc::sw128_desc(base + L::kV, kTile * 128);
        for (int t = 0; ok && t < tiles; ++t) {
          const uint32_t buf = t & 1;
          ok = wait(vfull0 + 8u * stage, phase) && wait(pfull0 + 8u * buf, (uint32_t)(t >> 1) & 1u);
          if (!ok) break;
          tc::tc_fence_after();
          if (tc::elect_one()) {
            const uint64_t vdesc = vdesc0 + (uint64_t)(stage * (L::kMatrix / 16));
#pragma unroll
            for (int kk = 0; kk < kTile / 16; ++kk)
              tc::mma_ts(t_o, tmem + 64u * buf + 8u * kk, vdesc + (uint64_t)(kk * 128), id_pv,
                         (t > 0 || kk > 0) ? 1u : 0u);
            tc::mma_commit(sfree0 + 8u * buf);
            tc::mma_commit(vempty0 + 8u * stage);
          }
          __syncwarp();
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (tc::elect_one()) {
        if (warp == 2 && ok && tiles > 0) tc::mma_commit(smem_u32(&bars.o_full));
        // every issued MMA must finish before the TMEM columns are released
        tc::mma_commit(smem_u32(&bars.drain[warp - 1]));
      }
      __syncwarp();
      tc::mbar_wait_drain(smem_u32(&bars.drain[warp - 1]), 0, kDrainNs);
    } else {
      fill_rows_of_no_sequence<T, D>(a);
    }
    return;  // what follows runs on the softmax warps alone
  }
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftRegs));
  const int stid = tid - 128;
  auto sync_softmax = [] { asm volatile("bar.sync 1, 128;" ::: "memory"); };
  {
    // ================= softmax: one query row per thread =================
    const int sub = warp & 3;  // TMEM lane quarter of this warp
    const uint32_t lane_off = (uint32_t)(sub * 32) << 16;
    const float c = p.scale_log2;
#pragma unroll
    for (int k = 0; k < kPieces; ++k) {
      const uint4 v = q_in[k];
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(
                       piece_at(sub * 32 + k * kAtOnce + lane / kPieces, piece)),
                   "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
                   : "memory");
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    tc::mbar_arrive(smem_u32(&bars.q_full));
    // counted from the run's first key, within one tile of its ends
    const int span = tiles * kTile;
    auto within = [&](int key) {
      const int n = key - first_key;
      return n < 0 ? 0 : (n < span ? n : span);
    };
    // a spare row masks nothing new
    const int lim_at = within(keys_of(a, rt, row < rows ? row : 0));
    const int least_at = within(keys_of(a, rt, 0)), most_at = within(keys_of(a, rt, rows - 1));
    const uint32_t sfull0 = smem_u32(&bars.s_full[0]), pfull0 = smem_u32(&bars.p_full[0]);
    auto wait = [&](uint32_t bar, uint32_t parity) {
      return tc::warp_wait(bar, parity, abort_flag, a.wait_ns);
    };
    // whether some row of the CTA does not see all of tile t (for all warps alike)
    auto is_edge = [&](int t) { return (t + 1) * kTile > least_at; };
    // The reference in score units, and what is added to a score's exponent:
    // PRange's shift less the reference, rounded down, so that the largest P is
    // known however large the scores are.  A row that has seen nothing keeps 0:
    // its masked scores give 0.
    float m_ref = -INFINITY, minus = 0.f;
    float_pair sum = pack_pair(0.f, 0.f);
    const float_pair c2 = pack_pair(c, c);
    const Exp2Poly poly;
    bool ok = true;
    for (int t = 0; t < tiles; ++t) {
      const uint32_t buf = t & 1;
      const uint32_t t_s = tmem + lane_off + 64u * buf;
      if (!wait(sfull0 + 8u * buf, (uint32_t)(t >> 1) & 1u)) {
        ok = false;
        break;
      }
      tc::tc_fence_after();
      uint32_t s[64];
      tc::tmem_ld32(t_s, s);
      tc::tmem_ld32(t_s + 32u, s + 32);
      tc::tmem_wait_ld();
      if (is_edge(t)) {
        // V: clear the rows that nobody sees, look at those that only some see
        const int stage = t % kStages;
        if (!wait(smem_u32(&bars.full[1][stage]), (uint32_t)((t / kStages) & 1))) {
          ok = false;
          break;
        }
        const int vkey = t * kTile + (row & 63);
        if (vkey >= least_at) {
          unsigned char* v = sbase + L::kV + stage * L::kMatrix + (row & 63) * 128;
          bool odd = false;
          for (int h = row >> 6; h < 2 * kHalves; h += 2) {  // 64 bytes each
            uint4* at = reinterpret_cast<uint4*>(v + (h >> 1) * (kTile * 128) + (h & 1) * 64);
            for (int i = 0; i < 4; ++i) {
              if (vkey >= most_at) {
                at[i] = make_uint4(0u, 0u, 0u, 0u);
              } else {
                const uint4 x = at[i];
                odd = odd || has_nonfinite<T>(x.x) || has_nonfinite<T>(x.y) ||
                      has_nonfinite<T>(x.z) || has_nonfinite<T>(x.w);
              }
            }
          }
          if (odd) s_odd = 1;
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        __syncwarp();
        const int seen = lim_at - t * kTile;
#pragma unroll
        for (int i = 0; i < kTile; ++i)
          if (i >= seen) s[i] = __float_as_uint(-INFINITY);
      }
      float mx[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float* f = reinterpret_cast<const float*>(s) + 8 * j;
        mx[j] = max3_nan(max3_nan(f[0], f[1], f[2]), max3_nan(f[3], f[4], f[5]),
                         max_nan(f[6], f[7]));
      }
      const float m = max3_nan(max3_nan(mx[0], mx[1], mx[2]), max3_nan(mx[3], mx[4], mx[5]),
                               max_nan(mx[6], mx[7]));
      // also true where m or m_ref is NaN; a tile of which the row sees nothing
      // changes nothing (a NaN in the sum stays)
      const bool grow = !((m - m_ref) * c <= PRange<T>::kLag) && m != -INFINITY;
      if (__any_sync(0xffffffffu, grow)) {
        const bool rescale = grow && m_ref != -INFINITY;
        const float moved = __fmaf_rd(-m, c, PRange<T>::kShift);
        if (__any_sync(0xffffffffu, rescale)) {
          // O must hold the products of all tiles before this one
          if (!wait(smem_u32(&bars.s_free[(t - 1) & 1]), (uint32_t)(((t - 1) >> 1) & 1))) {
            ok = false;
            break;
          }
          tc::tc_fence_after();
          const float f = rescale ? fast_exp2(moved - minus) : 1.f;
          sum = fma_pair(sum, pack_pair(f, f), pack_pair(0.f, 0.f));
#pragma unroll 1
          for (int h = 0; h < D / 16; ++h) {
            uint32_t r[16];
            tc::tmem_ld16(t_o + lane_off + 16u * h, r);
            tc::tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * f);
            tc::tmem_st16(t_o + lane_off + 16u * h, r);
          }
        }
        if (grow) {
          m_ref = m;
          minus = moved;
        }
      }
      const float_pair minus2 = pack_pair(minus, minus);
      float_pair part[2] = {sum, pack_pair(0.f, 0.f)};
      uint32_t pk[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const float_pair x = fma_pair(
            pack_pair(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), c2, minus2);
        float ea, eb;
        if ((kPolyPairs >> (i & 7)) & 1u) {
          float_pair q, scale;
          poly(q, scale, x);
          unpack_pair(ea, eb, mul_pair(q, scale));
        } else {
          unpack_pair(ea, eb, x);
          ea = fast_exp2(ea);
          eb = fast_exp2(eb);
        }
        part[i & 1] = add_pair(part[i & 1], pack_pair(ea, eb));
        pk[i] = ElemOps<T>::pack2(ea, eb);
      }
      sum = add_pair(part[0], part[1]);
      tc::tmem_st32(t_s, pk);
      tc::tmem_wait_st();
      tc::tc_fence_before();
      tc::mbar_arrive(pfull0 + 8u * buf);
    }
    if (ok && tiles > 0)
      ok = tc::warp_wait(smem_u32(&bars.o_full), 0, abort_flag, a.wait_ns);
    tc::tc_fence_after();
    const bool have = ok && tiles > 0;
    float l0, l1;
    unpack_pair(l0, l1, sum);
    const float l = have && m_ref != -INFINITY ? l0 + l1 : 0.f;
    s_m[row] = m_ref == -INFINITY ? -INFINITY : -minus;
    s_l[row] = l;
    const float inv = runs > 1 ? 1.f : (l == 0.f ? 0.f : 1.f / l);
    float4* part = reinterpret_cast<float4*>(
                       p.partial + (item * p.splits + split) * (int64_t)(kRows * (D + 2))) +
                   row;
#pragma unroll 1  // run once: its instructions come from afar, few are faster
    for (int h = 0; h < D / 32; ++h) {
      uint32_t r[32];
      if (have) {
        tc::tmem_ld32(t_o + lane_off + 32u * h, r);
        tc::tmem_wait_ld();
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) r[i] = 0u;
      }
      const float* f = reinterpret_cast<const float*>(r);
      if (runs > 1) {
        if (row < rows) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            part[(8 * h + i) * kRows] =
                make_float4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i, f += 8)
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(piece_at(row, 4 * h + i)),
                       "r"(ElemOps<T>::pack2(f[0] * inv, f[1] * inv)),
                       "r"(ElemOps<T>::pack2(f[2] * inv, f[3] * inv)),
                       "r"(ElemOps<T>::pack2(f[4] * inv, f[5] * inv)),
                       "r"(ElemOps<T>::pack2(f[6] * inv, f[7] * inv))
                       : "memory");
      }
    }
    if (runs == 1) {
      // through Q's place, which no MMA reads any more, so that neighbouring
      // lanes store neighbouring pieces
      const int r = rt.row0 + (row < rows ? row : 0);
      const int64_t mine = (rt.first + r / a.group) * a.o_token +
                           ((int64_t)head * a.group + r % a.group) * a.o_head;
      __syncwarp();
#pragma unroll 4
      for (int k = 0; k < kPieces; ++k) {
        const int from = k * kAtOnce + lane / kPieces;
        const int64_t at = __shfl_sync(0xffffffffu, mine, from);
        uint4 v;
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                     : "r"(piece_at(sub * 32 + from, piece))
                     : "memory");
        if (sub * 32 + from < rows)
          reinterpret_cast<uint4*>(static_cast<T*>(a.out) + at)[piece] = v;
      }
    }
  }

  tc::tc_fence_before();
  sync_softmax();
  if (warp == 4) {
    // every MMA must have ended before the columns go back
    for (int i = 0; i < 2; ++i) tc::mbar_wait_drain(smem_u32(&bars.drain[i]), 0, kDrainNs);
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, kTmemCols);
  }
  if (stid == 0 && s_abort) raise_status(a.t.status, VGGT_STATUS_TIMEOUT);
  float* mine = p.partial + (item * p.splits + split) * (int64_t)(kRows * (D + 2));
  if (s_odd) {
    // a value that only some rows see is not finite: zero times it is not zero
    float* rowbuf = reinterpret_cast<float*>(sbase) + (warp - 4) * D;  // the rings are free
    const RowTile here = rt;  // of which the call takes the address: not of rt
    for (int r = warp - 4; r < rows; r += 4) {
      slow_row<T, D>(a, here, r, head, p.scale_log2, first_key, (int64_t)first_key + tiles * kTile,
                     keys_of(a, rt, r), rowbuf, &s_m[r], &s_l[r]);
      __syncwarp();
      const float l = s_l[r], inv = l == 0.f ? 0.f : 1.f / l;
      const int q = rt.row0 + r;
      T* dst = static_cast<T*>(a.out) + (rt.first + q / a.group) * a.o_token +
               ((int64_t)head * a.group + q % a.group) * a.o_head;
      for (int d = lane; d < D; d += 32) {
        if (runs > 1)
          mine[(d / 4 * kRows + r) * 4 + d % 4] = rowbuf[d];
        else
          dst[d] = ElemOps<T>::from_float(rowbuf[d] * inv);
      }
      __syncwarp();
    }
    sync_softmax();
  }
  if (runs > 1) {  // the join kernel makes the output of these
    if (stid < rows) {
      mine[kRows * D + stid] = s_m[stid];
      mine[kRows * (D + 1) + stid] = s_l[stid];
    }
    return;
  }
  if (a.lse != nullptr && stid < rows) {
    const int q = rt.row0 + stid;
    a.lse[((rt.first + q / a.group) * p.heads + head) * a.group + q % a.group] =
        s_l[stid] == 0.f ? -INFINITY : (s_m[stid] + log2f(s_l[stid])) * 0.6931471805599453f;
  }
}

// Joins the runs of a row tile, in their order: a CTA takes 512 / D rows of an
// item, a thread 4 of their elements, 8 runs' loads in flight.  A launch of its
// own, since it spreads over the card: the CTA that finished last took 10 us
// for 5 runs of dim 64 and 40 for 40 runs of dim 128.  It is launched while the
// runs' last wave is at work (a frame 338 -> 335 us, 88 rows over 5,010 keys
// 18.8 -> 18.2).
constexpr int kJoinThreads = 128;

template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads)
    join_runs_kernel(const __grid_constant__ TcParams p) {
  constexpr int kHere = 4 * kJoinThreads / D;  // rows
  constexpr int64_t kRun = kRows * (D + 2);
  __shared__ float wgt[kMaxRuns][kHere], sums[kMaxRuns][kHere], inv_l[kHere];
  const PagedAttnArgs& a = p.a;
  // The runs' kernel has ended and its writes are visible from here on.  Every
  // thread waits, those that leave early too: what comes after this kernel on
  // the stream relies on the runs' kernel as well.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const unsigned item = blockIdx.x / (kRows / kHere);
  const int r0 = (int)(blockIdx.x % (kRows / kHere)) * kHere, tid = threadIdx.x;
  const int head = (int)(item / (unsigned)p.tiles);
  RowTile rt;
  if (!locate_tile(a.t, a.pool, a.group, kRows, item % (unsigned)p.tiles, rt)) return;
  const int in_tile = rt.rows - rt.row0 < kRows ? rt.rows - rt.row0 : kRows;
  const int rows = in_tile - r0 < kHere ? in_tile - r0 : kHere;
  const int count = runs_of(p, rt, in_tile).count;
  if (rows <= 0 || count == 1) return;
  const float* from = p.partial + (int64_t)item * p.splits * kRun;
  for (int i = tid; i < count * kHere; i += kJoinThreads) {
    const int s = i / kHere, r = i % kHere;
    if (r < rows) {
      wgt[s][r] = from[s * kRun + kRows * D + r0 + r];
      sums[s][r] = from[s * kRun + kRows * (D + 1) + r0 + r];
    }
  }
  __syncthreads();
  if (tid < rows) {
    float mx = -INFINITY, l = 0.f;
    for (int s = 0; s < count; ++s) mx = fmaxf(mx, wgt[s][tid]);
    const float b = mx == -INFINITY ? 0.f : mx;
    for (int s = 0; s < count; ++s) {
      const float f = fast_exp2(wgt[s][tid] - b);
      wgt[s][tid] = f;
      l = fmaf(f, sums[s][tid], l);
    }
    inv_l[tid] = l == 0.f ? 0.f : 1.f / l;
    if (a.lse != nullptr) {
      const int q = rt.row0 + r0 + tid;
      a.lse[((rt.first + q / a.group) * p.heads + head) * a.group + q % a.group] =
          l == 0.f ? -INFINITY : (mx + log2f(l)) * 0.6931471805599453f;
    }
  }
  __syncthreads();
  const int r = tid % kHere, d = tid / kHere * 4;
  if (r >= rows) return;
  const float* mine = from + d * kRows + (r0 + r) * 4;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = 0; s0 < count; s0 += 8) {
    float4 v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (s0 + j < count) v[j] = *reinterpret_cast<const float4*>(mine + (s0 + j) * kRun);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (s0 + j < count) {
        const float f = wgt[s0 + j][r];
        acc.x = fmaf(f, v[j].x, acc.x);
        acc.y = fmaf(f, v[j].y, acc.y);
        acc.z = fmaf(f, v[j].z, acc.z);
        acc.w = fmaf(f, v[j].w, acc.w);
      }
  }
  const float inv = inv_l[r];
  const int q = rt.row0 + r0 + r;
  T* dst = static_cast<T*>(a.out) + (rt.first + q / a.group) * a.o_token +
           ((int64_t)head * a.group + q % a.group) * a.o_head + d;
  *reinterpret_cast<uint2*>(dst) = make_uint2(ElemOps<T>::pack2(acc.x * inv, acc.y * inv),
                                              ElemOps<T>::pack2(acc.z * inv, acc.w * inv));
}

template <typename T, int D>
cudaError_t launch_tc05(const TcParams& p, const CUtensorMap& mk, const CUtensorMap& mv,
                        cudaStream_t st) {
  auto kernel = paged_tc05_kernel<T, D>;
  const size_t smem = Smem<D>::kEnd + 1024;
  // with another register count at launch the softmax's setmaxnreg would wait for ever
  cudaFuncAttributes fa;
  if (const cudaError_t r = cudaFuncGetAttributes(&fa, kernel); r != cudaSuccess) return r;
  if (fa.numRegs != kLaunchRegs) return cudaErrorInvalidConfiguration;
  const cudaError_t e =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  kernel<<<(unsigned)p.tiles * p.heads * p.splits, kThreads, smem, st>>>(mk, mv, p);
  const cudaError_t launched = cudaGetLastError();
  if (launched != cudaSuccess || p.splits == 1) return launched;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)p.tiles * p.heads * (kRows * D / (4 * kJoinThreads)));
  cfg.blockDim = dim3(kJoinThreads);
  cfg.stream = st;
  cudaLaunchAttribute early{};  // its launch overlaps the runs' last wave
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, join_runs_kernel<T, D>, p);
}

}  // namespace

PagedPlan paged_tc05_plan(int64_t total, int64_t seqs, int kv_heads, int group, int dim,
                          int64_t max_len) {
  PagedPlan plan{};
  plan.rows = kRows;
  plan.tiles = most_tiles(total, seqs, group, kRows);
  const int64_t items = plan.tiles * kv_heads, key_tiles = (max_len + kTile - 1) / kTile;
  // Runs per row tile: the number that ends the last wave of 2 CTAs per SM
  // soonest.  In units of a key tile (0.7 us, 1.0 at dim 128): a CTA's start and
  // end cost ten, the join's launch two, and a run's partial result, written and
  // read at 4 TB/s, 1/40 (1/30).  Of 15 shapes the rule takes the fastest number
  // for 13 and loses 4 % at two.  In us, taken ones in brackets: a frame over 31
  // cached ones, 176 items, 1 run 535, 3 runs 377, 5 runs (343), 10 runs 351; the
  // same of dim 128, 88 items, 1 run 517, 3 runs (235), 10 runs 248; 100 tokens
  // over 43,000 keys, 16 items, 8 runs 61, 18 runs (49), 32 runs 57; 4 prompts,
  // 1,840 items, 1 run (1,273), 2 runs 1,482; 8 chunks of 500 tokens, 976 items,
  // 1 run (451), 2 runs 528.
  plan.splits = 1;
  double best = -1;
  const int64_t slots = 2 * 148;
  const double partial = dim == 64 ? 1.0 / 40 : 1.0 / 30;
  for (int64_t s = 1; s <= kMaxRuns && s <= (key_tiles > 0 ? key_tiles : 1); ++s) {
    const int64_t waves = (items * s + slots - 1) / slots;
    const double cost = (double)(waves * ((key_tiles + s - 1) / s + 10)) +
                        (s > 1 ? 2 + (double)(items * s) * partial : 0);
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
  p.tiles = (int)plan.tiles;  // the entry point holds tiles * heads * splits below 2^31
  p.heads = a.pool.kv_heads;
  p.splits = (int)plan.splits;
  p.chunk = (int)plan.chunk;
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

