// Matrix product on the tensor cores with bias, activation, gate and residual in its epilogue.
//
// A tile of C is 128 CTA x 128 CTA elements, CTA = 1 or 2 CTAs (a pair works on one tile: each
// holds half of A's rows and half of B's, the MMA of the pair reads both halves of B).  Warp 0
// streams the operands by TMA through a ring of 64-element reduction blocks, warp 1 issues the
// MMAs into one of two accumulators in TMEM, and warps 4-19, four warpgroups of which each takes 64
// columns, run the epilogue of the tile before: TMEM -> registers -> bias, activation, gate,
// residual -> the group's swizzled 16 KB buffer -> TMA store.  The residual comes by TMA into the
// same buffer before.  What TMA cannot address (odd widths, other strides) is copied between
// buffer and memory by the warps that own the rows.  (With two warpgroups an activation's latencies
// bounded the kernel.)
//
// Bound by the tensor cores and by the operands' way from L2 (a pair's 256 x 256 tile needs
// 64 B a cycle and SM at the full rate, a single CTA's 128 x 128 twice that).
//
// Every wait is bounded; on expiry the CTA raises its abort flag, VGGT_STATUS_TIMEOUT is set and
// all roles leave.
#include "linear.cuh"

#include <algorithm>
#include <climits>
#include <type_traits>

#include "activation.cuh"
#include "tc05.cuh"

namespace vggt {
namespace lin {

constexpr int BM = 128, BK = 64;
constexpr int STAGES = 5;
constexpr int GROUPS = 4;                     // warpgroups of the epilogue
constexpr int THREADS = 128 + GROUPS * 128;
constexpr uint32_t HALF_BYTES = BM * BK * 2;         // one operand's block: 16 KB
constexpr uint32_t STAGE_BYTES = 2 * HALF_BYTES;
constexpr uint32_t BUF_BYTES = BM * 128;             // epilogue buffer: 128 rows of 128 bytes
constexpr uint32_t OFF_BUF = STAGES * STAGE_BYTES;           // [GROUPS]
constexpr uint32_t OFF_VEC = OFF_BUF + GROUPS * BUF_BYTES;   // float[GROUPS][bias 64, gate 64]
constexpr uint32_t OFF_BAR = OFF_VEC + GROUPS * 128 * 4;
constexpr int B_FULL = 0, B_EMPTY = B_FULL + STAGES, B_ACCFULL = B_EMPTY + STAGES,
              B_ACCEMPTY = B_ACCFULL + 2, B_RES = B_ACCEMPTY + 2 /* [GROUPS] */,
              B_DRAIN = B_RES + GROUPS, NBAR = B_DRAIN + 1;
constexpr uint32_t OFF_MISC = OFF_BAR + NBAR * 8;  // tmem base, abort flag, votes[GROUPS][2][2][4]
constexpr uint32_t SMEM_BYTES = OFF_MISC + 8 + GROUPS * 16 * 4;
static_assert(SMEM_BYTES <= 232448, "shared memory");

struct Params {
  int64_t m, n;
  int64_t tiles, tiles_n;
  int blocks;   // reduction blocks of a tile
  int workers;
  int split;
  int a_heads64, b_heads64, y_heads64;  // 64-element pieces of a row in one head
  const void* bias;
  const void* gate;
  int act;
  int y_fp32, y_tma, res_tma, z_tma;
  const void* residual;
  int64_t residual_stride;
  void* y;
  int64_t y_stride, y_head_stride;
  void* z;
  int64_t z_stride;
  float* slots;
  int32_t* status;
  uint64_t wait_ns;
  int wait_selftest;
};

// A worker's next piece of work: reduction blocks [k0, k1) of a tile.
struct Walk {
  int64_t at, end, step;
  int blocks;
  bool split;
  int64_t tile;
  int k0, k1;
  __device__ __forceinline__ Walk(const Params& p, int worker) : blocks(p.blocks), split(p.split) {
    if (split) {
      const int64_t units = p.tiles * p.blocks;
      at = worker * units / p.workers;
      end = (worker + 1) * units / p.workers;
    } else {
      at = worker;
      end = p.tiles;
      step = p.workers;
    }
  }
  __device__ __forceinline__ bool next() {
    if (at >= end) return false;
    if (split) {
      tile = at / blocks;
      k0 = (int)(at - tile * blocks);
      k1 = (int)min((int64_t)blocks, k0 + (end - at));
      at += k1 - k0;
    } else {
      tile = at;
      k0 = 0;
      k1 = blocks;
      at += step;
    }
    return true;
  }
};

// tc05.cuh's bounded wait with the clock read late and seldom: the waits here are mostly shorter
// than reading the clock takes, and the time from a block's release to its refill counts.
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, volatile int* abort_flag,
                                     uint64_t limit_ns) {
  uint64_t t0 = 0;
  for (uint32_t spin = 1;; ++spin) {
    if (tc::mbar_try_wait(bar, parity)) return true;
    if ((spin & 63u) == 0u) {
      if (*abort_flag) return false;
      const uint64_t now = tc::globaltimer_ns();
      if (t0 == 0) {
        t0 = now;
      } else if (now - t0 > limit_ns) {
        *abort_flag = 1;
        return false;
      }
    }
  }
}

// ---- what pairs of CTAs need beside tc05.cuh -------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
                   : "memory");
}
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar)
               : "memory");
}

template <int CTA>
struct Pair;
template <>
struct Pair<1> {
  static __device__ __forceinline__ void alloc(uint32_t dst) { tc::tmem_alloc(dst, 256); }
  static __device__ __forceinline__ void relinquish() { tc::tmem_relinquish(); }
  static __device__ __forceinline__ void dealloc(uint32_t t) { tc::tmem_dealloc(t, 256); }
  static __device__ __forceinline__ void load(uint32_t dst, const CUtensorMap* map, uint32_t bar,
                                              int c0, int c1, int c2) {
    tc::tma_load_3d(dst, map, bar, c0, c1, c2);
  }
  static __device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                             uint32_t acc) {
    tc::mma_ss(d, a, b, idesc, acc);
  }
  static __device__ __forceinline__ void commit(uint32_t bar) { tc::mma_commit(bar); }
};
template <>
struct Pair<2> {
  static __device__ __forceinline__ void alloc(uint32_t dst) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(dst)
                 : "memory");
  }
  static __device__ __forceinline__ void relinquish() {
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  static __device__ __forceinline__ void dealloc(uint32_t t) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(t) : "memory");
  }
  // into this CTA's memory, completion on a barrier of either CTA of the pair
  static __device__ __forceinline__ void load(uint32_t dst, const CUtensorMap* map, uint32_t bar,
                                              int c0, int c1, int c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
  }
  static __device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                             uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
  }
  // arrives on the barrier at this address in both CTAs
  static __device__ __forceinline__ void commit(uint32_t bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
        " [%0], %1;" ::"r"(bar),
        "h"((uint16_t)3)
        : "memory");
  }
};

__device__ __forceinline__ void store_3d(const CUtensorMap* map, uint32_t src, int c0, int c1,
                                         int c2) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::
                   "l"(reinterpret_cast<uint64_t>(map)),
               "r"(src), "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}
__device__ __forceinline__ void store_bulk(void* dst, uint32_t src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(src),
               "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void store_commit() {
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// all but the newest N stores have read their buffers
template <int N>
__device__ __forceinline__ void store_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void lds128(uint32_t a, uint32_t* r) {
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a));
}
__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w)
               : "memory");
}

template <typename E>
__device__ __forceinline__ float to_float(E v) {
  return (float)v;
}

// Address of 16-byte piece j of row r in an epilogue buffer (the 128-byte swizzle of TMA).
__device__ __forceinline__ uint32_t piece(uint32_t buf, int r, int j) {
  return buf + (uint32_t)(r * 128 + ((j ^ (r & 7)) << 4));
}

// Copies this warp's 32 rows between an epilogue buffer and memory, element by element: 128 bytes
// of a row, `left` elements of which exist, in the first `rows` rows.
template <typename E>
__device__ __forceinline__ void copy_rows(uint32_t buf, int row0, E* g, int64_t stride, int64_t rows,
                                          int64_t left, bool in) {
  constexpr int kPer = 128 / (int)sizeof(E) / 32, kPiece = 16 / (int)sizeof(E);
  const int lane = threadIdx.x & 31;
  for (int r = 0; r < 32 && r < rows; ++r) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int c = lane * kPer + i;
      if (c >= left) continue;
      const uint32_t a = piece(buf, row0 + r, c / kPiece) + (uint32_t)(c % kPiece) * sizeof(E);
      E* p = g + (int64_t)r * stride + c;
      if (sizeof(E) == 2) {
        uint16_t v;
        if (in) {
          v = *reinterpret_cast<const uint16_t*>(p);
          asm volatile("st.shared.u16 [%0], %1;" ::"r"(a), "h"(v) : "memory");
        } else {
          asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(a) : "memory");
          *reinterpret_cast<uint16_t*>(p) = v;
        }
      } else {
        uint32_t v;
        if (in) {
          v = *reinterpret_cast<const uint32_t*>(p);
          asm volatile("st.shared.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory");
        } else {
          asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
          *reinterpret_cast<uint32_t*>(p) = v;
        }
      }
    }
  }
}

// The stage that comes next and the parity of its round.
struct Ring {
  uint32_t at = 0, turn = 0;
  __device__ __forceinline__ void step() {
    if (++at == STAGES) {
      at = 0;
      turn ^= 1;
    }
  }
};

// The c-th 64 elements of a row whose heads hold `per` of them.
struct Place {
  int x = 0, head = 0;
  Place() = default;
  __device__ __forceinline__ Place(int c, int per) {
    head = c / per;
    x = (c - head * per) * 64;
  }
  __device__ __forceinline__ void step(int per) {
    x += 64;
    if (per != INT_MAX && x == per * 64) {
      x = 0;
      ++head;
    }
  }
};

// What one use of an epilogue buffer holds.
enum { kUseZ, kUseY, kUseSlot };

template <typename T, int CTA, bool AMN, bool BMN, bool SPLIT>
__global__ void __launch_bounds__(THREADS, 1)
    product_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                   const __grid_constant__ CUtensorMap tm_y,
                   const __grid_constant__ CUtensorMap tm_res,
                   const __grid_constant__ CUtensorMap tm_z, const Params p) {
  constexpr int BN = 128 * CTA;  // columns of a tile; 128 of B's rows lie in each CTA
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  // the swizzle wants 1024-byte borders, where dynamic shared memory begins as long as there is no
  // static one; there is no room to move up
  const uint32_t base = smem_u32(smem_raw);
  if (base & 1023u) {
    if (threadIdx.x == 0 && p.status != nullptr) atomicOr(p.status, VGGT_STATUS_TIMEOUT);
    return;
  }
  unsigned char* sbase = smem_raw;
  auto bar = [&](int i) { return base + OFF_BAR + 8u * (uint32_t)i; };
  uint32_t* misc = reinterpret_cast<uint32_t*>(sbase + OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(misc + 1);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = CTA == 2 ? (int)cluster_rank() : 0;
  const int worker = (int)blockIdx.x / CTA;

  if (tid == 0) {
    for (int s = 0; s < STAGES; ++s) {
      tc::mbar_init(bar(B_FULL + s), 1);
      tc::mbar_init(bar(B_EMPTY + s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      tc::mbar_init(bar(B_ACCFULL + b), 1);
      tc::mbar_init(bar(B_ACCEMPTY + b), 4 * GROUPS * CTA);
    }
    for (int b = 0; b < GROUPS; ++b) tc::mbar_init(bar(B_RES + b), 1);
    tc::mbar_init(bar(B_DRAIN), 1);
    misc[1] = 0u;
    tc::mbar_fence_init();
  }
  if (warp == 2) {
    Pair<CTA>::alloc(base + OFF_MISC);
    Pair<CTA>::relinquish();
  }
  tc::tc_fence_before();
  __syncthreads();
  if (CTA == 2) cluster_sync();
  tc::tc_fence_after();
  const uint32_t tmem = misc[0];

  if (warp == 0) {
    // ================= TMA producer =================
    if (lane == 0) {
      const uint32_t full0 = CTA == 2 ? map_rank(bar(B_FULL), 0) : bar(B_FULL);
      tc::prefetch_tmap(&tm_a);
      tc::prefetch_tmap(&tm_b);
      Walk w(p, worker);
      Ring ring;
      uint32_t issued = 0;
      bool ok = true;
      while (ok && w.next()) {
        const int m0 = (int)(w.tile / p.tiles_n) * BN + rank * BM;
        const int n0 = (int)(w.tile % p.tiles_n) * BN + rank * BM;
        // where the operands' first blocks lie: one thread feeds the tensor core here, so that
        // no division is left in the loop
        Place a0, a1, b0, b1;
        if (AMN) {
          a0 = Place(m0 / 64, p.a_heads64);
          a1 = Place(m0 / 64 + 1, p.a_heads64);
        } else {
          a0 = Place(w.k0, p.a_heads64);
        }
        if (BMN) {
          b0 = Place(n0 / 64, p.b_heads64);
          b1 = Place(n0 / 64 + 1, p.b_heads64);
        } else {
          b0 = Place(w.k0, p.b_heads64);
        }
        for (int k = w.k0; k < w.k1; ++k) {
          if (issued >= STAGES &&
              !wait(bar(B_EMPTY) + 8 * ring.at, ring.turn ^ 1, abort_flag, p.wait_ns)) {
            ok = false;
            break;
          }
          // the barrier is the first CTA's: it counts both CTAs' bytes
          const uint32_t full = full0 + 8 * ring.at;
          if (rank == 0) tc::mbar_expect_tx(bar(B_FULL) + 8 * ring.at, CTA * STAGE_BYTES);
          const uint32_t a = base + ring.at * STAGE_BYTES, b = a + HALF_BYTES;
          if (AMN) {
            Pair<CTA>::load(a, &tm_a, full, a0.x, k * BK, a0.head);
            Pair<CTA>::load(a + HALF_BYTES / 2, &tm_a, full, a1.x, k * BK, a1.head);
          } else {
            Pair<CTA>::load(a, &tm_a, full, a0.x, m0, a0.head);
            a0.step(p.a_heads64);
          }
          if (BMN) {
            Pair<CTA>::load(b, &tm_b, full, b0.x, k * BK, b0.head);
            Pair<CTA>::load(b + HALF_BYTES / 2, &tm_b, full, b1.x, k * BK, b1.head);
          } else {
            Pair<CTA>::load(b, &tm_b, full, b0.x, n0, b0.head);
            b0.step(p.b_heads64);
          }
          ring.step();
          ++issued;
        }
      }
      // the last copies have landed before the memory goes (the MMAs that read them are awaited
      // by their issuer)
      if (rank == 0)
        for (uint32_t t = issued > STAGES ? issued - STAGES : 0; t < issued; ++t)
          tc::mbar_wait_drain(bar(B_FULL + t % STAGES), (t / STAGES) & 1, p.wait_ns);
    }
  } else if (warp == 1) {
    // ================= MMA issuer (of the pair's first CTA) =================
    if (lane == 0 && rank == 0) {
      const uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
      const uint32_t idesc = tc::idesc_f16(fmt, BMN ? 1u : 0u, BN, BN) | (AMN ? 1u << 15 : 0u);
      // a step of 16 reduced elements: 32 bytes along a K-major row, 16 MN-major rows
      constexpr uint64_t kStepA = AMN ? 16 * 128 / 16 : 2, kStepB = BMN ? 16 * 128 / 16 : 2;
      const uint64_t desc0 = tc::sw128_desc(base, HALF_BYTES / 2);
      bool ok = true;
      if (p.wait_selftest) ok = wait(bar(B_DRAIN), 0, abort_flag, p.wait_ns);
      Walk w(p, worker);
      Ring ring;
      uint32_t i = 0;
      while (ok && w.next()) {
        const uint32_t b = i & 1;
        if (i >= 2 &&
            !wait(bar(B_ACCEMPTY + b), ((i >> 1) + 1) & 1, abort_flag, p.wait_ns)) {
          ok = false;
          break;
        }
        tc::tc_fence_after();
        const uint32_t acc = tmem + b * BN;
        for (int k = w.k0; k < w.k1; ++k) {
          if (!wait(bar(B_FULL) + 8 * ring.at, ring.turn, abort_flag, p.wait_ns)) {
            ok = false;
            break;
          }
          tc::tc_fence_after();
          const uint64_t ad = desc0 + ring.at * (STAGE_BYTES / 16), bd = ad + HALF_BYTES / 16;
#pragma unroll
          for (int kk = 0; kk < BK / 16; ++kk)
            Pair<CTA>::mma(acc, ad + kk * kStepA, bd + kk * kStepB, idesc,
                           (k > w.k0 || kk > 0) ? 1u : 0u);
          Pair<CTA>::commit(bar(B_EMPTY) + 8 * ring.at);
          ring.step();
        }
        if (ok) Pair<CTA>::commit(bar(B_ACCFULL + b));
        ++i;
      }
      if (!p.wait_selftest) {
        Pair<CTA>::commit(bar(B_DRAIN));
        tc::mbar_wait_drain(bar(B_DRAIN), 0, p.wait_ns);
      }
    }
  } else if (warp >= 4) {
    // ================= epilogue: group g takes columns 64 g .. 64 g + 63 of a tile =================
    const int g = (warp - 4) >> 2, sub = warp & 3, row = sub * 32 + lane, t = tid & 127;
    const uint32_t lanes = (uint32_t)(sub * 32) << 16;
    float* vec = reinterpret_cast<float*>(sbase + OFF_VEC) + g * 128;  // bias | gate
    int* votes = reinterpret_cast<int*>(misc + 2) + g * 16;
    const uint32_t buf = base + OFF_BUF + (uint32_t)g * BUF_BYTES, res_bar = bar(B_RES + g);
    auto group_sync = [&] { asm volatile("bar.sync %0, 128;" ::"r"(1 + g) : "memory"); };
    // true in all four warps or in none: the barriers of a group are not bounded, so that its
    // warps have to leave together
    auto agree = [&](int at, bool ok) {
      const bool all = __all_sync(0xffffffffu, ok);
      volatile int* v = votes + at;
      if (lane == 0) v[sub] = all ? 1 : 0;
      group_sync();
      return v[0] && v[1] && v[2] && v[3];
    };
    const bool has_res = !SPLIT && p.residual != nullptr, has_z = !SPLIT && p.z != nullptr;
    auto fetch_residual = [&](int64_t c0, int64_t m0) {  // by one thread
      store_wait_read<0>();  // the buffer's last store has read it
      tc::mbar_expect_tx(res_bar, BUF_BYTES);
      tc::tma_load_3d(buf, &tm_res, res_bar, (int)c0, (int)m0, 0);
    };
    Walk w(p, worker);
    uint32_t i = 0, uses = 0, res_uses = 0;
    bool ok = true;
    while (ok && w.next()) {
      const uint32_t b = i & 1;
      const int64_t m0 = w.tile / p.tiles_n * BN + rank * BM;
      const int64_t col = w.tile % p.tiles_n * BN + g * 64;
      const bool active = g < BN / 64 && col < p.n;
      bool fetched = false;
      if (!SPLIT && active) {
        // seen by the group after the next barrier; the last readers are before the last one
        const int64_t c = col + (t & 63);
        float v = t < 64 ? 0.f : 1.f;
        const T* src = static_cast<const T*>(t < 64 ? p.bias : p.gate);
        if (src != nullptr && c < p.n) v = to_float(src[c]);
        vec[t] = v;
        fetched = has_res && p.res_tma && !has_z;
        if (fetched && t == 0) fetch_residual(col, m0);
        __syncwarp();
      }
      const bool got = wait(bar(B_ACCFULL + b), (i >> 1) & 1, abort_flag, p.wait_ns);
      if (!agree(4 * b, got)) {
        ok = false;
        break;
      }
      tc::tc_fence_after();
      const uint32_t acc = tmem + b * BN + lanes + g * 64;
      const int first = has_z ? kUseZ : SPLIT ? kUseSlot : kUseY;
      for (int kind = first; active && ok && kind <= (SPLIT ? kUseSlot : kUseY); ++kind) {
        // a buffer row is 64 elements of T or 32 of fp32
        const bool wide = SPLIT || (kind == kUseY && p.y_fp32);
        for (int part = 0; part < (wide ? 2 : 1); ++part, ++uses) {
          const int64_t c0 = col + part * 32;  // first column of the use
          if (!SPLIT && c0 >= p.n) break;
          const bool res = kind == kUseY && has_res;
          bool fine = true;
          if (res && p.res_tma) {
            if (t == 0 && !fetched) fetch_residual(c0, m0);
            fetched = false;
            __syncwarp();
            fine = wait(res_bar, res_uses & 1, abort_flag, p.wait_ns);
            ++res_uses;
          } else if (t == 0) {
            store_wait_read<0>();
          }
          if (!agree(8 + 4 * (uses & 1), fine)) {
            ok = false;
            break;
          }
          const int64_t r0 = m0 + sub * 32, rows = p.m - r0, left = p.n - c0;  // this warp's rows
          if (res && !p.res_tma) {
            const int64_t at = r0 * p.residual_stride + c0;
            if (p.y_fp32)
              copy_rows(buf, sub * 32, const_cast<float*>(static_cast<const float*>(p.residual)) + at,
                        p.residual_stride, rows, left, true);
            else
              copy_rows(buf, sub * 32, const_cast<T*>(static_cast<const T*>(p.residual)) + at,
                        p.residual_stride, rows, left, true);
            __syncwarp();
          }
          // 32 columns at a time: TMEM -> registers -> buffer
          for (int h = wide ? part : 0; h < (wide ? part + 1 : 2); ++h) {
            uint32_t r[32];
            tc::tmem_ld32(acc + h * 32, r);
            tc::tmem_wait_ld();
            if (SPLIT) {
#pragma unroll
              for (int j = 0; j < 8; ++j)
                sts128(piece(buf, row, j), r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
              continue;
            }
            const ulonglong2* bv = reinterpret_cast<const ulonglong2*>(vec + h * 32);
            float_pair v[16];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const ulonglong2 q = bv[j];
              v[2 * j] = add_pair(
                  pack_pair(__uint_as_float(r[4 * j]), __uint_as_float(r[4 * j + 1])), q.x);
              v[2 * j + 1] = add_pair(
                  pack_pair(__uint_as_float(r[4 * j + 2]), __uint_as_float(r[4 * j + 3])), q.y);
            }
            if (kind == kUseY) {
              act::dispatch(p.act, [&](auto k) {
#pragma unroll
                for (int j = 0; j < 16; ++j) v[j] = act::value_pair<decltype(k)::value>(v[j]);
              });
              if (p.gate != nullptr) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                  const ulonglong2 q = bv[16 + j];
                  v[2 * j] = mul_pair(v[2 * j], q.x);
                  v[2 * j + 1] = mul_pair(v[2 * j + 1], q.y);
                }
              }
            }
            if (wide) {
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const uint32_t a = piece(buf, row, j);
                uint32_t q[4];
                if (res) {
                  lds128(a, q);
                  v[2 * j] =
                      add_pair(v[2 * j], pack_pair(__uint_as_float(q[0]), __uint_as_float(q[1])));
                  v[2 * j + 1] = add_pair(v[2 * j + 1],
                                          pack_pair(__uint_as_float(q[2]), __uint_as_float(q[3])));
                }
                float o[4];
                unpack_pair(o[0], o[1], v[2 * j]);
                unpack_pair(o[2], o[3], v[2 * j + 1]);
                sts128(a, __float_as_uint(o[0]), __float_as_uint(o[1]), __float_as_uint(o[2]),
                       __float_as_uint(o[3]));
              }
            } else {
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const uint32_t a = piece(buf, row, h * 4 + j);
                uint32_t q[4];
                if (res) {
                  lds128(a, q);
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    const float2 f = ElemOps<T>::to_float2(q[e]);
                    v[4 * j + e] = add_pair(v[4 * j + e], pack_pair(f.x, f.y));
                  }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  float x0, x1;
                  unpack_pair(x0, x1, v[4 * j + e]);
                  q[e] = ElemOps<T>::pack2(x0, x1);
                }
                sts128(a, q[0], q[1], q[2], q[3]);
              }
            }
          }
          if (SPLIT || (kind == kUseZ ? p.z_tma : p.y_tma)) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            group_sync();
            if (t == 0) {
              if (SPLIT) {
                const int64_t slot = worker + w.tile;
                store_bulk(reinterpret_cast<unsigned char*>(p.slots) +
                               ((slot * CTA + rank) * (BN / 32) + g * 2 + part) * BUF_BYTES,
                           buf, BUF_BYTES);
              } else if (m0 < p.m) {
                const int head = (int)(c0 / 64) / p.y_heads64;
                if (kind == kUseZ)
                  store_3d(&tm_z, buf, (int)c0, (int)m0, 0);
                else
                  store_3d(&tm_y, buf, (int)(c0 - (int64_t)head * p.y_heads64 * 64), (int)m0, head);
              }
              store_commit();
            }
          } else {
            __syncwarp();
            if (kind == kUseZ) {
              copy_rows(buf, sub * 32, static_cast<T*>(p.z) + r0 * p.z_stride + c0, p.z_stride, rows,
                        left, false);
            } else if (p.y_fp32) {
              copy_rows(buf, sub * 32, static_cast<float*>(p.y) + r0 * p.y_stride + c0, p.y_stride,
                        rows, left, false);
            } else {
              const int64_t head = c0 / 64 / p.y_heads64, in_head = c0 - head * p.y_heads64 * 64;
              copy_rows(buf, sub * 32,
                        static_cast<T*>(p.y) + head * p.y_head_stride + r0 * p.y_stride + in_head,
                        p.y_stride, rows, left, false);
            }
            // the buffer's next use may begin with a copy by TMA
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            group_sync();
          }
        }
      }
      if (!ok) break;
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (CTA == 2)
          arrive_cluster(map_rank(bar(B_ACCEMPTY + b), 0));
        else
          tc::mbar_arrive(bar(B_ACCEMPTY + b));
      }
      ++i;
    }
    if (t == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }

  tc::tc_fence_before();
  __syncthreads();
  __syncwarp();
  if (CTA == 2) cluster_sync();
  tc::tc_fence_after();
  if (tid == 0 && *abort_flag && p.status != nullptr) atomicOr(p.status, VGGT_STATUS_TIMEOUT);
  if (warp == 2) Pair<CTA>::dealloc(tmem);
}

// Adds up a split product's partial sums and runs the epilogue: a thread takes 8 columns of a row.
template <typename T>
__global__ void __launch_bounds__(256)
    finish_kernel(const Slots s, int64_t m, int64_t n, const Epilogue e, bool wide) {
  const int64_t groups = (n + 7) / 8, all = m * groups;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < all;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / groups, c = (i - r * groups) * 8;
    const int k = (int)min((int64_t)8, n - c);
    float v[8];
    s.get8(r, c, v);
    float t[8];
    if (e.bias != nullptr) {
      get8(static_cast<const T*>(e.bias) + c, k, wide, t);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += t[j];
    }
    if (e.z != nullptr) put8(static_cast<T*>(e.z) + r * e.z_stride + c, k, wide, v);
    act::dispatch(e.act, [&](auto kind) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = act::value<decltype(kind)::value>(v[j]);
    });
    if (e.gate != nullptr) {
      get8(static_cast<const T*>(e.gate) + c, k, wide, t);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= t[j];
    }
    const bool fp32 = e.y_type == VGGT_DTYPE_FP32;
    if (e.residual != nullptr) {
      const int64_t at = r * e.residual_stride + c;
      if (fp32)
        get8(static_cast<const float*>(e.residual) + at, k, wide, t);
      else
        get8(static_cast<const T*>(e.residual) + at, k, wide, t);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += t[j];
    }
    const int64_t head = c / e.y_dim;
    const int64_t at = head * e.y_head_stride + r * e.y_stride + (c - head * e.y_dim);
    if (fp32)
      put8(static_cast<float*>(e.y) + at, k, wide, v);
    else
      put8(static_cast<T*>(e.y) + at, k, wide, v);
  }
}

// ---- host -------------------------------------------------------------------------------------
size_t Plan::slot_bytes() const {
  return split ? (size_t)(workers + tiles_m * tiles_n) * cta * cta * BM * 128 * 4 : 0;
}

static int sm_count() {
  int sms = 0;
  return device_sms(&sms) == cudaSuccess && sms > 0 ? sms : 148;
}

// The way a product is cut is the one of the least estimated time, in SM cycles: a reduction block
// takes a pair of CTAs 512 cycles (the MMAs' time) and a single CTA 256, or up to twice that when
// all SMs read their operands from L2 at once.  Splitting evens the load out where tiles are few
// or the last round is short, at the price of partial sums through memory and another launch.
Plan plan_product(int64_t m, int64_t n, int64_t red, bool must_split) {
  const int sms = sm_count();
  Plan best;
  double least = 0;
  for (int cta = 1; cta <= 2; ++cta)
    for (int split = must_split ? 1 : 0; split < 2; ++split) {
      Plan p;
      p.cta = cta;
      p.split = split;
      p.tiles_m = (m + 128 * cta - 1) / (128 * cta);
      p.tiles_n = (n + 128 * cta - 1) / (128 * cta);
      p.blocks = (red + BK - 1) / BK;
      const int64_t tiles = p.tiles_m * p.tiles_n, units = split ? tiles * p.blocks : tiles;
      p.workers = (int)std::min<int64_t>(sms / cta, units);
      const double busy = (double)p.workers * cta / sms;
      const double block = cta == 2 ? 512 : 256 * std::max(1.0, 2 * busy);
      const int64_t rounds = (units + p.workers - 1) / p.workers;
      double t = (double)rounds * (split ? 1 : p.blocks) * block;
      if (split) t += 5000 + (double)p.slot_bytes() * 2 / 2500;
      if (least == 0 || t < least) {
        least = t;
        best = p;
      }
    }
  return best;
}

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

static bool operand_map(CUtensorMap* map, const Operand& o, int dtype, int64_t rows) {
  const uint64_t dims[3] = {(uint64_t)o.dim, (uint64_t)rows, (uint64_t)o.heads};
  // a stride that is never used may be anything: give a valid one
  const int64_t row = rows > 1 ? o.stride : (o.dim + 7) / 8 * 8;
  const uint64_t strides[2] = {(uint64_t)row * 2,
                               (uint64_t)(o.heads > 1 ? o.head_stride : row * rows) * 2};
  const uint32_t box[3] = {64, o.mn_major ? (uint32_t)BK : (uint32_t)BM, 1};
  return encode_tmap_sw128(map, o.p, dtype, 3, dims, strides, box);
}

// Rows of an output or of the residual, for copies of 128 rows x 128 bytes; false where TMA
// cannot address them.
static bool rows_map(CUtensorMap* map, const void* p, int type, int64_t stride, int64_t head_stride,
                     int64_t heads, int64_t dim, int64_t rows) {
  const int per = type == VGGT_DTYPE_FP32 ? 4 : 8, size = 16 / per;
  if (!aligned16(p) || dim % per || (rows > 1 && stride % per) || (heads > 1 && head_stride % per))
    return false;
  const int64_t row = rows > 1 ? stride : dim;
  const uint64_t dims[3] = {(uint64_t)dim, (uint64_t)rows, (uint64_t)heads};
  const uint64_t strides[2] = {(uint64_t)row * size,
                               (uint64_t)(heads > 1 ? head_stride : row * rows) * size};
  const uint32_t box[3] = {(uint32_t)(128 / size), (uint32_t)BM, 1};
  return encode_tmap_sw128(map, p, type, 3, dims, strides, box);
}

template <typename T, int CTA, bool AMN, bool BMN, bool SPLIT>
static cudaError_t launch_kernel(const CUtensorMap* maps, const Params& p, cudaStream_t stream) {
  auto k = product_kernel<T, CTA, AMN, BMN, SPLIT>;
  cudaError_t e =
      cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM_BYTES);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(p.workers * CTA));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = SMEM_BYTES;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CTA;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, k, maps[0], maps[1], maps[2], maps[3], maps[4], p);
  return e != cudaSuccess ? e : cudaGetLastError();
}

template <typename T, int CTA>
static cudaError_t launch_majors(bool amn, bool bmn, bool split, const CUtensorMap* maps,
                                 const Params& p, cudaStream_t stream) {
  if (!amn && !bmn)
    return split ? launch_kernel<T, CTA, false, false, true>(maps, p, stream)
                 : launch_kernel<T, CTA, false, false, false>(maps, p, stream);
  if (!amn)
    return split ? launch_kernel<T, CTA, false, true, true>(maps, p, stream)
                 : launch_kernel<T, CTA, false, true, false>(maps, p, stream);
  // the weight's gradient is always split
  return split && bmn ? launch_kernel<T, CTA, true, true, true>(maps, p, stream)
                      : cudaErrorInvalidValue;
}

cudaError_t launch_product(const Plan& plan, int dtype, int64_t m, int64_t n, int64_t red,
                           const Operand& a, const Operand& b, const Epilogue& e, float* slots,
                           int32_t* status, cudaStream_t stream) {
  CUtensorMap maps[5] = {};
  if (!operand_map(&maps[0], a, dtype, a.mn_major ? red : m) ||
      !operand_map(&maps[1], b, dtype, b.mn_major ? red : n))
    return cudaErrorInvalidValue;
  Params p{};
  p.m = m;
  p.n = n;
  p.tiles = plan.tiles_m * plan.tiles_n;
  p.tiles_n = plan.tiles_n;
  p.blocks = (int)plan.blocks;
  p.workers = plan.workers;
  p.split = plan.split;
  auto heads64 = [](int64_t heads, int64_t dim) { return heads > 1 ? (int)(dim / 64) : INT_MAX; };
  p.a_heads64 = heads64(a.heads, a.dim);
  p.b_heads64 = heads64(b.heads, b.dim);
  p.y_heads64 = heads64(e.y_heads, e.y_dim);
  p.bias = e.bias;
  p.gate = e.gate;
  p.act = e.act;
  p.y_fp32 = e.y_type == VGGT_DTYPE_FP32;
  p.residual = e.residual;
  p.residual_stride = e.residual_stride;
  p.y = e.y;
  p.y_stride = e.y_stride;
  p.y_head_stride = e.y_head_stride;
  p.z = e.z;
  p.z_stride = e.z_stride;
  if (!plan.split) {
    p.y_tma = rows_map(&maps[2], e.y, e.y_type, e.y_stride, e.y_head_stride, e.y_heads, e.y_dim, m);
    p.res_tma = e.residual &&
                rows_map(&maps[3], e.residual, e.y_type, e.residual_stride, 0, 1, n, m);
    p.z_tma = e.z && rows_map(&maps[4], e.z, dtype, e.z_stride, 0, 1, n, m);
  }
  p.slots = slots;
  p.status = status;
  p.wait_ns = api_wait_ns();
  p.wait_selftest = api_wait_selftest();
  const bool am = a.mn_major, bm = b.mn_major;
  if (dtype == VGGT_DTYPE_BF16)
    return plan.cta == 2 ? launch_majors<__nv_bfloat16, 2>(am, bm, plan.split, maps, p, stream)
                         : launch_majors<__nv_bfloat16, 1>(am, bm, plan.split, maps, p, stream);
  return plan.cta == 2 ? launch_majors<__half, 2>(am, bm, plan.split, maps, p, stream)
                       : launch_majors<__half, 1>(am, bm, plan.split, maps, p, stream);
}

Slots slots_of(const Plan& plan, const float* p) {
  return {p, plan.tiles_m * plan.tiles_n * plan.blocks, plan.tiles_n, plan.cta, (int)plan.blocks,
          plan.workers};
}

cudaError_t finish_product(const Plan& plan, int dtype, int64_t m, int64_t n, const Epilogue& e,
                           const float* slots, cudaStream_t stream) {
  const int64_t all = m * ((n + 7) / 8);
  const unsigned grid = (unsigned)std::min<int64_t>((all + 255) / 256, 148 * 16);
  const bool wide = wide_rows(e.y, e.y_stride, e.y_type) && e.y_dim % 8 == 0 &&
                    (e.y_heads <= 1 || e.y_head_stride % 8 == 0) &&
                    wide_rows(e.z, e.z_stride, dtype) && wide_rows(e.bias, 8, dtype) &&
                    wide_rows(e.gate, 8, dtype) &&
                    wide_rows(e.residual, e.residual_stride, e.y_type);
  const Slots s = slots_of(plan, slots);
  if (dtype == VGGT_DTYPE_BF16)
    finish_kernel<__nv_bfloat16><<<grid, 256, 0, stream>>>(s, m, n, e, wide);
  else
    finish_kernel<__half><<<grid, 256, 0, stream>>>(s, m, n, e, wide);
  return cudaGetLastError();
}

}  // namespace lin
}  // namespace vggt

// ---- C ABI ------------------------------------------------------------------------------------
namespace vggt {
namespace lin {

int check(const vggt_linear_args* a) {
  if (!a) return api_fail("args must be non-NULL");
  if (a->dtype != VGGT_DTYPE_BF16 && a->dtype != VGGT_DTYPE_FP16)
    return api_fail("linear requires BF16 or FP16");
  if (a->stream_dtype != a->dtype && a->stream_dtype != VGGT_DTYPE_FP32)
    return api_fail("the residual and y are of x's type or FP32");
  if (a->rows < 0 || a->inner < 1 || a->outer < 1) return api_fail("bad size argument");
  if (a->rows > INT_MAX - 512 || a->inner > INT_MAX - 512 || a->outer > INT_MAX - 512)
    return api_fail("too many rows or too wide");
  if (a->inner % 8) return api_fail("inner (%lld) must be a multiple of 8", (long long)a->inner);
  if (a->heads > 1 && (a->inner % a->heads || a->inner / a->heads % 64))
    return api_fail("a head-major x needs heads of a multiple of 64 elements");
  if (a->activation < VGGT_ACT_NONE || a->activation > VGGT_ACT_RELU)
    return api_fail("unknown activation %d", a->activation);
  if (a->rows == 0) return 0;
  if (!a->x || !a->weight) return api_fail("x and weight must be non-NULL");
  const int64_t dim = a->heads > 1 ? a->inner / a->heads : a->inner;
  if (!aligned16(a->x) || !aligned16(a->weight) || (a->rows > 1 && a->x_stride % 8) ||
      (a->heads > 1 && a->x_head_stride % 8) || (a->outer > 1 && a->weight_stride % 8))
    return api_fail("x and weight must start on 16 bytes, with strides that are multiples of 8");
  if ((a->rows > 1 && a->x_stride < dim) || (a->heads > 1 && a->x_head_stride < dim) ||
      (a->outer > 1 && a->weight_stride < a->inner))
    return api_fail("a stride of x or weight is below the row's width");
  if (a->residual && a->rows > 1 && a->residual_stride < 0) return api_fail("negative stride");
  return 0;
}

Operand x_operand(const vggt_linear_args* a, bool mn_major) {
  const int64_t heads = a->heads > 1 ? a->heads : 1;
  Operand o;
  o.p = a->x;
  o.stride = a->x_stride;
  o.head_stride = a->x_head_stride;
  o.heads = heads;
  o.dim = a->inner / heads;
  o.mn_major = mn_major;
  return o;
}

Operand matrix(const void* p, int64_t width, int64_t stride, bool mn_major) {
  Operand o;
  o.p = p;
  o.stride = stride;
  o.dim = width;
  o.mn_major = mn_major;
  return o;
}

}  // namespace lin
}  // namespace vggt

extern "C" size_t vggt_linear_workspace_size(const vggt_linear_args* a) {
  using namespace vggt::lin;
  if (!a || a->rows <= 0 || a->inner < 1 || a->outer < 1) return 0;
  return plan_product(a->rows, a->outer, a->inner, false).slot_bytes();
}

extern "C" int vggt_linear(const vggt_linear_args* a, void* y, int64_t y_stride, void* z,
                           int64_t z_stride, int32_t* status, void* workspace,
                           size_t workspace_bytes, void* stream) {
  using namespace vggt;
  using namespace vggt::lin;
  if (int rc = check(a)) return rc;
  if (a->rows == 0) return api_fail(nullptr);
  if (!y) return api_fail("y must be non-NULL");
  if (a->rows > 1 && (y_stride < a->outer || (z && z_stride < a->outer)))
    return api_fail("an output's rows overlap: its stride is below outer");
  const Plan plan = plan_product(a->rows, a->outer, a->inner, false);
  if (plan.slot_bytes() > 0 &&
      (!workspace || !aligned16(workspace) || workspace_bytes < plan.slot_bytes()))
    return api_fail("the workspace is too small or not 16-byte aligned");
  Epilogue e;
  e.bias = a->bias;
  e.gate = a->gate;
  e.act = a->activation;
  e.residual = a->residual;
  e.residual_stride = a->residual_stride;
  e.y = y;
  e.y_stride = y_stride;
  e.y_dim = a->outer;
  e.y_type = a->stream_dtype;
  e.z = z;
  e.z_stride = z_stride;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  float* slots = static_cast<float*>(workspace);
  cudaError_t rc = launch_product(plan, a->dtype, a->rows, a->outer, a->inner, x_operand(a, false),
                                  matrix(a->weight, a->inner, a->weight_stride, false), e, slots,
                                  status, st);
  if (rc == cudaSuccess && plan.split)
    rc = finish_product(plan, a->dtype, a->rows, a->outer, e, slots, st);
  return api_cuda(rc);
}
