// Matrix product on the tensor cores with bias, activation, gate and residual in its epilogue.
//
// A tile of C is worked on by one CTA (128 x 64 or 128 x 128 elements) or by a pair (256 x 128 or
// 256 x 256: each holds half of A's rows and half of B's, the MMA of the pair reads both halves of
// B).  Warp 0 streams the operands by TMA through a ring of 64-element reduction blocks, warp 1
// issues the MMAs into one of two accumulators in TMEM, and warps 4-19, four warpgroups of which
// each takes a quarter of the columns, 32 at least (of 64 columns two take all), run the epilogue of
// the tile before: TMEM -> registers -> bias, activation, gate, residual -> the group's swizzled
// 16 KB buffer -> TMA store.  The residual comes by TMA into the same buffer before.  What TMA
// cannot address (odd widths, other strides) is copied between buffer and memory by the warps that
// own the rows.  (With two warpgroups an activation's latencies bounded the kernel.)
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
constexpr int GROUPS = 4;                     // warpgroups of the epilogue
constexpr int THREADS = 128 + GROUPS * 128;
constexpr uint32_t A_BYTES = BM * BK * 2;     // A's block: 16 KB
constexpr uint32_t BUF_BYTES = BM * 128;      // epilogue buffer: 128 rows of up to 128 bytes

// BNC of B's rows (columns of C) lie in each CTA.
template <int CTA, int BNC>
struct Shape {
  static constexpr int BN = BNC * CTA;
  static constexpr int COLS = BN / GROUPS > 32 ? BN / GROUPS : 32;  // of one epilogue group
  static constexpr uint32_t B_BYTES = BNC * BK * 2, STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int STAGES = BNC == 128 ? 5 : 6;
  static constexpr uint32_t TMEM_COLS = 2 * BN;                       // two accumulators
  static constexpr uint32_t OFF_BUF = STAGES * STAGE_BYTES;           // [GROUPS]
  static constexpr uint32_t OFF_VEC = OFF_BUF + GROUPS * BUF_BYTES;   // float[GROUPS][bias 64, gate 64]
  static constexpr uint32_t OFF_BAR = OFF_VEC + GROUPS * 128 * 4;
  static constexpr int B_FULL = 0, B_EMPTY = B_FULL + STAGES, B_ACCFULL = B_EMPTY + STAGES,
                       B_ACCEMPTY = B_ACCFULL + 2, B_RES = B_ACCEMPTY + 2 /* [GROUPS] */,
                       B_DRAIN = B_RES + GROUPS, NBAR = B_DRAIN + 1;
  // tmem base, abort flag, votes[GROUPS][2][4]
  static constexpr uint32_t OFF_MISC = OFF_BAR + NBAR * 8;
  static constexpr uint32_t SMEM_BYTES = OFF_MISC + 8 + GROUPS * 8 * 4;
  static_assert(SMEM_BYTES <= 232448 && TMEM_COLS <= 512, "shared memory and TMEM");
};

struct Params {
  int64_t m, n;
  uint32_t tiles, tiles_n;
  uint32_t blocks;     // reduction blocks of a tile
  uint32_t workers;
  uint32_t per, rest;  // of a split product, see Slots
  int a_heads64, b_heads64, y_heads64;  // 64-element pieces of a row in one head
  const void* bias;
  const void* gate;
  int act;
  int y_fp32, z_fp32, gate_fp32, y_tma, res_tma, z_tma;
  const void* residual;
  int64_t residual_stride;
  void* y;
  int64_t y_stride, y_head_stride;
  void* z;
  int64_t z_stride;
  const void* row_gate;  // see Epilogue
  float* row_dot;
  float* slots;
  int32_t* status;
  uint64_t wait_ns;
  int wait_selftest;
};

// A worker's next piece of work: reduction blocks [k0, k1) of tile (tm, tn).
template <bool SPLIT>
struct Walk {
  const Params& p;
  uint32_t at, end;
  uint32_t tile, tm, tn;
  int k0, k1;
  __device__ __forceinline__ Walk(const Params& params, uint32_t worker) : p(params) {
    at = SPLIT ? worker * p.per + min(worker, p.rest) : worker;
    end = SPLIT ? at + p.per + (worker < p.rest ? 1 : 0) : p.tiles;
  }
  __device__ __forceinline__ bool next() {
    if (at >= end) return false;
    if (SPLIT) {
      tile = at / p.blocks;
      k0 = (int)(at - tile * p.blocks);
      k1 = (int)min(p.blocks, k0 + (end - at));
      at += k1 - k0;
    } else {
      tile = at;
      k0 = 0;
      k1 = (int)p.blocks;
      at += p.workers;
    }
    tm = tile / p.tiles_n;
    tn = tile - tm * p.tiles_n;
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

// The wait of a full warp: true on all lanes or on none, and the branch on it is uniform.  (The roles
// that feed the tensor core run as whole warps and elect a lane to issue: the instructions take
// their descriptors from uniform registers then.  Issued under `lane == 0` an MMA took 63 cycles to
// get out, and four of them as long as a 128 x 128 block's multiplication.)
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, volatile int* abort_flag,
                                          uint64_t limit_ns) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "vote.sync.all.pred q, p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  if (ok) return true;
  return __all_sync(0xffffffffu, wait(bar, parity, abort_flag, limit_ns));
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
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

template <int CTA>
struct Pair;
template <>
struct Pair<1> {
  static __device__ __forceinline__ void alloc(uint32_t dst, uint32_t n) { tc::tmem_alloc(dst, n); }
  static __device__ __forceinline__ void relinquish() { tc::tmem_relinquish(); }
  static __device__ __forceinline__ void dealloc(uint32_t t, uint32_t n) { tc::tmem_dealloc(t, n); }
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
  static __device__ __forceinline__ void alloc(uint32_t dst, uint32_t n) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst),
                 "r"(n)
                 : "memory");
  }
  static __device__ __forceinline__ void relinquish() {
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  static __device__ __forceinline__ void dealloc(uint32_t t, uint32_t n) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(t), "r"(n) : "memory");
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

// Address of 16-byte piece j of row r in an epilogue buffer with rows of 128 or 64 bytes (TMA's
// swizzle of that many bytes).
template <int ROW>
__device__ __forceinline__ uint32_t piece(uint32_t buf, int r, int j) {
  if (ROW == 64) return buf + (uint32_t)(r * 64 + ((j ^ ((r >> 1) & 3)) << 4));
  return buf + (uint32_t)(r * 128 + ((j ^ (r & 7)) << 4));
}

// Copies this warp's 32 rows between an epilogue buffer and memory, element by element: ROW bytes
// of a row, `left` elements of which exist, in the first `rows` rows.
template <int ROW, typename E>
__device__ __forceinline__ void copy_rows(uint32_t buf, int row0, E* g, int64_t stride, int64_t rows,
                                          int64_t left, bool in) {
  constexpr int kPer = ROW / (int)sizeof(E) / 32, kPiece = 16 / (int)sizeof(E), kAhead = 8;
  typedef std::conditional_t<sizeof(E) == 2, uint16_t, uint32_t> Bits;
  const int lane = threadIdx.x & 31;
  for (int r0 = 0; r0 < 32 && r0 < rows; r0 += kAhead) {
    Bits v[kAhead][kPer];  // loads of several rows in flight
    auto at = [&](int q, int i) {
      const int c = lane + i * 32;
      return piece<ROW>(buf, row0 + r0 + q, c / kPiece) + (uint32_t)(c % kPiece * sizeof(E));
    };
#pragma unroll
    for (int q = 0; q < kAhead; ++q)
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        if (in) {
          v[q][i] = 0;
          if (r0 + q < rows && lane + i * 32 < left)
            v[q][i] = *reinterpret_cast<const Bits*>(g + (r0 + q) * stride + lane + i * 32);
        } else if constexpr (sizeof(E) == 2) {
          uint16_t w;
          asm volatile("ld.shared.u16 %0, [%1];" : "=h"(w) : "r"(at(q, i)) : "memory");
          v[q][i] = (Bits)w;
        } else {
          uint32_t w;
          asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(at(q, i)) : "memory");
          v[q][i] = (Bits)w;
        }
      }
#pragma unroll
    for (int q = 0; q < kAhead; ++q)
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        if (!in) {
          if (r0 + q < rows && lane + i * 32 < left)
            *reinterpret_cast<Bits*>(g + (r0 + q) * stride + lane + i * 32) = v[q][i];
        } else if constexpr (sizeof(E) == 2) {
          asm volatile("st.shared.u16 [%0], %1;" ::"r"(at(q, i)), "h"(v[q][i]) : "memory");
        } else {
          asm volatile("st.shared.u32 [%0], %1;" ::"r"(at(q, i)), "r"(v[q][i]) : "memory");
        }
      }
  }
}

// The stage that comes next and the parity of its round.
template <int STAGES>
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
    if (x == per * 64) {
      x = 0;
      ++head;
    }
  }
};

template <typename T, int CTA, int BNC, bool AMN, bool BMN, bool SPLIT>
__global__ void __launch_bounds__(THREADS, 1)
    product_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                   const __grid_constant__ CUtensorMap tm_y,
                   const __grid_constant__ CUtensorMap tm_res,
                   const __grid_constant__ CUtensorMap tm_z, const Params p) {
  typedef Shape<CTA, BNC> SH;
  constexpr int BN = SH::BN, STAGES = SH::STAGES, COLS = SH::COLS;
  constexpr uint32_t STAGE_BYTES = SH::STAGE_BYTES;
  extern __shared__ __align__(1024) unsigned char smem[];
  // the swizzle wants 1024-byte borders, where dynamic shared memory begins as long as there is no
  // static one; there is no room to move up
  const uint32_t base = smem_u32(smem);
  if (base & 1023u) {
    if (threadIdx.x == 0 && p.status != nullptr) atomicOr(p.status, VGGT_STATUS_TIMEOUT);
    return;
  }
  auto bar = [&](int i) { return base + SH::OFF_BAR + 8u * (uint32_t)i; };
  uint32_t* misc = reinterpret_cast<uint32_t*>(smem + SH::OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(misc + 1);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = CTA == 2 ? (int)cluster_rank() : 0;
  const uint32_t worker = blockIdx.x / CTA;

  if (tid == 0) {
    tc::prefetch_tmap(&tm_a);
    tc::prefetch_tmap(&tm_b);
    if (!SPLIT) tc::prefetch_tmap(&tm_y);
    for (int s = 0; s < STAGES; ++s) {
      tc::mbar_init(bar(SH::B_FULL + s), 1);
      tc::mbar_init(bar(SH::B_EMPTY + s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      tc::mbar_init(bar(SH::B_ACCFULL + b), 1);
      tc::mbar_init(bar(SH::B_ACCEMPTY + b), 4 * GROUPS * CTA);
    }
    for (int b = 0; b < GROUPS; ++b) tc::mbar_init(bar(SH::B_RES + b), 1);
    tc::mbar_init(bar(SH::B_DRAIN), 1);
    misc[1] = 0u;
    tc::mbar_fence_init();
  }
  if (warp == 2) {
    Pair<CTA>::alloc(base + SH::OFF_MISC, SH::TMEM_COLS);
    Pair<CTA>::relinquish();
  }
  tc::tc_fence_before();
  __syncthreads();
  if (CTA == 2) cluster_sync();
  tc::tc_fence_after();
  const uint32_t tmem = misc[0];
  // Up to here the kernel may run beside the end of the one before it in the stream, from here on
  // it has that one's results; the next one may begin its own preparations.
  grid_wait();

  if (warp == 0) {
    // ================= TMA producer =================
    const uint32_t full0 = CTA == 2 ? map_rank(bar(SH::B_FULL), 0) : bar(SH::B_FULL);
    Walk<SPLIT> w(p, worker);
    Ring<STAGES> ring;
    uint32_t issued = 0;
    bool ok = true;
    while (ok && w.next()) {
      const int m0 = (int)w.tm * (BM * CTA) + rank * BM;
      const int n0 = (int)w.tn * BN + rank * BNC;
      // where the operands' first blocks lie: no division is left in the loop
      Place a0, a1, b0, b1;
      if (AMN) {
        a0 = Place(m0 / 64, p.a_heads64);
        a1 = Place(m0 / 64 + 1, p.a_heads64);
      } else {
        a0 = Place(w.k0, p.a_heads64);
      }
      if (BMN) {
        b0 = Place(n0 / 64, p.b_heads64);
        if (BNC == 128) b1 = Place(n0 / 64 + 1, p.b_heads64);
      } else {
        b0 = Place(w.k0, p.b_heads64);
      }
      for (int k = w.k0; k < w.k1; ++k) {
        if (issued >= STAGES &&
            !wait_warp(bar(SH::B_EMPTY) + 8 * ring.at, ring.turn ^ 1, abort_flag, p.wait_ns)) {
          ok = false;
          break;
        }
        // the barrier is the first CTA's: it counts both CTAs' bytes
        const uint32_t full = full0 + 8 * ring.at;
        const uint32_t a = base + ring.at * STAGE_BYTES, b = a + A_BYTES;
        if (tc::elect_one()) {
          if (rank == 0) tc::mbar_expect_tx(bar(SH::B_FULL) + 8 * ring.at, CTA * STAGE_BYTES);
          if (AMN) {
            Pair<CTA>::load(a, &tm_a, full, a0.x, k * BK, a0.head);
            Pair<CTA>::load(a + A_BYTES / 2, &tm_a, full, a1.x, k * BK, a1.head);
          } else {
            Pair<CTA>::load(a, &tm_a, full, a0.x, m0, a0.head);
          }
          if (BMN) {
            Pair<CTA>::load(b, &tm_b, full, b0.x, k * BK, b0.head);
            if (BNC == 128) Pair<CTA>::load(b + A_BYTES / 2, &tm_b, full, b1.x, k * BK, b1.head);
          } else {
            Pair<CTA>::load(b, &tm_b, full, b0.x, n0, b0.head);
          }
        }
        __syncwarp();
        if (!AMN) a0.step(p.a_heads64);
        if (!BMN) b0.step(p.b_heads64);
        ring.step();
        ++issued;
      }
    }
    // The last copies have landed before the memory goes (the MMAs that read them are awaited by
    // their issuer).  A pair's second CTA, whose copies count on the first one's barriers, waits
    // instead for what the first one's MMAs announce here: the last blocks' release, which follows
    // their copies, and the end.  After a wait that gave up some of that never comes, and the
    // limit's time is far more than a copy on its way takes.  (Here, beside the last epilogue: at the
    // kernel's end the six waits made 0.4 us of a frame's 8.4.)
    if (lane == 0) {
      const uint32_t first = issued > STAGES ? issued - STAGES : 0;
      if (rank == 0) {
        for (uint32_t t = first; t < issued; ++t)
          tc::mbar_wait_drain(bar(SH::B_FULL + t % STAGES), (t / STAGES) & 1, p.wait_ns);
      } else {
        for (uint32_t t = first; t < issued; ++t)
          if (!tc::mbar_wait_drain(bar(SH::B_EMPTY + t % STAGES), (t / STAGES) & 1, p.wait_ns)) break;
        if (!p.wait_selftest) tc::mbar_wait_drain(bar(SH::B_DRAIN), 0, p.wait_ns);
      }
    }
  } else if (warp == 1) {
    // ================= MMA issuer (of the pair's first CTA) =================
    if (rank == 0) {
      const uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
      const uint32_t idesc =
          tc::idesc_f16(fmt, BMN ? 1u : 0u, BM * CTA, BN) | (AMN ? 1u << 15 : 0u);
      // a step of 16 reduced elements: 32 bytes along a K-major row, 16 MN-major rows
      constexpr uint64_t kStepA = AMN ? 16 * 128 / 16 : 2, kStepB = BMN ? 16 * 128 / 16 : 2;
      const uint64_t desc0 = tc::sw128_desc(base, A_BYTES / 2);
      bool ok = true;
      if (p.wait_selftest) ok = wait_warp(bar(SH::B_DRAIN), 0, abort_flag, p.wait_ns);
      Walk<SPLIT> w(p, worker);
      Ring<STAGES> ring;
      uint32_t i = 0;
      while (ok && w.next()) {
        const uint32_t b = i & 1;
        if (i >= 2 &&
            !wait_warp(bar(SH::B_ACCEMPTY + b), ((i >> 1) + 1) & 1, abort_flag, p.wait_ns)) {
          ok = false;
          break;
        }
        tc::tc_fence_after();
        const uint32_t acc = tmem + b * BN;
        for (int k = w.k0; k < w.k1; ++k) {
          if (!wait_warp(bar(SH::B_FULL) + 8 * ring.at, ring.turn, abort_flag, p.wait_ns)) {
            ok = false;
            break;
          }
          tc::tc_fence_after();
          const uint64_t ad = desc0 + ring.at * (STAGE_BYTES / 16), bd = ad + A_BYTES / 16;
          if (tc::elect_one()) {
#pragma unroll
            for (int kk = 0; kk < BK / 16; ++kk)
              Pair<CTA>::mma(acc, ad + kk * kStepA, bd + kk * kStepB, idesc,
                             (k > w.k0 || kk > 0) ? 1u : 0u);
            Pair<CTA>::commit(bar(SH::B_EMPTY) + 8 * ring.at);
            if (k + 1 == w.k1) Pair<CTA>::commit(bar(SH::B_ACCFULL + b));
          }
          __syncwarp();
          ring.step();
        }
        ++i;
      }
      if (!p.wait_selftest) {
        if (tc::elect_one()) Pair<CTA>::commit(bar(SH::B_DRAIN));
        __syncwarp();
        if (lane == 0) tc::mbar_wait_drain(bar(SH::B_DRAIN), 0, p.wait_ns);
      }
    }
  } else if (warp >= 4) {
    // ================= epilogue: group g takes COLS columns of a tile =================
    const int g = (warp - 4) >> 2, sub = warp & 3, row = sub * 32 + lane, t = tid & 127;
    float* vec = reinterpret_cast<float*>(smem + SH::OFF_VEC) + g * 128;  // bias | gate
    int* votes = reinterpret_cast<int*>(misc + 2) + g * 8;
    const uint32_t buf = base + SH::OFF_BUF + (uint32_t)g * BUF_BYTES, res_bar = bar(SH::B_RES + g);
    auto group_sync = [&] { asm volatile("bar.sync %0, 128;" ::"r"(1 + g) : "memory"); };
    uint32_t turns = 0;
    // true in all four warps or in none: the barriers of a group are not bounded, so that its
    // warps have to leave together
    auto agree = [&](bool ok) {
      const bool all = __all_sync(0xffffffffu, ok);
      volatile int* v = votes + 4 * (turns++ & 1);
      if (lane == 0) v[sub] = all ? 1 : 0;
      group_sync();
      return v[0] && v[1] && v[2] && v[3];
    };
    const bool has_res = !SPLIT && p.residual != nullptr, has_z = !SPLIT && p.z != nullptr;
    // a use of the buffer: COLS elements of T or 32 of fp32 in a row
    const bool y_wide = SPLIT || p.y_fp32;
    uint32_t i = 0, res_uses = 0;
    bool ok = true;
    Walk<SPLIT> w(p, worker);
    while (ok && w.next()) {
      const uint32_t b = i & 1;
      const int m0 = (int)w.tm * (BM * CTA) + rank * BM, col = (int)w.tn * BN + g * COLS;
      const bool active = g < BN / COLS && col < p.n;
      const int r0 = m0 + sub * 32;  // this warp's first row
      const int64_t rows = p.m - r0;
      // the buffer is free once its last store has read it; the residual comes into it
      auto open = [&](int c0, bool residual) {
        if (t == 0) {
          store_wait_read<0>();
          if (residual && p.res_tma) {
            constexpr uint32_t narrow = BM * COLS * 2;
            tc::mbar_expect_tx(res_bar, y_wide ? BUF_BYTES : narrow);
            tc::tma_load_3d(buf, &tm_res, res_bar, c0, m0, 0);
          }
        }
        __syncwarp();
      };
      if (active) {
        if (!SPLIT) {
          // seen by the group after the next barrier; the last readers are before the last one
          const int c = col + (t & 63);
          float v = t < 64 ? 0.f : 1.f;
          const void* src = t < 64 ? p.bias : p.gate;
          if (src != nullptr && (t & 63) < COLS && c < p.n)
            v = vector_at<T>(src, t >= 64 && p.gate_fp32, c);
          vec[t] = v;
        }
        open(col, has_res && !has_z);
      }
      // the first use's residual is there before the accumulator as a rule: one vote on both
      bool got = true;
      if (active && has_res && !has_z && p.res_tma)
        got = wait(res_bar, res_uses++ & 1, abort_flag, p.wait_ns);
      got = got && wait(bar(SH::B_ACCFULL + b), (i >> 1) & 1, abort_flag, p.wait_ns);
      if (!agree(got)) {
        ok = false;
        break;
      }
      tc::tc_fence_after();
      const uint32_t acc = tmem + b * BN + ((uint32_t)(sub * 32) << 16) + g * COLS;
      // of a weight's gradient: this row's gate, and its product with the weight's row
      float_pair row_gate = pack_pair(1.f, 1.f), dot = pack_pair(0.f, 0.f);
      if (AMN && !SPLIT && p.row_gate != nullptr && m0 + row < p.m) {
        const float v = vector_at<T>(p.row_gate, p.gate_fp32, m0 + row);
        row_gate = pack_pair(v, v);
      }
      bool opened = true;
      for (int which = has_z ? 0 : 1; active && ok && which < 2; ++which) {  // z, then y
        const bool wide = which == 1 ? y_wide : p.z_fp32, res = which == 1 && has_res;
        for (int c = 0; c < COLS; c += wide ? 32 : COLS) {
          const int c0 = col + c;  // first column of the use
          if (!SPLIT && c0 >= p.n) break;
          const int64_t left = p.n - c0;
          if (!opened) {
            open(c0, res);
            const bool fine = !(res && p.res_tma) ||
                              wait(res_bar, res_uses++ & 1, abort_flag, p.wait_ns);
            if (!agree(fine)) {
              ok = false;
              break;
            }
          }
          opened = false;
          if (res && !p.res_tma) {
            const int64_t at = (int64_t)r0 * p.residual_stride + c0;
            if (wide)
              copy_rows<128>(buf, sub * 32,
                             const_cast<float*>(static_cast<const float*>(p.residual)) + at,
                             p.residual_stride, rows, left, true);
            else
              copy_rows<COLS * 2>(buf, sub * 32,
                                  const_cast<T*>(static_cast<const T*>(p.residual)) + at,
                                  p.residual_stride, rows, left, true);
            __syncwarp();
          }
          // 32 columns at a time: TMEM -> registers -> buffer
          for (int h = c; h < (wide ? c + 32 : COLS); h += 32) {
            uint32_t r[32];
            tc::tmem_ld32(acc + h, r);
            tc::tmem_wait_ld();
            if (SPLIT) {
#pragma unroll
              for (int j = 0; j < 8; ++j)
                sts128(piece<128>(buf, row, j), r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
              continue;
            }
            const ulonglong2* bv = reinterpret_cast<const ulonglong2*>(vec + h);
            float_pair v[16];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const ulonglong2 q = bv[j];
              v[2 * j] = add_pair(
                  pack_pair(__uint_as_float(r[4 * j]), __uint_as_float(r[4 * j + 1])), q.x);
              v[2 * j + 1] = add_pair(
                  pack_pair(__uint_as_float(r[4 * j + 2]), __uint_as_float(r[4 * j + 3])), q.y);
            }
            if (which == 1) {
              if (p.act != VGGT_ACT_NONE)
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
                const uint32_t a = piece<128>(buf, row, j);
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
                const uint32_t a = piece<COLS * 2>(buf, row, h / 8 + j);
                uint32_t q[4];
                if (res) {
                  lds128(a, q);
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    const float2 f = ElemOps<T>::to_float2(q[e]);
                    if (AMN && p.row_dot != nullptr)
                      dot = fma_pair(v[4 * j + e], pack_pair(f.x, f.y), dot);
                    else
                      v[4 * j + e] = add_pair(v[4 * j + e], pack_pair(f.x, f.y));
                  }
                }
                if (AMN)
#pragma unroll
                  for (int e = 0; e < 4; ++e) v[4 * j + e] = mul_pair(v[4 * j + e], row_gate);
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
          if (AMN && !SPLIT && p.row_dot != nullptr && m0 + row < p.m) {
            float d0, d1;
            unpack_pair(d0, d1, dot);
            p.row_dot[(int64_t)(col / COLS) * p.m + m0 + row] = d0 + d1;
          }
          if (AMN && !SPLIT && p.y == nullptr) {  // the rows' products alone are wanted
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            group_sync();
          } else if (SPLIT || (which == 0 ? p.z_tma : p.y_tma)) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            group_sync();
            if (t == 0) {
              if (SPLIT) {
                const int64_t slot = (int64_t)worker + w.tile;
                store_bulk(reinterpret_cast<unsigned char*>(p.slots) +
                               ((slot * CTA + rank) * (BN / 32) + (g * COLS + c) / 32) * BUF_BYTES,
                           buf, BUF_BYTES);
              } else if (m0 < p.m) {
                if (which == 0) {
                  store_3d(&tm_z, buf, c0, m0, 0);
                } else {
                  const int head = c0 / 64 / p.y_heads64;
                  store_3d(&tm_y, buf, c0 - head * p.y_heads64 * 64, m0, head);
                }
              }
              store_commit();
            }
          } else {
            __syncwarp();
            void* const to = which == 0 ? p.z : p.y;
            const int64_t stride = which == 0 ? p.z_stride : p.y_stride;
            if (wide) {
              copy_rows<128>(buf, sub * 32, static_cast<float*>(to) + (int64_t)r0 * stride + c0,
                             stride, rows, left, false);
            } else if (which == 0) {
              copy_rows<COLS * 2>(buf, sub * 32, static_cast<T*>(to) + (int64_t)r0 * stride + c0,
                                  stride, rows, left, false);
            } else {
              const int head = c0 / 64 / p.y_heads64;
              copy_rows<COLS * 2>(buf, sub * 32,
                                  static_cast<T*>(p.y) + head * p.y_head_stride +
                                      (int64_t)r0 * p.y_stride + (c0 - head * p.y_heads64 * 64),
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
          arrive_cluster(map_rank(bar(SH::B_ACCEMPTY + b), 0));
        else
          tc::mbar_arrive(bar(SH::B_ACCEMPTY + b));
      }
      ++i;
    }
    // after a wait that gave up: a residual on its way lands before the block ends
    if (!ok && res_uses > 0) tc::mbar_wait_drain(res_bar, (res_uses - 1) & 1, p.wait_ns);
    if (t == 0) store_wait_read<0>();  // the memory outlives the stores' reads of it
  }

  tc::tc_fence_before();
  __syncthreads();
  __syncwarp();
  if (CTA == 2) cluster_sync();
  tc::tc_fence_after();
  if (tid == 0 && *abort_flag && p.status != nullptr) atomicOr(p.status, VGGT_STATUS_TIMEOUT);
  if (warp == 2) Pair<CTA>::dealloc(tmem, SH::TMEM_COLS);
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
    if (e.z != nullptr && e.z_type == VGGT_DTYPE_FP32)
      put8(static_cast<float*>(e.z) + r * e.z_stride + c, k, wide, v);
    else if (e.z != nullptr)
      put8(static_cast<T*>(e.z) + r * e.z_stride + c, k, wide, v);
    act::dispatch(e.act, [&](auto kind) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = act::value<decltype(kind)::value>(v[j]);
    });
    if (e.gate != nullptr) {
      vector_get8<T>(e.gate, e.gate_fp32, c, k, wide, t);
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
  return split ? (size_t)(workers + tiles_m * tiles_n) * cta * BM * (bnc * cta) * 4 : 0;
}

static int sm_count() {
  int sms = 0;
  return device_sms(&sms) == cudaSuccess && sms > 0 ? sms : 148;
}

// The way a product is cut is the one of the least estimated time, in SM cycles: what a launch and a
// reduction block take, measured alone and (block: + busy) with all SMs at work, and for a split one
// the partial sums' way through memory and another launch.  Splitting evens the load out where
// tiles are few or the last round is short.
Plan plan_product(int64_t m, int64_t n, int64_t red) {
  // cta, bnc, a launch, a block, a block's share that grows with the load
  static const int kShapes[][5] = {
      {1, 64, 6500, 420, 40}, {1, 128, 7700, 450, 60}, {2, 64, 8200, 320, 60}, {2, 128, 10500, 530, 80}};
  const int sms = sm_count();
  Plan best;
  double least = 0;
  for (const int* shape : kShapes)
    for (int split = 0; split < 2; ++split) {
      Plan p;
      p.cta = shape[0];
      p.bnc = shape[1];
      p.split = split;
      p.tiles_m = (m + BM * p.cta - 1) / (BM * p.cta);
      p.tiles_n = (n + p.bnc * p.cta - 1) / (p.bnc * p.cta);
      p.blocks = (red + BK - 1) / BK;
      p.workers = (int)std::min<int64_t>(sms / p.cta, p.units());
      const int64_t rounds = (p.units() + p.workers - 1) / p.workers;
      const double busy = (double)p.workers * p.cta / sms;
      double t = shape[2] + (double)rounds * (split ? 1 : p.blocks) * (shape[3] + shape[4] * busy);
      if (split) t += 7000 + (double)p.slot_bytes() * 2 / 2500;
      // workers that begin in different places of long operands do not meet in L2 (44,000 rows'
      // weight gradient 254 us whole, 351 split)
      if (split && (double)(m + n) * red * 2 > 60e6)
        t = std::max(t, (double)p.tiles_m * p.tiles_n * red * 2 * (BM + p.bnc) * p.cta / 3500);
      if (least == 0 || t < least) {
        least = t;
        best = p;
      }
    }
  return best;
}

int64_t dot_groups(const Plan& plan, int64_t n) {
  const int cols = std::max(plan.bnc * plan.cta / GROUPS, 32);
  return (n + cols - 1) / cols;
}

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

static bool operand_map(CUtensorMap* map, const Operand& o, int dtype, int64_t rows, int box_rows) {
  const uint64_t dims[3] = {(uint64_t)o.dim, (uint64_t)rows, (uint64_t)o.heads};
  // a stride that is never used may be anything: give a valid one
  const int64_t row = rows > 1 ? o.stride : (o.dim + 7) / 8 * 8;
  const uint64_t strides[2] = {(uint64_t)row * 2,
                               (uint64_t)(o.heads > 1 ? o.head_stride : row * rows) * 2};
  const uint32_t box[3] = {64, o.mn_major ? (uint32_t)BK : (uint32_t)box_rows, 1};
  return encode_tmap_sw128(map, o.p, dtype, 3, dims, strides, box);
}

// Rows of an output or of the residual, for copies of 128 rows of `cols` elements; false where TMA
// cannot address them.
static bool rows_map(CUtensorMap* map, const void* p, int type, int64_t stride, int64_t head_stride,
                     int64_t heads, int64_t dim, int64_t rows, int cols) {
  const int per = type == VGGT_DTYPE_FP32 ? 4 : 8, size = 16 / per;
  if (!aligned16(p) || dim % per || (rows > 1 && (stride % per || stride < dim)) ||
      (heads > 1 && (head_stride % per || head_stride < dim)))
    return false;
  const int64_t row = rows > 1 ? stride : dim;
  const uint64_t dims[3] = {(uint64_t)dim, (uint64_t)rows, (uint64_t)heads};
  const uint64_t strides[2] = {(uint64_t)row * size,
                               (uint64_t)(heads > 1 ? head_stride : row * rows) * size};
  const uint32_t box[3] = {(uint32_t)cols, (uint32_t)BM, 1};
  return encode_tmap(map, p, type, 3, dims, strides, box, cols * size);
}

template <typename T, int CTA, int BNC, bool AMN, bool BMN, bool SPLIT>
static cudaError_t launch_kernel(const CUtensorMap* maps, const Params& p, cudaStream_t stream) {
  auto k = product_kernel<T, CTA, BNC, AMN, BMN, SPLIT>;
  constexpr int smem = (int)Shape<CTA, BNC>::SMEM_BYTES;
  static OncePerDevice allowed;
  cudaError_t e = allow_shared(k, smem, &allowed);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(p.workers * CTA));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CTA;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CTA == 2 ? 2 : 1;
  e = cudaLaunchKernelEx(&cfg, k, maps[0], maps[1], maps[2], maps[3], maps[4], p);
  return e != cudaSuccess ? e : cudaGetLastError();
}

template <typename T, int CTA, int BNC>
static cudaError_t launch_majors(bool amn, bool bmn, bool split, const CUtensorMap* maps,
                                 const Params& p, cudaStream_t stream) {
  if (!amn && !bmn)
    return split ? launch_kernel<T, CTA, BNC, false, false, true>(maps, p, stream)
                 : launch_kernel<T, CTA, BNC, false, false, false>(maps, p, stream);
  if (!amn)
    return split ? launch_kernel<T, CTA, BNC, false, true, true>(maps, p, stream)
                 : launch_kernel<T, CTA, BNC, false, true, false>(maps, p, stream);
  if (!bmn) return cudaErrorInvalidValue;  // no product has these
  return split ? launch_kernel<T, CTA, BNC, true, true, true>(maps, p, stream)
               : launch_kernel<T, CTA, BNC, true, true, false>(maps, p, stream);
}

template <typename T>
static cudaError_t launch_shapes(const Plan& plan, bool amn, bool bmn, const CUtensorMap* maps,
                                 const Params& p, cudaStream_t stream) {
  const bool s = plan.split;
  if (plan.cta == 2)
    return plan.bnc == 128 ? launch_majors<T, 2, 128>(amn, bmn, s, maps, p, stream)
                           : launch_majors<T, 2, 64>(amn, bmn, s, maps, p, stream);
  return plan.bnc == 128 ? launch_majors<T, 1, 128>(amn, bmn, s, maps, p, stream)
                         : launch_majors<T, 1, 64>(amn, bmn, s, maps, p, stream);
}

cudaError_t launch_product(const Plan& plan, int dtype, int64_t m, int64_t n, int64_t red,
                           const Operand& a, const Operand& b, const Epilogue& e, float* slots,
                           int32_t* status, cudaStream_t stream) {
  CUtensorMap maps[5] = {};
  if (!operand_map(&maps[0], a, dtype, a.mn_major ? red : m, BM) ||
      !operand_map(&maps[1], b, dtype, b.mn_major ? red : n, plan.bnc))
    return cudaErrorInvalidValue;
  Params p{};
  p.m = m;
  p.n = n;
  p.tiles = (uint32_t)(plan.tiles_m * plan.tiles_n);
  p.tiles_n = (uint32_t)plan.tiles_n;
  p.blocks = (uint32_t)plan.blocks;
  p.workers = (uint32_t)plan.workers;
  p.per = (uint32_t)(plan.units() / plan.workers);
  p.rest = (uint32_t)(plan.units() % plan.workers);
  auto heads64 = [](int64_t heads, int64_t dim) { return heads > 1 ? (int)(dim / 64) : INT_MAX / 64; };
  p.a_heads64 = heads64(a.heads, a.dim);
  p.b_heads64 = heads64(b.heads, b.dim);
  p.y_heads64 = heads64(e.y_heads, e.y_dim);
  p.bias = e.bias;
  p.gate = e.gate;
  p.gate_fp32 = e.gate_fp32;
  p.act = e.act;
  p.y_fp32 = e.y_type == VGGT_DTYPE_FP32;
  p.residual = e.residual;
  p.residual_stride = e.residual_stride;
  p.y = e.y;
  p.y_stride = e.y_stride;
  p.y_head_stride = e.y_head_stride;
  p.z = e.z;
  p.z_stride = e.z_stride;
  p.z_fp32 = e.z_type == VGGT_DTYPE_FP32;
  if (!plan.split) {
    // columns of a buffer's row, as the kernel's Shape has them
    const int cols = std::max(plan.bnc * plan.cta / GROUPS, 32), y_cols = p.y_fp32 ? 32 : cols;
    p.y_tma = e.y && rows_map(&maps[2], e.y, e.y_type, e.y_stride, e.y_head_stride, e.y_heads, e.y_dim, m,
                       y_cols);
    p.res_tma = e.residual && rows_map(&maps[3], e.residual, e.y_type, e.residual_stride, 0, 1, n, m,
                                       y_cols);
    p.z_tma = e.z && rows_map(&maps[4], e.z, e.z_type, e.z_stride, 0, 1, n, m,
                              p.z_fp32 ? 32 : cols);
  }
  p.row_gate = e.row_gate;
  p.row_dot = e.row_dot;
  p.slots = slots;
  p.status = status;
  p.wait_ns = api_wait_ns();
  p.wait_selftest = api_wait_selftest();
  return dtype == VGGT_DTYPE_BF16
             ? launch_shapes<__nv_bfloat16>(plan, a.mn_major, b.mn_major, maps, p, stream)
             : launch_shapes<__half>(plan, a.mn_major, b.mn_major, maps, p, stream);
}

Slots slots_of(const Plan& plan, const float* p) {
  return {p, (uint32_t)plan.tiles_n, (uint32_t)plan.blocks, (uint32_t)(plan.units() / plan.workers),
          (uint32_t)(plan.units() % plan.workers), plan.cta, plan.bnc * plan.cta};
}

cudaError_t finish_product(const Plan& plan, int dtype, int64_t m, int64_t n, const Epilogue& e,
                           const float* slots, cudaStream_t stream) {
  const int64_t all = m * ((n + 7) / 8);
  const unsigned grid = (unsigned)std::min<int64_t>((all + 255) / 256, 148 * 16);
  const bool wide = wide_rows(e.y, e.y_stride, e.y_type) && e.y_dim % 8 == 0 &&
                    (e.y_heads <= 1 || e.y_head_stride % 8 == 0) &&
                    wide_rows(e.z, e.z_stride, e.z_type) && wide_rows(e.bias, 8, dtype) &&
                    wide_rows(e.gate, 8, dtype) &&
                    wide_rows(e.residual, e.residual_stride, e.y_type);
  const Slots s = slots_of(plan, slots);
  if (dtype == VGGT_DTYPE_BF16)
    finish_kernel<__nv_bfloat16><<<grid, 256, 0, stream>>>(s, m, n, e, wide);
  else
    finish_kernel<__half><<<grid, 256, 0, stream>>>(s, m, n, e, wide);
  return cudaGetLastError();
}

// ---- operands that TMA cannot address ----------------------------------------------------------
struct Copy {
  const uint16_t* from;
  uint16_t* to;
  int64_t rows, width, pad, stride, head_stride, dim;
};

__global__ void __launch_bounds__(256) copy_operand_kernel(const Copy c) {
  const int64_t r = blockIdx.x;
  for (int k = threadIdx.x; k < (int)c.pad; k += 256) {
    const int head = k / (int)c.dim;
    c.to[r * c.pad + k] =
        k < c.width ? c.from[head * c.head_stride + r * c.stride + (k - head * (int)c.dim)] : 0;
  }
}

Laid plan_operands(const vggt_linear_args* a, bool need_x, bool need_w) {
  Laid l{};
  const int64_t heads = a->heads > 1 ? a->heads : 1, dim = a->inner / heads;
  auto rows_fit = [](const void* p, int64_t rows, int64_t stride, int64_t width) {
    return aligned16(p) && (rows <= 1 || (stride % 8 == 0 && stride >= width));
  };
  l.copy_x = need_x && !(rows_fit(a->x, a->rows, a->x_stride, dim) &&
                         (heads == 1 || (dim % 64 == 0 && a->x_head_stride % 8 == 0 &&
                                         a->x_head_stride >= dim)));
  l.copy_w = need_w && !rows_fit(a->weight, a->outer, a->weight_stride, a->inner);
  l.pad = (a->inner + 7) / 8 * 8;
  auto take = [&](bool need, int64_t rows) {
    const size_t at = l.bytes;
    if (need) l.bytes += ((size_t)rows * l.pad * 2 + 255) / 256 * 256;
    return at;
  };
  l.x_at = take(l.copy_x, a->rows);
  l.w_at = take(l.copy_w, a->outer);
  return l;
}

cudaError_t copy_operands(const vggt_linear_args* a, const Laid& l, unsigned char* ws,
                          cudaStream_t stream) {
  const int64_t heads = a->heads > 1 ? a->heads : 1;
  for (int which = 0; which < 2; ++which) {
    if (!(which == 0 ? l.copy_x : l.copy_w)) continue;
    Copy c;
    c.from = static_cast<const uint16_t*>(which == 0 ? a->x : a->weight);
    c.to = reinterpret_cast<uint16_t*>(ws + (which == 0 ? l.x_at : l.w_at));
    c.rows = which == 0 ? a->rows : a->outer;
    c.width = a->inner;
    c.pad = l.pad;
    c.stride = which == 0 ? a->x_stride : a->weight_stride;
    c.head_stride = a->x_head_stride;
    c.dim = which == 0 ? a->inner / heads : l.pad;
    if (c.dim == a->inner) c.dim = l.pad;  // one head
    copy_operand_kernel<<<(unsigned)c.rows, 256, 0, stream>>>(c);
    if (cudaError_t e = cudaGetLastError()) return e;
  }
  return cudaSuccess;
}

Operand matrix(const void* p, int64_t width, int64_t stride, bool mn_major) {
  Operand o;
  o.p = p;
  o.stride = stride;
  o.dim = width;
  o.mn_major = mn_major;
  return o;
}

Operand x_operand(const vggt_linear_args* a, const Laid& l, const unsigned char* ws, bool mn_major) {
  if (l.copy_x) return matrix(ws + l.x_at, a->inner, l.pad, mn_major);
  Operand o = matrix(a->x, a->inner, a->x_stride, mn_major);
  if (a->heads > 1) {
    o.heads = a->heads;
    o.head_stride = a->x_head_stride;
    o.dim = a->inner / a->heads;
  }
  return o;
}

Operand w_operand(const vggt_linear_args* a, const Laid& l, const unsigned char* ws, bool mn_major) {
  return l.copy_w ? matrix(ws + l.w_at, a->inner, l.pad, mn_major)
                  : matrix(a->weight, a->inner, a->weight_stride, mn_major);
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
  if (a->activation != VGGT_ACT_NONE && a->z_dtype != a->dtype && a->z_dtype != VGGT_DTYPE_FP32)
    return api_fail("z is of x's type or FP32");
  if (a->rows < 0 || a->inner < 1 || a->outer < 1) return api_fail("bad size argument");
  if (a->rows > INT_MAX - 512 || a->inner > INT_MAX - 512 || a->outer > INT_MAX - 512)
    return api_fail("too many rows or too wide");
  if (a->heads > 1 && a->inner % a->heads)
    return api_fail("inner (%lld) must be a multiple of heads (%lld)", (long long)a->inner,
                    (long long)a->heads);
  if (a->activation < VGGT_ACT_NONE || a->activation > VGGT_ACT_RELU)
    return api_fail("unknown activation %d", a->activation);
  if (a->rows == 0) return 0;
  if (!a->x || !a->weight) return api_fail("x and weight must be non-NULL");
  if ((a->rows > 1 && a->x_stride < 0) || (a->heads > 1 && a->x_head_stride < 0) ||
      (a->outer > 1 && a->weight_stride < 0))
    return api_fail("negative stride");
  if ((a->rows + 127) / 128 * ((a->outer + 63) / 64) * ((a->inner + 63) / 64) > INT_MAX ||
      (a->outer + 127) / 128 * ((a->inner + 63) / 64) * ((a->rows + 63) / 64) > INT_MAX)
    return api_fail("the product is too large");
  if (a->residual && a->rows > 1 && a->residual_stride < 0) return api_fail("negative stride");
  return 0;
}

}  // namespace lin
}  // namespace vggt

extern "C" size_t vggt_linear_workspace_size(const vggt_linear_args* a) {
  using namespace vggt::lin;
  if (!a || a->rows <= 0 || a->inner < 1 || a->outer < 1) return 0;
  const size_t copies = plan_operands(a, true, true).bytes;
  if (few_rows(a->rows, a->outer, a->inner)) return copies;
  return copies + plan_product(a->rows, a->outer, a->inner).slot_bytes();
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
  const Laid laid = plan_operands(a, true, true);
  const bool few = few_rows(a->rows, a->outer, a->inner);
  const Plan plan = few ? Plan{} : plan_product(a->rows, a->outer, a->inner);
  const size_t bytes = laid.bytes + plan.slot_bytes();
  if (bytes > 0 && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255u) ||
                    workspace_bytes < bytes))
    return api_fail("the workspace is too small or not 256-byte aligned");
  Epilogue e;
  e.bias = a->bias;
  e.gate = a->gate;
  e.gate_fp32 = a->gate_fp32 != 0;
  e.act = a->activation;
  e.residual = a->residual;
  e.residual_stride = a->residual_stride;
  e.y = y;
  e.y_stride = y_stride;
  e.y_dim = a->outer;
  e.y_type = a->stream_dtype;
  e.z = z;
  e.z_stride = z_stride;
  e.z_type = a->z_dtype;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  float* slots = reinterpret_cast<float*>(ws + laid.bytes);
  cudaError_t rc = copy_operands(a, laid, ws, st);
  if (rc == cudaSuccess && few)
    return api_cuda(launch_rows(a->dtype, a->rows, a->outer, a->inner, x_operand(a, laid, ws, false),
                                w_operand(a, laid, ws, false), e, st));
  if (rc == cudaSuccess)
    rc = launch_product(plan, a->dtype, a->rows, a->outer, a->inner, x_operand(a, laid, ws, false),
                        w_operand(a, laid, ws, false), e, slots, status, st);
  if (rc == cudaSuccess && plan.split)
    rc = finish_product(plan, a->dtype, a->rows, a->outer, e, slots, st);
  return api_cuda(rc);
}
