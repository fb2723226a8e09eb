// What the forward and the backward kernels of the gated residual with its norms share.
//
//   p = post(branch)             post: none, or a norm with post_weight, post_bias
//   h = x + gate * p             gate: per channel, or per channel and run of rows
//   y = norm(h) * weight + bias  norm: (h - mean) / sqrt(var + eps), or h / sqrt(mean h^2 + eps)
//
// A row is held in registers by WPR warps, 8 * J elements a lane, in chunks of 8: chunk j of lane
// l of the row's warp w starts at column 8 * ((j * WPR + w) * 32 + l).  A block has 16 warps or a
// few more, one block to an SM, and each of its groups of WPR warps (a slot) works through rows of its own.
// While it works on one row, its threads copy their chunks of the next one into shared memory
// (cp.async, where the layout allows 16-byte accesses: `vec`), and the parameters lie there too, in
// fp32, read once per block: what a thread needs of either is its own or its warp's, so that no
// barrier is needed.  (Read from global memory where they are used, the parameters' latencies took
// a third of the time: 32 frames of width 1024, fp32 stream, 159 us.)  Few rows, unaligned ones and
// the widest are read straight into registers, the parameters once for all rows (DIRECT).  All
// arithmetic is in fp32, in packed pairs; means are formed first and variances from what is left
// after them, so that a row far from zero loses nothing.
#pragma once

#include <type_traits>

#include "exp2.cuh"
#include "vec8.cuh"

namespace vggt {
namespace rnorm {

constexpr int kMaxThreads = 512;  // of a block
constexpr int kNormLayer = VGGT_NORM_LAYER, kNormRms = VGGT_NORM_RMS;

// A vector of parameters in any of the three element types, or none.
struct Param {
  const void* p = nullptr;
  int type = VGGT_DTYPE_FP32;
};

__device__ __forceinline__ float_pair both(float a) { return pack_pair(a, a); }
__device__ __forceinline__ float sum_pair(float_pair v) {
  float a, b;
  unpack_pair(a, b, v);
  return a + b;
}

// Eight elements as pairs, of which the first `n` exist (the rest are zero).
template <typename E>
__device__ __forceinline__ void get_pairs(const E* p, int n, bool vec, float_pair* v) {
  float f[8];
  get8(p, n, vec, f);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = pack_pair(f[2 * i], f[2 * i + 1]);
}
// VEC: 16-byte accesses, with n 0 or 8.
template <bool VEC, typename E>
__device__ __forceinline__ void put_pairs(E* p, int n, bool vec, const float_pair* v) {
  float f[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) unpack_pair(f[2 * i], f[2 * i + 1], v[i]);
  if (!VEC)
    put8(p, n, vec, f);
  else if (n > 0)
    Elem<E>::store8(p, f);
}
__device__ __forceinline__ void get_param(const Param& q, int64_t at, int n, bool vec,
                                          float_pair* v) {
  if (q.type == VGGT_DTYPE_FP32)
    get_pairs(static_cast<const float*>(q.p) + at, n, vec, v);
  else if (q.type == VGGT_DTYPE_BF16)
    get_pairs(static_cast<const __nv_bfloat16*>(q.p) + at, n, vec, v);
  else
    get_pairs(static_cast<const __half*>(q.p) + at, n, vec, v);
}

// A call's tensors (vggt_block.h).
struct Args {
  const void* x;
  const void* branch;
  Param gate, weight, bias, post_weight, post_bias;
  int64_t rows, width, x_stride, branch_stride, rows_per_gate;
  int stream_type, type;  // of x and h, and of branch and y
  int norm, post;         // VGGT_NORM_*
  float eps;
  bool vec;
};

constexpr int kStages = 2;
constexpr uint32_t kSharedBytes = 224 * 1024;

enum { kWeight, kBias, kGate, kPostWeight, kPostBias, kArrays };

// Shared memory of a block: rows to come (UNITS 16-byte units a thread and stage) and parameters,
// all slots' the same but for a gate of several, which each slot has for itself.  Parameters that do
// not fit are read where they are used; rows that do not are DIRECT.
template <int TH, int WPR, int J, int UNITS, bool DIRECT>
struct Shared {
  static constexpr int kThreads = TH;
  static constexpr uint32_t kRowBytes = TH * kStages * UNITS * 16;
  static constexpr uint32_t kParamBytes = WPR * 32 * J * 32, kOwnBytes = TH * J * 32;
  static constexpr bool kFits = kRowBytes <= kSharedBytes;
  static constexpr bool kParams = !DIRECT && kRowBytes + kArrays * kParamBytes <= kSharedBytes;
  // room for a gate of each slot's own
  static constexpr bool kOwnGate =
      kParams && kRowBytes + 4 * kParamBytes + kOwnBytes <= kSharedBytes;
  static constexpr uint32_t kAfterRows = DIRECT ? 0 : kRowBytes;
  static constexpr uint32_t kBytes =
      kAfterRows + (kParams ? 4 * kParamBytes + (kOwnGate ? kOwnBytes : kParamBytes) : 0);
};

// Eight elements as they lie in memory, converted later: loads of several tensors are in flight at
// once only if nothing is done with the first before the last is issued.
struct Raw8 {
  uint4 a, b;
  bool fp32, bf16;
  // of 16-byte aligned memory, n 0 or 8
  __device__ __forceinline__ void load(const void* base, int type, int64_t at, int n) {
    fp32 = type == VGGT_DTYPE_FP32;
    bf16 = type == VGGT_DTYPE_BF16;
    const unsigned char* p = static_cast<const unsigned char*>(base) + at * (fp32 ? 4 : 2);
    a = b = make_uint4(0, 0, 0, 0);
    if (n > 0) {
      a = *reinterpret_cast<const uint4*>(p);
      if (fp32) b = *reinterpret_cast<const uint4*>(p + 16);
    }
  }
  __device__ __forceinline__ void convert(float_pair* v) const {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w}, u[4] = {b.x, b.y, b.z, b.w};
    if (fp32) {
      v[0] = pack_pair(__uint_as_float(w[0]), __uint_as_float(w[1]));
      v[1] = pack_pair(__uint_as_float(w[2]), __uint_as_float(w[3]));
      v[2] = pack_pair(__uint_as_float(u[0]), __uint_as_float(u[1]));
      v[3] = pack_pair(__uint_as_float(u[2]), __uint_as_float(u[3]));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f =
            bf16 ? ElemOps<__nv_bfloat16>::to_float2(w[i]) : ElemOps<__half>::to_float2(w[i]);
        v[i] = pack_pair(f.x, f.y);
      }
    }
  }
};

template <typename E>
struct TypeOf {
  static constexpr int value = std::is_same<E, float>::value           ? VGGT_DTYPE_FP32
                               : std::is_same<E, __nv_bfloat16>::value ? VGGT_DTYPE_BF16
                                                                       : VGGT_DTYPE_FP16;
};

// The parameters as one thread sees them.
template <int WPR, int J, typename SH, bool DIRECT>
struct Params {
  const Args& a;
  unsigned char* at;  // this thread's place among the parameters
  int first;
  const int* n;
  int64_t gate_row = 0;
  float_pair reg[DIRECT ? kArrays : 1][DIRECT ? J : 1][4];

  static constexpr int kStep = 8 * WPR * 32;
  __device__ __forceinline__ const Param& param(int k) const {
    return k == kWeight  ? a.weight
           : k == kBias  ? a.bias
           : k == kGate  ? a.gate
           : k == kPostWeight ? a.post_weight : a.post_bias;
  }
  // whether parameter k lies in shared memory
  __device__ __forceinline__ bool held(int k) const {
    return SH::kParams && (k != kGate || SH::kOwnGate || a.rows_per_gate == 0);
  }
  // place of chunk j's half u of parameter k
  __device__ __forceinline__ unsigned char* place(int k, int j, int u) const {
    if (k == kGate && SH::kOwnGate)
      return at + 4 * SH::kParamBytes + ((j * 2 + u) * SH::kThreads + threadIdx.x) * 16;
    const int slot = k < kGate ? k : k == kGate ? 4 : k - 1;
    return at + slot * SH::kParamBytes +
           ((j * 2 + u) * (WPR * 32) + (int)threadIdx.x % (WPR * 32)) * 16;
  }
  __device__ __forceinline__ void fill(int k) {
#pragma unroll
    for (int j = 0; j < J; ++j) {
      float_pair v[4];
      get_param(param(k), (k == kGate ? gate_row * a.width : 0) + first + j * kStep, n[j], a.vec, v);
      *reinterpret_cast<ulonglong2*>(place(k, j, 0)) = make_ulonglong2(v[0], v[1]);
      *reinterpret_cast<ulonglong2*>(place(k, j, 1)) = make_ulonglong2(v[2], v[3]);
    }
  }
  // DIRECT: reads all that the call uses; else fills the shared places (a barrier has to follow)
  __device__ __forceinline__ Params(const Args& args, unsigned char* smem, int first_, const int* n_,
                                    int64_t gate_row_)
      : a(args), at(smem), first(first_), n(n_), gate_row(gate_row_) {
    if (DIRECT && a.vec) {
      Raw8 raw[kArrays][J];
#pragma unroll
      for (int k = 0; k < kArrays; ++k)
        if (param(k).p != nullptr)
#pragma unroll
          for (int j = 0; j < J; ++j)
            raw[k][j].load(param(k).p, param(k).type,
                           (k == kGate ? gate_row * a.width : 0) + first + j * kStep, n[j]);
#pragma unroll
      for (int k = 0; k < kArrays; ++k)
        if (param(k).p != nullptr)
#pragma unroll
          for (int j = 0; j < J; ++j) raw[k][j].convert(reg[DIRECT ? k : 0][DIRECT ? j : 0]);
    } else if (DIRECT) {
#pragma unroll
      for (int k = 0; k < kArrays; ++k)
        if (param(k).p != nullptr)
#pragma unroll
          for (int j = 0; j < J; ++j)
            get_param(param(k), (k == kGate ? gate_row * a.width : 0) + first + j * kStep, n[j],
                      false, reg[DIRECT ? k : 0][DIRECT ? j : 0]);
    } else if (SH::kParams) {
#pragma unroll
      for (int k = 0; k < kArrays; ++k)
        if (param(k).p != nullptr && held(k) &&
            ((k == kGate && SH::kOwnGate) || threadIdx.x < WPR * 32))
          fill(k);
    }
  }
  // the gate of another run of rows
  __device__ __forceinline__ void turn_to(int64_t row) {
    if (row == gate_row) return;
    gate_row = row;
    if (DIRECT) {
#pragma unroll
      for (int j = 0; j < J; ++j)
        get_param(a.gate, row * a.width + first + j * kStep, n[j], a.vec,
                  reg[DIRECT ? kGate : 0][DIRECT ? j : 0]);
    } else if (SH::kOwnGate) {
      fill(kGate);
    }
  }
  __device__ __forceinline__ void get(int k, int j, float_pair* v) const {
    if (DIRECT) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = reg[DIRECT ? k : 0][DIRECT ? j : 0][i];
    } else if (held(k)) {
      const ulonglong2 lo = *reinterpret_cast<const ulonglong2*>(place(k, j, 0));
      const ulonglong2 hi = *reinterpret_cast<const ulonglong2*>(place(k, j, 1));
      v[0] = lo.x, v[1] = lo.y, v[2] = hi.x, v[3] = hi.y;
    } else {
      get_param(param(k), (k == kGate ? gate_row * a.width : 0) + first + j * kStep, n[j], a.vec, v);
    }
  }
  __device__ __forceinline__ void scale(int k, int j, float_pair* v) const {
    if (param(k).p == nullptr) return;
    float_pair w[4];
    get(k, j, w);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = mul_pair(v[i], w[i]);
  }
  __device__ __forceinline__ void shift(int k, int j, float_pair* v) const {
    if (param(k).p == nullptr) return;
    float_pair w[4];
    get(k, j, w);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = add_pair(v[i], w[i]);
  }
  // h += gate * p
  __device__ __forceinline__ void gated(int j, const float_pair* p, float_pair* h) const {
    if (a.gate.p != nullptr) {
      float_pair w[4];
      get(kGate, j, w);
#pragma unroll
      for (int i = 0; i < 4; ++i) h[i] = fma_pair(w[i], p[i], h[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) h[i] = add_pair(h[i], p[i]);
    }
  }
};

// A thread's chunks of the rows to come: stage, then 16-byte unit, then thread, so that a warp's
// accesses lie side by side.  A chunk of 8 fp32 elements is two units, and lanes that copied their
// own would touch every 32-byte sector twice: the warp copies its 64 units in order instead, each to
// its owner's place, and stores go the same way round (__syncwarp on both sides).  (32 frames, fp32
// stream: 116 us without.)
template <int TH, int UNITS>
struct Pipe {
  unsigned char* mine;
  int lane;
  __device__ __forceinline__ explicit Pipe(unsigned char* smem)
      : mine(smem + threadIdx.x * 16), lane(threadIdx.x & 31) {}
  // what is never fetched (past the row's end, tensors that are not there) reads as zeros
  __device__ __forceinline__ void clear() const {
#pragma unroll
    for (int u = 0; u < kStages * UNITS; ++u)
      *reinterpret_cast<uint4*>(mine + u * (TH * 16)) = make_uint4(0, 0, 0, 0);
    __syncwarp();
  }
  __device__ __forceinline__ unsigned char* place(int stage, int unit, int owner) const {
    return mine + (stage * UNITS + unit) * (TH * 16) + (owner - lane) * 16;
  }
  // a chunk of the row that `p` (this lane's elements) lies in, `there` for this lane's elements
  template <typename E>
  __device__ __forceinline__ void fetch(int stage, int unit0, const E* p, bool there) const {
    if (sizeof(E) == 2) {
      if (there) cp_async_16(smem_u32(place(stage, unit0, lane)), p, 16);
      return;
    }
    const unsigned lanes = __ballot_sync(0xffffffffu, there);
    const E* base = p - 8 * lane;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int q = k * 32 + lane, owner = q >> 1;
      if (lanes >> owner & 1)
        cp_async_16(smem_u32(place(stage, unit0 + (q & 1), owner)), base + 4 * q, 16);
    }
  }
  template <typename E>
  __device__ __forceinline__ void read(int stage, int unit0, float_pair* v) const {
    const unsigned char* p = place(stage, unit0, lane);
    if (sizeof(E) == 4) {
      const ulonglong2 lo = *reinterpret_cast<const ulonglong2*>(p);
      const ulonglong2 hi = *reinterpret_cast<const ulonglong2*>(p + TH * 16);
      v[0] = lo.x, v[1] = lo.y, v[2] = hi.x, v[3] = hi.y;
    } else {
      get_pairs(reinterpret_cast<const E*>(p), 8, true, v);
    }
  }
  // stores a chunk, by way of the places of one that has been read
  template <typename E>
  __device__ __forceinline__ void store(int stage, int unit0, E* p, bool there,
                                        const float_pair* v) const {
    if (sizeof(E) == 2) {
      put_pairs<true>(p, there ? 8 : 0, true, v);
      return;
    }
    const unsigned lanes = __ballot_sync(0xffffffffu, there);
    *reinterpret_cast<ulonglong2*>(place(stage, unit0, lane)) = make_ulonglong2(v[0], v[1]);
    *reinterpret_cast<ulonglong2*>(place(stage, unit0 + 1, lane)) = make_ulonglong2(v[2], v[3]);
    __syncwarp();
    E* base = p - 8 * lane;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int q = k * 32 + lane, owner = q >> 1;
      if (lanes >> owner & 1)
        *reinterpret_cast<uint4*>(base + 4 * q) =
            *reinterpret_cast<const uint4*>(place(stage, unit0 + (q & 1), owner));
    }
    // places past the row's end keep their zeros
    if (!there) {
      *reinterpret_cast<uint4*>(place(stage, unit0, lane)) = make_uint4(0, 0, 0, 0);
      *reinterpret_cast<uint4*>(place(stage, unit0 + 1, lane)) = make_uint4(0, 0, 0, 0);
    }
  }
};

// v - c in the first n of 8 elements, the others (zeros) left as they are.
template <bool VEC>
__device__ __forceinline__ void subtract(float_pair* v, int n, float c) {
  if (VEC || n == 8) {
    const float_pair m = both(n > 0 ? -c : 0.f);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = add_pair(v[i], m);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[i] = add_pair(v[i], pack_pair(2 * i < n ? -c : 0.f, 2 * i + 1 < n ? -c : 0.f));
  }
}

// Sums over the row's WPR warps; every thread gets them, added in the same order.  `scratch`
// holds two floats per warp of the block, twice: consecutive calls alternate (`turn`), so that
// one barrier is enough between a call's writes and the next but one's.
template <int WPR>
struct RowSum {
  float* scratch;
  int slot, warp, lane, turn = 0;
  __device__ __forceinline__ RowSum(float* s) : scratch(s) {
    slot = (threadIdx.x >> 5) / WPR;
    warp = (threadIdx.x >> 5) % WPR;
    lane = threadIdx.x & 31;
  }
  __device__ __forceinline__ float* row() {
    float* s = scratch + (turn * 32 + slot * WPR) * 2;
    turn ^= 1;
    return s;
  }
  __device__ __forceinline__ void meet() const {
    asm volatile("bar.sync %0, %1;" ::"r"(1 + slot), "n"(WPR * 32) : "memory");
  }
  // lanes below 16 go on with a, the others with b
  __device__ __forceinline__ void two(float& a, float& b) {
    const bool high = lane >= 16;
    float v = (high ? b : a) + __shfl_xor_sync(0xffffffffu, high ? a : b, 16);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (WPR > 1) {
      float* s = row();
      if ((lane & 15) == 0) s[(lane >> 4) * WPR + warp] = v;
      meet();
      if (WPR <= 4) {
        a = b = 0.f;
#pragma unroll
        for (int i = 0; i < WPR; ++i) {
          a += s[i];
          b += s[WPR + i];
        }
        return;
      }
      v = s[(lane >> 4) * WPR + (lane & (WPR - 1))];
#pragma unroll
      for (int o = WPR / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    }
    a = __shfl_sync(0xffffffffu, v, 0);
    b = __shfl_sync(0xffffffffu, v, 16);
  }
  __device__ __forceinline__ float one(float a) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
    if (WPR > 1) {
      float* s = row();
      if (lane == 0) s[warp] = a;
      meet();
      if (WPR <= 4) {
        a = 0.f;
#pragma unroll
        for (int i = 0; i < WPR; ++i) a += s[i];
        return a;
      }
      a = s[lane & (WPR - 1)];
#pragma unroll
      for (int o = WPR / 2; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
    }
    return a;
  }
};

// v normed in place (elements past the row's end stay zero); returns 1 / deviation.
template <bool VEC, int WPR, int J>
__device__ __forceinline__ float norm_row(float_pair (*v)[4], const int* n, int kind,
                                          float inv_width, float eps, RowSum<WPR>& sum) {
  if (kind == kNormLayer) {
    float_pair s = both(0.f);
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) s = add_pair(s, v[j][i]);
    const float mean = sum.one(sum_pair(s)) * inv_width;
#pragma unroll
    for (int j = 0; j < J; ++j) subtract<VEC>(v[j], n[j], mean);
  }
  float_pair q = both(0.f);
#pragma unroll
  for (int j = 0; j < J; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) q = fma_pair(v[j][i], v[j][i], q);
  const float r = 1.f / sqrtf(sum.one(sum_pair(q)) * inv_width + eps);
  const float_pair rr = both(r);
#pragma unroll
  for (int j = 0; j < J; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) v[j][i] = mul_pair(v[j][i], rr);
  return r;
}

// residual_norm.cu: checks a call's arguments and fills `a`; 0, or the error
int check(const vggt_residual_norm_args* c, Args* a);

// Warps to a row: 16 elements a lane, or 8 where a backward pass also has the sums of the branch's
// norm, whose registers take the room; the widest rows have 32 (and spill).
inline int row_warps(int64_t width, bool half) {
  const int64_t per_warp = half || width <= 256 ? 256 : 512;
  int w = 1;
  while (w < 16 && w * per_warp < width) w *= 2;
  return w;
}

}  // namespace rnorm
}  // namespace vggt
