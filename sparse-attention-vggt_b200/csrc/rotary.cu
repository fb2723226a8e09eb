// Rotary positions, and the append of rotated keys and of values to a paged
// cache.
//
// A pair (x, y) of a head turns by the angle a = position * freq:
//   (x cos a - y sin a, x sin a + y cos a) * lengthen.
// No table of cosines is read.  The angle is kept as a fraction of a turn in
// 64-bit fixed point: step = round(freq / 2 pi * 2^64) modulo 2^64, and
// position * step wraps to exactly the fraction that the product has, so the
// reduction is exact for every 32-bit position (a 32-bit float product
// position * freq is off by 4e-3 radians at position 65,536).  Its upper 32
// bits name the quarter turn and what is left of it, which keeps 24 bits as a
// float: the angle is within 2^-24 of a radian.
//
// The kernels are bound by memory: every element is read and written once (32
// frames' queries, 180 MB, in 34.7 us: 5.2 TB/s, 0.81 of the measured copy
// rate).
// A thread owns up to 8 pairs (two 16-byte vectors of a 2-byte type) of a
// token, takes their sines once and walks over heads with them, four heads'
// loads in flight at a time.  With few tokens the heads are dealt to more
// threads, until the grid fills the card.  (Sines of a CTA's tokens in shared
// memory and rows in the order of memory: 47.9 us.)
#include "kernels.h"
#include "paged.cuh"

namespace vggt {
namespace {

constexpr int kThreads = 256;

// `N` bytes, moved by one instruction where N is 2, 4, 8 or 16.
template <int N>
struct Bytes;
template <>
struct Bytes<2> { using T = uint16_t; };
template <>
struct Bytes<4> { using T = uint32_t; };
template <>
struct Bytes<8> { using T = uint2; };
template <>
struct Bytes<16> { using T = uint4; };

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// N elements in vectors of at most 16 bytes.
template <typename T, int N>
struct Vec {
  static constexpr int kBytes = N * (int)sizeof(T) > 16 ? 16 : N * (int)sizeof(T);
  static constexpr int kCount = N * (int)sizeof(T) / kBytes;
  using V = typename Bytes<kBytes>::T;
  V v[kCount];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < kCount; ++i) v[i] = reinterpret_cast<const V*>(p)[i];
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < kCount; ++i) reinterpret_cast<V*>(p)[i] = v[i];
  }
  __device__ __forceinline__ T* e() { return reinterpret_cast<T*>(v); }
};

// Sine and cosine of `turn` / 2^32 of a turn.  The nearest quarter comes off
// as an integer, exactly; the rest, at most pi/4, goes through the Taylor
// series, whose first terms left out are 1.8e-9 (x^11 / 11!) and 1.2e-10
// (x^12 / 12!).  Odd quarters swap the two, the signs follow the quarter.
__device__ __forceinline__ void sine(uint32_t turn, float& s, float& c) {
  const uint32_t quarter = (turn + 0x20000000u) >> 30;
  const float x = (float)(int32_t)(turn - (quarter << 30)) * 1.4629180792671596e-9f;  // 2 pi / 2^32
  const float y = x * x;
  float u = fmaf(y, 1.f / 362880.f, -1.f / 5040.f), w = fmaf(y, -1.f / 3628800.f, 1.f / 40320.f);
  u = fmaf(y, u, 1.f / 120.f);
  w = fmaf(y, w, -1.f / 720.f);
  u = fmaf(y, u, -1.f / 6.f);
  w = fmaf(y, w, 1.f / 24.f);
  u = fmaf(x * y, u, x);
  w = fmaf(y, fmaf(y, w, -0.5f), 1.f);
  const uint32_t a = __float_as_uint(quarter & 1 ? w : u), b = __float_as_uint(quarter & 1 ? u : w);
  s = __uint_as_float(a ^ ((quarter << 30) & 0x80000000u));
  c = __uint_as_float(b ^ (((quarter + 1) << 30) & 0x80000000u));
}

struct Angles {
  const int32_t* positions;  // [tokens][axes]
  const double* freq;        // [pairs]
  int axes, pairs, interleaved;
  float lengthen, sign;
};

// One unit of a head: 2 * N elements, as two runs of N at offsets a and b.
// Units below axes * pairs / N rotate N pairs; the rest copy.
template <int N>
struct Unit {
  int a, b;
  int axis;  // -1: copies
  uint64_t step[N];
  float c[N], s[N];

  __device__ __forceinline__ Unit(const Angles& g, int unit) {
    const int first = unit * N;  // pair number over all axes
    if (first >= g.axes * g.pairs) {
      axis = -1;
      a = 2 * first;
      b = a + N;
      return;
    }
    axis = first / g.pairs;
    const int i0 = first % g.pairs;
    if (g.interleaved) {
      a = 2 * first;
      b = a + N;
    } else {
      a = 2 * axis * g.pairs + i0;
      b = a + g.pairs;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      double t = __ldg(g.freq + i0 + i) * 0.15915494309189535;  // turns per position
      t -= rint(t);
      step[i] = (uint64_t)__double2ll_rn(t * 9223372036854775808.0) << 1;
    }
  }

  // the sines of a token's position
  __device__ __forceinline__ void at(const Angles& g, int64_t token) {
    if (axis < 0) return;
    const uint64_t pos = (uint64_t)(int64_t)__ldg(g.positions + token * g.axes + axis);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      sine((uint32_t)((pos * step[i]) >> 32), s[i], c[i]);
      c[i] *= g.lengthen;
      s[i] *= g.lengthen * g.sign;
    }
  }

  template <typename T>
  __device__ __forceinline__ void turn(T* x, T* y, bool interleaved) const {
    if (axis < 0) return;
    if (interleaved) {  // pairs lie side by side over both runs
#pragma unroll
      for (int i = 0; i < N; ++i) {
        T* p = 2 * i < N ? x + 2 * i : y + (2 * i - N);
        T* q = 2 * i + 1 < N ? x + 2 * i + 1 : y + (2 * i + 1 - N);
        const float u = to_f(*p), w = to_f(*q);
        *p = from_f<T>(u * c[i] - w * s[i]);
        *q = from_f<T>(u * s[i] + w * c[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float u = to_f(x[i]), w = to_f(y[i]);
        x[i] = from_f<T>(u * c[i] - w * s[i]);
        y[i] = from_f<T>(u * s[i] + w * c[i]);
      }
    }
  }
};

// at / d and at % d, in 32 bits where `at` has no more.
__device__ __forceinline__ int64_t divided(int64_t at, int d, int& rest) {
  if ((at >> 32) == 0) {
    const uint32_t q = (uint32_t)at / (uint32_t)d;
    rest = (int)((uint32_t)at - q * (uint32_t)d);
    return q;
  }
  const int64_t q = at / d;
  rest = (int)(at - q * d);
  return q;
}

constexpr int kBatch = 4;  // rows of a token or tokens whose loads are in flight together

struct RotaryArgs {
  const void* x;
  void* out;
  int64_t tokens, xt, xh, ot, oh;
  int heads, units, deal;  // units per head; threads that share a token's heads
  int64_t stride;          // few heads: a thread's tokens are this far apart
  Angles g;
};

template <typename T, int N>
__global__ void __launch_bounds__(kThreads) rotary_kernel(RotaryArgs p) {
  int unit, part;
  const int64_t token =
      divided(divided((int64_t)blockIdx.x * kThreads + threadIdx.x, p.units, unit), p.deal, part);
  if (token >= p.tokens) return;
  Unit<N> u(p.g, unit);
  const T* x = static_cast<const T*>(p.x) + token * p.xt;
  T* o = static_cast<T*>(p.out) + token * p.ot;
#pragma unroll 1
  for (int h0 = part; h0 < p.heads; h0 += kBatch * p.deal) {
    Vec<T, N> a[kBatch], b[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int64_t h = h0 + j * p.deal;
      if (h < p.heads) {
        a[j].load(x + h * p.xh + u.a);
        b[j].load(x + h * p.xh + u.b);
      }
    }
    if (h0 == part) u.at(p.g, token);
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int64_t h = h0 + j * p.deal;
      if (h < p.heads) {
        u.turn(a[j].e(), b[j].e(), p.g.interleaved);
        a[j].store(o + h * p.oh + u.a);
        b[j].store(o + h * p.oh + u.b);
      }
    }
  }
}

// Few heads: a thread takes kBatch tokens of one head, so that as many loads
// are in flight as with many heads, and the steps are formed once for them.
// (One head of 64, 703,488 tokens: 53 us, against 99; what is left are the
// sines, 50 instructions each.  With 8 pairs to a thread three CTAs to an SM
// spill 28 bytes and take 53 us, two without a spill 61.)
template <typename T, int N>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 4 ? 2 : 3)
    rotary_few_heads_kernel(RotaryArgs p) {
  int unit, head;
  const int64_t first =
      divided(divided((int64_t)blockIdx.x * kThreads + threadIdx.x, p.units, unit), p.heads, head);
  if (first >= p.stride) return;
  Unit<N> u(p.g, unit);
  const T* x = static_cast<const T*>(p.x) + head * p.xh;
  T* o = static_cast<T*>(p.out) + head * p.oh;
  Vec<T, N> a[kBatch], b[kBatch];
#pragma unroll
  for (int j = 0; j < kBatch; ++j) {
    const int64_t token = first + j * p.stride;
    if (token < p.tokens) {
      a[j].load(x + token * p.xt + u.a);
      b[j].load(x + token * p.xt + u.b);
    }
  }
#pragma unroll
  for (int j = 0; j < kBatch; ++j) {
    const int64_t token = first + j * p.stride;
    if (token < p.tokens) {
      u.at(p.g, token);
      u.turn(a[j].e(), b[j].e(), p.g.interleaved);
      a[j].store(o + token * p.ot + u.a);
      b[j].store(o + token * p.ot + u.b);
    }
  }
}

struct AppendArgs {
  const void *k, *v;
  void *kp, *vp;
  int64_t kt, kh, vt, vh;
  Pool pool;
  PageTable t;  // lengths: before the call
  int units, deal;
  int64_t main_blocks;
  Angles g;
  int32_t *ids, *after;
  const int32_t* new_ids;
  float* weights;
  const float* new_weights;
};

// Slot of packed row `row`, or -1 (no sequence, or past the last slot).
__device__ __forceinline__ int64_t append_slot(const AppendArgs& p, int64_t row, int64_t& seq) {
  seq = sequence_of_row(p.t.starts, p.t.seqs, row);
  if (seq < 0) {
    raise_status(p.t.status, VGGT_STATUS_BAD_LENGTH);
    return -1;
  }
  const int64_t slot = checked_length(p.t, p.pool, seq) + row - __ldg(p.t.starts + seq);
  if (slot < (p.t.width << p.pool.page_shift)) return slot;
  raise_status(p.t.status, VGGT_STATUS_BAD_LENGTH);
  return -1;
}

// (Three CTAs to an SM at least, which spills 4 bytes in one form: 4 prompts of
// up to 2,048 tokens 17.1 us, at the 106 registers of two CTAs 20.1.)
template <typename T, int N>
__global__ void __launch_bounds__(kThreads, 3) append_kernel(AppendArgs p) {
  if (blockIdx.x >= p.main_blocks) {
    // ids, weights (tokens along the lanes, so that a warp writes neighbours)
    // and the new lengths
    const int64_t at = ((int64_t)blockIdx.x - p.main_blocks) * kThreads + threadIdx.x;
    if (at < p.t.seqs) {
      int64_t first;
      const int64_t n = checked_length(p.t, p.pool, at) + checked_rows(p.t, at, first);
      const int64_t slots = p.t.width << p.pool.page_shift;
      p.after[at] = (int32_t)(n < slots ? n : slots);
    }
    if (at >= p.t.total || (p.ids == nullptr && p.weights == nullptr)) return;
    int64_t seq;
    const int64_t slot = append_slot(p, at, seq);
    if (slot < 0) return;
    const int64_t slots = p.t.width << p.pool.page_shift;
    const int64_t dst = seq * p.pool.kv_heads * slots + slot;
    const int32_t id = p.ids != nullptr ? __ldg(p.new_ids + at) : 0;
    const float w = p.new_weights != nullptr ? __ldg(p.new_weights + at) : 0.f;
    for (int h = 0; h < p.pool.kv_heads; ++h) {
      if (p.ids != nullptr) p.ids[dst + h * slots] = id;
      if (p.weights != nullptr) p.weights[dst + h * slots] = w;
    }
    return;
  }
  int unit, part;
  const int64_t row =
      divided(divided((int64_t)blockIdx.x * kThreads + threadIdx.x, p.units, unit), p.deal, part);
  if (row >= p.t.total) return;
  int64_t seq;
  const int64_t slot = append_slot(p, row, seq);
  if (slot < 0) return;
  const int page = checked_page(p.t, p.pool, seq, slot >> p.pool.page_shift);
  if (page < 0) return;
  Unit<N> u(p.g, unit);
  u.at(p.g, row);
  const int64_t dst = page * p.pool.page_stride + (slot & (p.pool.page - 1)) * p.pool.row_stride;
  const T* k = static_cast<const T*>(p.k) + row * p.kt;
  const T* v = static_cast<const T*>(p.v) + row * p.vt;
  T* kp = static_cast<T*>(p.kp) + dst;
  T* vp = static_cast<T*>(p.vp) + dst;
  constexpr int kBatch = 2;  // of keys and of values
  for (int h0 = part; h0 < p.pool.kv_heads; h0 += kBatch * p.deal) {
    Vec<T, N> a[kBatch], b[kBatch], c[kBatch], d[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int64_t h = h0 + j * p.deal;
      if (h < p.pool.kv_heads) {
        a[j].load(k + h * p.kh + u.a);
        b[j].load(k + h * p.kh + u.b);
        c[j].load(v + h * p.vh + u.a);
        d[j].load(v + h * p.vh + u.b);
      }
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int64_t h = h0 + j * p.deal;
      if (h < p.pool.kv_heads) {
        u.turn(a[j].e(), b[j].e(), p.g.interleaved);
        a[j].store(kp + h * p.pool.head_stride + u.a);
        b[j].store(kp + h * p.pool.head_stride + u.b);
        c[j].store(vp + h * p.pool.head_stride + u.a);
        d[j].store(vp + h * p.pool.head_stride + u.b);
      }
    }
  }
}

// Pairs per thread: the widest vector that divides the pairs of an axis and
// the rest of the head, and that every address is aligned to.
int pairs_per_thread(int size, int dim, int axes, int pairs, std::initializer_list<int64_t> strides,
                     std::initializer_list<const void*> bases) {
  for (int n = 8; n > 1; n >>= 1) {
    const int64_t bytes = (int64_t)n * size > 16 ? 16 : (int64_t)n * size;
    bool ok = (axes == 0 || pairs % n == 0) && (dim - 2 * axes * pairs) % (2 * n) == 0;
    for (int64_t s : strides) ok = ok && (s * size) % bytes == 0;
    for (const void* b : bases) ok = ok && reinterpret_cast<uintptr_t>(b) % bytes == 0;
    if (ok) return n;
  }
  return 1;
}

constexpr int64_t kFill = 148 * 1024;  // threads that fill the card

// Threads that share a token's heads: one, or as many as it takes to fill the
// card.
int deal_heads(int64_t threads, int heads) {
  int64_t d = threads > 0 ? (kFill + threads - 1) / threads : 1;
  return (int)(d < 1 ? 1 : (d > heads ? heads : d));
}

template <typename T, int N>
void launch_rotary(const RotaryArgs& a, unsigned grid, cudaStream_t st) {
  if (a.stride < a.tokens)
    rotary_few_heads_kernel<T, N><<<grid, kThreads, 0, st>>>(a);
  else
    rotary_kernel<T, N><<<grid, kThreads, 0, st>>>(a);
}

template <typename T>
cudaError_t rotary_n(int n, const RotaryArgs& a, unsigned grid, cudaStream_t st) {
  switch (n) {
    case 8: launch_rotary<T, 8>(a, grid, st); break;
    case 4: launch_rotary<T, 4>(a, grid, st); break;
    case 2: launch_rotary<T, 2>(a, grid, st); break;
    default: launch_rotary<T, 1>(a, grid, st); break;
  }
  return cudaGetLastError();
}

template <typename T>
cudaError_t append_n(int n, const AppendArgs& a, unsigned grid, cudaStream_t st) {
  switch (n) {
    case 8: append_kernel<T, 8><<<grid, kThreads, 0, st>>>(a); break;
    case 4: append_kernel<T, 4><<<grid, kThreads, 0, st>>>(a); break;
    case 2: append_kernel<T, 2><<<grid, kThreads, 0, st>>>(a); break;
    default: append_kernel<T, 1><<<grid, kThreads, 0, st>>>(a); break;
  }
  return cudaGetLastError();
}

}  // namespace
}  // namespace vggt

using namespace vggt;

namespace {

int check_rotation(int dim, const int32_t* positions, int axes, const double* freq, int pairs,
                   int layout, float lengthen) {
  if (layout != VGGT_ROTARY_HALF && layout != VGGT_ROTARY_INTERLEAVED)
    return api_fail("unknown rotary layout %d", layout);
  if (axes < 1 || axes > 4) return api_fail("axes %d outside [1, 4]", axes);
  if (pairs < 1 || (int64_t)2 * axes * pairs > dim)
    return api_fail("2 * axes * pairs = %lld elements rotate in heads of %d",
                    (long long)2 * axes * pairs, dim);
  if (!(lengthen - lengthen == 0.f)) return api_fail("lengthen must be finite");
  if (!positions || !freq) return api_fail("positions and freq must be non-NULL");
  return 0;
}

}  // namespace

extern "C" int vggt_rotary(const void* x, int dtype, int64_t tokens, int heads, int dim,
                           int64_t x_token_stride, int64_t x_head_stride,
                           const int32_t* positions, int axes, const double* freq, int pairs,
                           int layout, float lengthen, int inverse, void* out,
                           int64_t out_token_stride, int64_t out_head_stride, void* stream) {
  if (dtype != VGGT_DTYPE_BF16 && dtype != VGGT_DTYPE_FP16 && dtype != VGGT_DTYPE_FP32)
    return api_fail("rotary requires BF16, FP16 or FP32 (dtype code %d)", dtype);
  if (tokens < 0 || heads < 0) return api_fail("negative size argument");
  if (dim < 2 || dim % 2 || dim > 65536) return api_fail("head dim %d must be even and positive", dim);
  if (tokens == 0 || heads == 0) return api_fail(nullptr);
  if (int rc = check_rotation(dim, positions, axes, freq, pairs, layout, lengthen)) return rc;
  if (!x || !out) return api_fail("x and out must be non-NULL");
  const int size = dtype == VGGT_DTYPE_FP32 ? 4 : 2;
  const int n = pairs_per_thread(size, dim, axes, pairs,
                                 {x_token_stride, x_head_stride, out_token_stride, out_head_stride},
                                 {x, out});
  RotaryArgs a{x, out, tokens, x_token_stride, x_head_stride, out_token_stride, out_head_stride,
               heads, dim / (2 * n), 1, tokens,
               {positions, freq, axes, pairs, layout == VGGT_ROTARY_INTERLEAVED, lengthen,
                inverse ? -1.f : 1.f}};
  a.deal = deal_heads(tokens * a.units, heads);
  // Half a batch of heads at most (two heads: 53 against 64 us; three: 52
  // against 42), and tokens that fill the card with a thread for each
  if (heads <= kBatch / 2 && tokens * a.units * heads >= kFill) {
    a.stride = (tokens + kBatch - 1) / kBatch;
    a.deal = heads;
  }
  const int64_t grid = (a.stride * a.units * a.deal + kThreads - 1) / kThreads;
  if (grid > 0x7fffffffLL) return api_fail("too many tokens (%lld)", (long long)tokens);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return api_cuda(dtype == VGGT_DTYPE_FP32   ? rotary_n<float>(n, a, (unsigned)grid, st)
                  : dtype == VGGT_DTYPE_FP16 ? rotary_n<__half>(n, a, (unsigned)grid, st)
                                             : rotary_n<__nv_bfloat16>(n, a, (unsigned)grid, st));
}

extern "C" int vggt_paged_append(
    const void* k, const void* v, int dtype, int64_t total, int64_t k_token_stride,
    int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride, void* k_pages,
    void* v_pages, int64_t n_pages, int kv_heads, int page, int dim, int64_t page_stride,
    int64_t head_stride, int64_t row_stride, const int32_t* table, int64_t table_width,
    int64_t seqs, const int32_t* before, const int32_t* starts, const int32_t* positions, int axes,
    const double* freq, int pairs, int layout, float lengthen, int32_t* ids,
    const int32_t* new_ids, float* weights, const float* new_weights, int32_t* after,
    int32_t* status, void* stream) {
  AppendArgs a{};
  if (int rc = check_pool(dtype, n_pages, kv_heads, page, dim, page_stride, head_stride,
                          row_stride, table_width, seqs, total, &a.pool))
    return rc;
  if (seqs == 0) return api_fail(nullptr);
  if (positions != nullptr) {
    if (int rc = check_rotation(dim, positions, axes, freq, pairs, layout, lengthen)) return rc;
  } else {
    axes = 0;
    pairs = 1;
  }
  if (!before || !starts || !after) return api_fail("before, starts and after must be non-NULL");
  if (total > 0 && (!k || !v || !k_pages || !v_pages || !table))
    return api_fail("k, v, the pools and the table must be non-NULL");
  if (ids != nullptr && new_ids == nullptr) return api_fail("ids needs new_ids");
  const int n = pairs_per_thread(2, dim, axes, pairs,
                                 {k_token_stride, k_head_stride, v_token_stride, v_head_stride,
                                  page_stride, head_stride, row_stride},
                                 {k, v, k_pages, v_pages});
  a.k = k;
  a.v = v;
  a.kp = k_pages;
  a.vp = v_pages;
  a.kt = k_token_stride;
  a.kh = k_head_stride;
  a.vt = v_token_stride;
  a.vh = v_head_stride;
  a.t = {table, before, starts, table_width, seqs, total, status};
  a.units = dim / (2 * n);
  a.deal = deal_heads(total * a.units, kv_heads);
  a.main_blocks = (total * a.units * a.deal + kThreads - 1) / kThreads;
  a.g = {positions, freq, axes, pairs, layout == VGGT_ROTARY_INTERLEAVED, lengthen, 1.f};
  a.ids = ids;
  a.after = after;
  a.new_ids = new_ids;
  a.weights = weights;
  a.new_weights = new_weights;
  const int64_t grid = a.main_blocks + ((total > seqs ? total : seqs) + kThreads - 1) / kThreads;
  if (grid > 0x7fffffffLL) return api_fail("too many new tokens (%lld)", (long long)total);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return api_cuda(dtype == VGGT_DTYPE_FP16 ? append_n<__half>(n, a, (unsigned)grid, st)
                                           : append_n<__nv_bfloat16>(n, a, (unsigned)grid, st));
}
