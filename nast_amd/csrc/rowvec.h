// Rows of fp32 / bf16 / fp16 logits read in 16-byte vectors at any alignment, and the arithmetic the vocabulary-row
// operators of toplogits.hip and verify.hip share: exponentials, (max, sum) pairs, order-preserving keys.
#pragma once
#include <float.h>

#include "common.h"

// One struct per storage type: EPV elements in 16 bytes, their conversion to fp32 (exact) and back (to nearest even); the low
// KEY_ZEROS bits of an fp32 mantissa that no value of the type uses.
// Vectors are kept as four words: as eight halves the compiler gives each a register.
struct RowF32 {
  using store = float;
  static constexpr int EPV = 4, KEY_ZEROS = 0;
  static __device__ __forceinline__ float get(store v) { return v; }
  static __device__ __forceinline__ store put(float v) { return v; }
  static __device__ __forceinline__ float unpack(uint32_t w, int) { return __builtin_bit_cast(float, w); }
  static __device__ __forceinline__ uint32_t pack(const float* f) { return __builtin_bit_cast(uint32_t, f[0]); }
};
struct RowBF16 {
  using store = __bf16;
  using pair = __bf16 __attribute__((ext_vector_type(2)));
  static constexpr int EPV = 8, KEY_ZEROS = 16;
  static __device__ __forceinline__ float get(store v) { return (float)v; }
  static __device__ __forceinline__ store put(float v) { return (store)v; }
  static __device__ __forceinline__ float unpack(uint32_t w, int half) { return __builtin_bit_cast(float, half ? w & 0xffff0000u : w << 16); }
  static __device__ __forceinline__ uint32_t pack(const float* f) { return __builtin_bit_cast(uint32_t, pair{(store)f[0], (store)f[1]}); }
};
struct RowF16 {
  using store = _Float16;
  using pair = _Float16 __attribute__((ext_vector_type(2)));
  static constexpr int EPV = 8, KEY_ZEROS = 13;
  static __device__ __forceinline__ float get(store v) { return (float)v; }
  static __device__ __forceinline__ store put(float v) { return (store)v; }
  static __device__ __forceinline__ float unpack(uint32_t w, int half) { return (float)__builtin_bit_cast(pair, w)[half]; }
  static __device__ __forceinline__ uint32_t pack(const float* f) { return __builtin_bit_cast(uint32_t, pair{(store)f[0], (store)f[1]}); }
};

template <class D>
struct RowVec {
  static constexpr int PER = D::EPV / 4;   // elements a word
  uint32_t w[4];
  __device__ __forceinline__ float get(int i) const { return D::unpack(w[i / PER], i % PER); }
  __device__ __forceinline__ void put(const float (&f)[D::EPV]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = D::pack(f + i * PER);
  }
};
template <class D>
__device__ __forceinline__ RowVec<D> vec_of(float f) {   // one value in every element
  const float two[2] = {f, f};
  const uint32_t w = D::pack(two);
  return {{w, w, w, w}};
}
template <class D>
__device__ __forceinline__ RowVec<D> vec_load(const typename D::store* p) {   // p 16-byte aligned
  const uint4 q = *reinterpret_cast<const uint4*>(p);
  return {{q.x, q.y, q.z, q.w}};
}
template <class D>
__device__ __forceinline__ void vec_store(typename D::store* p, const RowVec<D>& v) {
  *reinterpret_cast<uint4*>(p) = make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]);
}
typedef uint32_t raw16 __attribute__((ext_vector_type(4)));
template <class D>
__device__ __forceinline__ void vec_store_around(typename D::store* p, const RowVec<D>& v) {   // not kept in the last-level cache
  __builtin_nontemporal_store(raw16{v.w[0], v.w[1], v.w[2], v.w[3]}, reinterpret_cast<raw16*>(p));
}
// 16 bytes from any element: global_load_dwordx4 takes any alignment on this target
typedef uint32_t raw16_any __attribute__((ext_vector_type(4), aligned(2)));
template <class D>
__device__ __forceinline__ RowVec<D> vec_load_any(const typename D::store* p) {
  const raw16_any q = *reinterpret_cast<const raw16_any*>(p);
  return {{q.x, q.y, q.z, q.w}};
}

// Elements [lo, hi) of a row: a body of whole 16-byte aligned vectors, slot s at element body + s * EPV, and at most EPV - 1 elements
// in front of it and behind it.  Those are dealt out one to a thread (threads 0.. and 64..), so that no vector has holes.
template <class D>
struct RowSpan16 {
  int lo, hi, body, n, tail;
  __device__ __forceinline__ RowSpan16(const typename D::store* p, int lo_, int hi_) : lo(lo_), hi(hi_) {
    const int lead = (int)((0 - reinterpret_cast<uintptr_t>(p + lo_)) & 15) / (int)sizeof(typename D::store);
    body = min(lo_ + lead, hi_);
    n = (hi_ - body) / D::EPV;
    tail = body + n * D::EPV;
  }
  __device__ __forceinline__ int elem(int s) const { return body + s * D::EPV; }
  __device__ __forceinline__ RowVec<D> load(const typename D::store* p, int s) const {
    return vec_load<D>(p + body + s * D::EPV);
  }
  // the element thread t has to look after besides its slots, or -1
  __device__ __forceinline__ int edge(int t) const {
    if (t < body - lo) return lo + t;
    return t >= 64 && t - 64 < hi - tail ? tail + (t - 64) : -1;
  }
};

// exp(t / T) as 2^(t * c), c = log2(e) / T rounded to fp32.  t is a difference to a maximum (<= 0 or -inf or NaN).  The product's
// rounding and c's make the result wrong by at most |t * c| * 2^-23 * ln 2 relative: 4e-6 where it is 2^-40, 1e-7 where it is near 1.
static inline float exp_scale(double temp) { return (float)(1.4426950408889634 / temp); }
__device__ __forceinline__ float exp_t(float t, float c) { return __builtin_amdgcn_exp2f(t * c); }

// Sum of exponentials relative to a maximum.  The maximum starts at the lowest finite value, so that no -inf is subtracted from
// -inf: a row of -inf ends with s = 0 (log-sum-exp -inf), a row of the type's lowest value counts as any other row.  A NaN or
// +inf among the elements leaves s = NaN.  Vectors are summed in fp32 (at most 32 terms), everything from there in double.
// What a row's s is off by, relative.  An element's term is a product of powers 2^-a: its own, and one for each time the sum it is in was
// brought to a larger maximum: at most R times in its thread (once a batch of for_slots and once for the edge), then over the wavefront, the
// workgroup and the row's chunks.  A power has 3 roundings of its argument (difference, product, c), 1.24e-7 * a, and the instruction's
// 1.2e-7 (one unit; 8.5e-8 measured over [-1, 0]).  The a's of an element add up to log2 of the largest term over its own; weighted by
// the terms that is 15.2 on average at most for V = 2^20 and 18.9 for 2^24 (one element with 0.09 or 0.07 of the sum, the others alike).
// 12 roundings of a sum add 7e-7:  1.24e-7 * 15.2 + 1.2e-7 * (R + 4) + 7e-7.
//   chunks of 2^15 elements (verification): 8 batches whole, or 7, 4 vectors and an edge: R = 12, 4.5e-6, below ROW_SUM_REL
//   chunks of 2^15 vectors (distillation): 32 batches, or 31, 4 vectors and an edge: R = 36, 7.9e-6 for V = 2^24
#define ROW_SUM_REL 5e-6
struct MaxSum {
  float m;
  double s;
};
// U vectors at a time: one comparison with the running maximum and at most one rescaling for all of them
template <class D, int U>
__device__ __forceinline__ void fold(MaxSum& a, const RowVec<D> (&v)[U], float c) {
  float top = -FLT_MAX;
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int i = 0; i < D::EPV; ++i) top = fmaxf(top, v[u].get(i));
  if (top > a.m) {
    a.s *= (double)exp_t(a.m - top, c);
    a.m = top;
  }
  float all = 0.f;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < D::EPV; ++i) s += exp_t(v[u].get(i) - a.m, c);
    all += s;
  }
  a.s += (double)all;
}
__device__ __forceinline__ void fold_one(MaxSum& a, float f, float c) {
  if (f > a.m) {
    a.s *= (double)exp_t(a.m - f, c);
    a.m = f;
  }
  a.s += (double)exp_t(f - a.m, c);
}

// The slots of a span in batches of U vectors a thread: full(v, first slot) for a batch that every thread has whole, part(v, slot) for
// each vector of the last one.  No branch around a load: the compiler would wait for each before the next.
template <class D, int NT, int U, class L, class F, class P>
__device__ __forceinline__ void for_slots(const RowSpan16<D>& rs, L&& load, F&& full, P&& part) {
  const int tid = threadIdx.x;
  int b = 0;
  for (; b + NT * U <= rs.n; b += NT * U) {
    RowVec<D> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = load(b + NT * u + tid);
    full(v, b + tid);
  }
  if (b >= rs.n) return;
  RowVec<D> v[U];
#pragma unroll
  for (int u = 0; u < U; ++u) v[u] = load(min(b + NT * u + tid, rs.n - 1));
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (b + NT * u + tid < rs.n) part(v[u], b + NT * u + tid);
}

// a thread's share of elements [lo, hi) of a row
template <class D, int NT, int U = 4>
__device__ __forceinline__ MaxSum span_max_sum(const typename D::store* p, int lo, int hi, float c) {
  const RowSpan16<D> rs(p, lo, hi);
  const int e = rs.edge(threadIdx.x);
  const typename D::store edge = p[e >= 0 ? e : lo];
  MaxSum a{-FLT_MAX, 0.0};
  for_slots<D, NT, U>(rs, [&](int s) { return rs.load(p, s); }, [&](const RowVec<D>(&v)[U], int) { fold<D, U>(a, v, c); },
                      [&](const RowVec<D>& v, int) {
                        const RowVec<D> one[1] = {v};
                        fold<D, 1>(a, one, c);
                      });
  if (e >= 0) fold_one(a, D::get(edge), c);
  return a;
}

struct MaxSumD {
  double m, s;   // m in units of the logits (not divided by T)
};
__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
__device__ __forceinline__ double wave_max_d(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmax(v, __shfl_xor(v, o, 64));
  return v;
}
// every thread gets the block's pair; red: LDS of 2 * NT / 64 doubles; two barriers
template <int NT>
__device__ __forceinline__ MaxSumD block_max_sum(MaxSum a, float c, double* red) {
  const float wm = wave_max(a.m);
  const double ws = wave_sum_d(a.s * (double)exp_t(a.m - wm, c));
  const int w = threadIdx.x >> 6;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) {
    red[2 * w] = wm;
    red[2 * w + 1] = ws;
  }
  __syncthreads();
  double m = red[0];
#pragma unroll
  for (int i = 1; i < NT / 64; ++i) m = fmax(m, red[2 * i]);
  double s = 0;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) s += red[2 * i + 1] * (double)exp_t((float)(red[2 * i] - m), c);
  return {m, s};
}

__device__ __forceinline__ int lanes_below(uint64_t mask) {    // how many bits of the mask lie below this lane's
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}
// what a lane has written to LDS is there for the other lanes of its wavefront
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Key whose unsigned order is the order of the values: -0 equals +0, NaN (any) above +inf.
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t b = __builtin_bit_cast(uint32_t, v + 0.0f);
  const uint32_t k = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return v != v ? 0xffffffffu : k;
}

__device__ __forceinline__ float key_value(uint32_t k) {
  return __builtin_bit_cast(float, (k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

// Into how many chunks a row of V elements is cut: as few as `most` elements a chunk allow; more while rows * chunks is below 512
// workgroups (two a compute unit), but none shorter than `least`.  Chunks of ceil(V / n) elements then leave none empty, as long as
// n * n <= V: `least` and `most` here are 2048 and more, n is 512 and less.
static inline int row_chunks(int64_t rows, int V, int most, int least) {
  const int need = (V + most - 1) / most;
  int n = rows > 0 && rows < 512 ? (int)((512 + rows - 1) / rows) : 1;
  if (n > V / least) n = V / least;
  return n > need ? n : need;
}

static inline int row_size(int dtype) { return dtype == NAST_F32 ? 4 : 2; }
static inline bool row_dtype_ok(int dtype) { return dtype == NAST_F32 || dtype == NAST_BF16 || dtype == NAST_F16; }
static inline bool row_aligned(const void* p, int dtype) { return (reinterpret_cast<uintptr_t>(p) & (row_size(dtype) - 1)) == 0; }

// `call` with D = the struct of the dtype
#define NAST_ROW_DTYPE(dtype, ...)                       \
  do {                                                   \
    if ((dtype) == NAST_F32) { using D = RowF32; __VA_ARGS__; }        \
    else if ((dtype) == NAST_BF16) { using D = RowBF16; __VA_ARGS__; } \
    else { using D = RowF16; __VA_ARGS__; }              \
  } while (0)
