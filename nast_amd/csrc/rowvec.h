// Rows of fp32 / bf16 / fp16 logits read in 16-byte vectors at any alignment, and the arithmetic the vocabulary-row
// operators of toplogits.hip and verify.hip share: exponentials, (max, sum) pairs, order-preserving keys.
#pragma once
#include <float.h>

#include "common.h"

// One struct per storage type: EPV elements in 16 bytes, their conversion to fp32 (exact) and back (to nearest even).
struct RowF32 {
  using store = float;
  static constexpr int EPV = 4;
  static constexpr float neg_inf() { return -INFINITY; }
  static __device__ __forceinline__ float get(store v) { return v; }
  static __device__ __forceinline__ store put(float v) { return v; }
};
struct RowBF16 {
  using store = __bf16;
  static constexpr int EPV = 8;
  static __device__ __forceinline__ float get(store v) { return (float)v; }
  static __device__ __forceinline__ store put(float v) { return (store)v; }
};
struct RowF16 {
  using store = _Float16;
  static constexpr int EPV = 8;
  static __device__ __forceinline__ float get(store v) { return (float)v; }
  static __device__ __forceinline__ store put(float v) { return (store)v; }
};

template <class D>
union RowVec {
  uint4 raw;
  typename D::store e[D::EPV];
};

// Elements [lo, hi) of a row in vector slots: slot s holds elements first + s * EPV ..., where `first` <= lo is the element
// whose address is 16-byte aligned.  The slots at the two ends may stick out of [lo, hi); those are read and written element
// by element, what lies outside reads as -inf and is never touched.
template <class D>
struct RowSlots {
  int first, lo, hi, n;
  __device__ __forceinline__ RowSlots(const typename D::store* p, int lo_, int hi_) : lo(lo_), hi(hi_) {
    const int lead = (int)((reinterpret_cast<uintptr_t>(p + lo_) & 15) / sizeof(typename D::store));
    first = lo_ - lead;
    n = (hi_ - first + D::EPV - 1) / D::EPV;
  }
  __device__ __forceinline__ int elem(int s) const { return first + s * D::EPV; }
  __device__ __forceinline__ bool whole(int s) const { return elem(s) >= lo && elem(s) + D::EPV <= hi; }
  __device__ __forceinline__ RowVec<D> load(const typename D::store* p, int s) const {
    RowVec<D> v;
    const int e0 = elem(s);
    if (whole(s)) {
      v.raw = *reinterpret_cast<const uint4*>(p + e0);
    } else {
#pragma unroll
      for (int i = 0; i < D::EPV; ++i) v.e[i] = (e0 + i >= lo && e0 + i < hi) ? p[e0 + i] : D::put(-INFINITY);
    }
    return v;
  }
};

// exp(t / T) = 2^(t * log2(e) / T) with the factor held in two floats: one rounding of the product's magnitude, ~1e-7 relative in
// the result for t / T > -30 instead of ~1e-6.  t is a difference to a maximum: <= 0 or -inf or NaN.  (The low part is taken of a
// clamped t: -inf times a low part of 0 or of the other sign would be NaN.)
struct ExpScale {
  float hi, lo;
};
static inline ExpScale exp_scale(double temp) {
  const double c = 1.4426950408889634 / temp;
  ExpScale e;
  e.hi = (float)c;
  e.lo = (float)(c - (double)e.hi);
  return e;
}
__device__ __forceinline__ float exp_t(float t, ExpScale c) {
  return __builtin_amdgcn_exp2f(__builtin_fmaf(t, c.hi, fmaxf(t, -1e30f) * c.lo));
}

// Sum of exponentials relative to a maximum.  The maximum starts at the lowest finite value, so that no -inf is subtracted from
// -inf: a row of -inf ends with s = 0 (log-sum-exp -inf), a row of the type's lowest value counts as any other row.  A NaN or
// +inf among the elements leaves s = NaN.  s is fp32 inside a thread (at most a few hundred terms), double across threads.
struct MaxSum {
  float m, s;
};
template <class D>
__device__ __forceinline__ void fold(MaxSum& a, const RowVec<D>& v, ExpScale c) {
  float f[D::EPV], top = -FLT_MAX;
#pragma unroll
  for (int i = 0; i < D::EPV; ++i) {
    f[i] = D::get(v.e[i]);
    top = fmaxf(top, f[i]);
  }
  if (top > a.m) {
    a.s *= exp_t(a.m - top, c);
    a.m = top;
  }
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < D::EPV; ++i) s += exp_t(f[i] - a.m, c);
  a.s += s;
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
__device__ __forceinline__ MaxSumD block_max_sum(MaxSum a, ExpScale c, double* red) {
  const float wm = wave_max(a.m);
  const double ws = wave_sum_d((double)(a.s * exp_t(a.m - wm, c)));
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

// Key whose unsigned order is the order of the values: -0 equals +0, NaN (any) above +inf.
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t b = __builtin_bit_cast(uint32_t, v + 0.0f);
  const uint32_t k = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return v != v ? 0xffffffffu : k;
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
