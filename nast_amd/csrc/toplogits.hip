// A teacher's top logits and the distillation loss of a student against them (forward and backward).
//
//   top:      the k largest logits of a row with their ids, and lse = log sum_v exp(x_v / T)
//   distill:  p_j = exp(t_j / T - c) over the used slots j of the teacher's list, q = softmax(z / T),
//             loss = sum_j p_j (log p_j - log q_{id_j})  [+ p_r (log p_r - log q_r)]
//             dz_v = g / T * (q_v - [rest] p_r q_v / q_r - sum_{j: id_j = v} p_j)
//             p_r = 1 - sum p_j and q_r = sum of q over the tokens no used slot names: the rest bucket (only with the teacher's lse)
#include "rowvec.h"

// ---------------------------------------------------------------------------------------------
// top logits
// ---------------------------------------------------------------------------------------------
#define TOP_MAX_K 256

// One workgroup per row.  Elements are ordered by (key, lower id first): the 64-bit number key << 32 | ~id differs for any two
// elements of a row.  The k-th largest such number is found by bisection over its bits, counting the elements at or above a
// candidate; the k elements at or above it are collected and ranked by comparison with each other.
template <class D>
__global__ __launch_bounds__(256) void nast_top_logits_kernel(const typename D::store* __restrict__ x, nast_rows xr,
                                                              typename D::store* __restrict__ values, int64_t* __restrict__ index,
                                                              float* __restrict__ lse, int V, int k, double inv_temp, ExpScale c) {
  __shared__ double red[8];
  __shared__ int cnt[4];
  __shared__ uint64_t cand[TOP_MAX_K];
  __shared__ int n_cand;
  const int64_t r = blockIdx.x;
  const typename D::store* p = x + row_offset(r, xr);
  const RowSlots<D> rs(p, 0, V);
  MaxSum a{-FLT_MAX, 0.f};
  for (int s = threadIdx.x; s < rs.n; s += 256) fold<D>(a, rs.load(p, s), c);
  const MaxSumD t = block_max_sum<256>(a, c, red);
  if (threadIdx.x == 0) lse[r] = (float)(t.m * inv_temp + log(t.s));

  uint64_t bound = 0;
  for (int bit = 63; bit >= 0; --bit) {
    const uint64_t mid = bound | (1ull << bit);
    int n = 0;
    for (int s = threadIdx.x; s < rs.n; s += 256) {
      const RowVec<D> v = rs.load(p, s);
#pragma unroll
      for (int i = 0; i < D::EPV; ++i) {
        const int e = rs.elem(s) + i;
        const uint64_t o = ((uint64_t)order_key(D::get(v.e[i])) << 32) | (uint32_t)~e;
        n += (e >= 0 && e < V && o >= mid) ? 1 : 0;
      }
    }
    n = (int)wave_sum((float)n);       // <= V < 2^24 per wavefront: exact in fp32
    __syncthreads();
    if ((threadIdx.x & 63) == 0) cnt[threadIdx.x >> 6] = n;
    __syncthreads();
    if (cnt[0] + cnt[1] + cnt[2] + cnt[3] >= k) bound = mid;
  }
  if (threadIdx.x == 0) n_cand = 0;
  __syncthreads();
  for (int s = threadIdx.x; s < rs.n; s += 256) {
    const RowVec<D> v = rs.load(p, s);
#pragma unroll
    for (int i = 0; i < D::EPV; ++i) {
      const int e = rs.elem(s) + i;
      const uint64_t o = ((uint64_t)order_key(D::get(v.e[i])) << 32) | (uint32_t)~e;
      if (e >= 0 && e < V && o >= bound) {
        const int at = atomicAdd(&n_cand, 1);
        if (at < TOP_MAX_K) cand[at] = o;
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < k; i += 256) {
    const uint64_t o = cand[i];
    int rank = 0;
    for (int j = 0; j < k; ++j) rank += cand[j] > o ? 1 : 0;
    const int e = (int)~(uint32_t)o;
    index[r * k + rank] = e;
    values[r * k + rank] = p[e];
  }
}

extern "C" int64_t nast_top_logits_workspace_bytes(int rows, int V, int k, int dtype) { return 0; }

extern "C" int nast_top_logits(const void* x, int dtype, nast_rows xr, void* values, int64_t* index, float* lse, int rows, int V,
                               int k, double temp, void* workspace, void* stream) {
  NAST_REQUIRE(row_dtype_ok(dtype), "nast_top_logits: unknown dtype %d", dtype);
  NAST_REQUIRE(rows >= 0 && V >= 1 && V < (1 << 24), "nast_top_logits: bad sizes rows=%d V=%d", rows, V);
  NAST_REQUIRE(k >= 1 && k <= TOP_MAX_K && k <= V, "nast_top_logits: k=%d must lie in [1, %d] and not exceed V=%d", k, TOP_MAX_K, V);
  NAST_REQUIRE(temp > 0 && temp < 1e30, "nast_top_logits: temperature must be > 0 and finite");
  if (rows == 0) return NAST_OK;
  NAST_REQUIRE(rows < (1 << 24), "nast_top_logits: too many rows (%d)", rows);
  NAST_REQUIRE(x && values && index && lse, "nast_top_logits: NULL pointer");
  NAST_REQUIRE(row_aligned(x, dtype) && row_aligned(values, dtype), "nast_top_logits: misaligned pointer");
  nast_prof_before(2, (hipStream_t)stream);
  NAST_ROW_DTYPE(dtype, hipLaunchKernelGGL((nast_top_logits_kernel<D>), dim3(rows), dim3(256), 0, (hipStream_t)stream,
                                           (const typename D::store*)x, xr, (typename D::store*)values, index, lse, V, k, 1.0 / temp,
                                           exp_scale(temp)));
  nast_prof_after(2, (hipStream_t)stream, (double)row_size(dtype) * rows * (double)V);
  NAST_CHECK_LAUNCH("nast_top_logits");
  return NAST_OK;
}

// ---------------------------------------------------------------------------------------------
// distillation
// ---------------------------------------------------------------------------------------------
#define DISTILL_MAX_K 256
#define DISTILL_SLOTS (DISTILL_MAX_K / 64)
#define DISTILL_CHUNK 32768       // elements one workgroup reads at most: 4 KB of membership bits
#define DISTILL_NO_ID 0xffffffffu

// teacher's list in its own type
__device__ __forceinline__ float teacher_logit(const void* t, int dtype, int64_t i) {
  if (dtype == NAST_F32) return ((const float*)t)[i];
  if (dtype == NAST_BF16) return (float)((const __bf16*)t)[i];
  return (float)((const _Float16*)t)[i];
}
// a slot counts when its id is one of the student's and the teacher gives it a probability
__device__ __forceinline__ bool slot_used(int64_t id, float t, int V) { return id >= 0 && id < V && t != -INFINITY; }

// What the backward pass needs of a row: the rest's maximum and the factor of its exponentials, and the normalisers of
// log q_v = (z_v - M) / T - L and log p_j = (t_j - C) / T - c (in two parts: next to a logit of -3e38 a logarithm of a sum would be lost).
struct DistillStats {
  double m_rest, coef, M, L, C, c;
};

// The end of a row's forward pass by ONE wavefront; slot j = lane + 64 * i.  m, s: maximum and exponential sum of the tokens that no
// used slot names.  Everything here is in double: the loss is a small difference of terms near 1 (with one slot of p = 0.01 and
// q = 0.0075 it is 3e-4, while p_r log p_r alone is rounded by 6e-8 in fp32), and it is a few slots per row.
template <class D>
__device__ void distill_finish(int64_t r, MaxSumD rest, const typename D::store* p, const void* t, int t_dtype,
                               const int64_t* idx, int K, const float* lse_t, float* loss, DistillStats* stats, int V, double it,
                               uint32_t* ids) {
  const int lane = threadIdx.x & 63;
  float tj[DISTILL_SLOTS], zj[DISTILL_SLOTS];
  uint32_t id[DISTILL_SLOTS];
  float tm = -FLT_MAX, zm = -FLT_MAX;
#pragma unroll
  for (int i = 0; i < DISTILL_SLOTS; ++i) {
    const int j = lane + 64 * i;
    id[i] = DISTILL_NO_ID;
    tj[i] = zj[i] = -INFINITY;
    if (j < K) {
      const int64_t v = idx[r * K + j];
      const float tv = teacher_logit(t, t_dtype, r * K + j);
      if (slot_used(v, tv, V)) {
        id[i] = (uint32_t)v;
        tj[i] = tv;
        zj[i] = D::get(p[v]);
        tm = fmaxf(tm, tv);
        zm = fmaxf(zm, zj[i]);
      }
      ids[j] = id[i];
    }
  }
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  tm = wave_max(tm);
  const double M = fmax(rest.m, (double)wave_max(zm));
  double ts = 0, zs = 0, any = 0;
#pragma unroll
  for (int i = 0; i < DISTILL_SLOTS; ++i) {
    if (id[i] == DISTILL_NO_ID) continue;
    any = 1;
    ts += exp(((double)tj[i] - tm) * it);
    bool first = true;                       // an id named twice is one token of the student's
    for (int j = 0; j < lane + 64 * i; ++j) first = first && ids[j] != id[i];
    if (first) zs += exp(((double)zj[i] - M) * it);
  }
  ts = wave_sum_d(ts);
  zs = wave_sum_d(zs);
  any = wave_max_d(any);
  const double sr = rest.s * exp((rest.m - M) * it);
  const double L = log(zs + sr), C = lse_t ? 0.0 : (double)tm, c = lse_t ? (double)lse_t[r] : log(ts);
  double sum_p = 0, l = 0;
#pragma unroll
  for (int i = 0; i < DISTILL_SLOTS; ++i) {
    if (id[i] == DISTILL_NO_ID) continue;
    const double logp = ((double)tj[i] - C) * it - c, pj = exp(logp);
    sum_p += pj;
    if (pj != 0) l += pj * (logp - (((double)zj[i] - M) * it - L));
  }
  sum_p = wave_sum_d(sum_p);
  l = wave_sum_d(l);
  const double log_qr = (rest.m - M) * it + log(rest.s) - L, qr = exp(log_qr);
  double pr = lse_t ? fmax(1.0 - sum_p, 0.0) : 0.0;
  if (rest.s == 0) pr = 0;                   // no token of the student's is left for the bucket
  if (pr > 0) l += pr * (log(pr) - log_qr);
  if (lane == 0) {
    DistillStats o;
    o.m_rest = rest.m;
    o.M = M;
    o.L = L;
    o.C = C;
    o.c = c;
    // q_v - p_r q_v / q_r = exp((z_v - m_r) / T) / s_r * (q_r - p_r): no quotient of small numbers; 0 for a row without a list and
    // for one without a rest, NaN for a row of nothing but -inf
    o.coef = any == 0 ? 0.0 : rest.s == 0 ? (L > -INFINITY ? 0.0 : NAN) : (qr - pr) / rest.s;
    stats[r] = o;
    loss[r] = any == 0 ? 0.f : (float)l;
  }
}

// One workgroup per chunk of a row: (max, exponential sum) of the tokens that no used slot names.  The named ones are marked in LDS,
// one bit per element, and left out of both: their terms are added in double at the end, and q_r is a sum and no difference.
template <class D, bool SPLIT>
__global__ __launch_bounds__(256) void nast_top_distill_fwd_kernel(const typename D::store* __restrict__ x, nast_rows xr,
                                                                   const void* __restrict__ t, int t_dtype,
                                                                   const int64_t* __restrict__ idx, int K,
                                                                   const float* __restrict__ lse_t, float* __restrict__ loss,
                                                                   DistillStats* __restrict__ stats, MaxSumD* __restrict__ parts, int V,
                                                                   int chunk, int n_chunk, double it, ExpScale c) {
  __shared__ uint32_t bits[DISTILL_CHUNK / 32 + 1];
  __shared__ double red[8];
  __shared__ uint32_t ids[DISTILL_MAX_K];
  const int64_t r = blockIdx.x / n_chunk;
  const int lo = (int)(blockIdx.x % n_chunk) * chunk, hi = min(V, lo + chunk);
  const typename D::store* p = x + row_offset(r, xr);
  const RowSlots<D> rs(p, lo, hi);
  for (int w = threadIdx.x; w < (hi - rs.first + 31) / 32; w += 256) bits[w] = 0;
  __syncthreads();
  for (int j = threadIdx.x; j < K; j += 256) {
    const int64_t id = idx[r * K + j];
    if (id >= lo && id < hi && slot_used(id, teacher_logit(t, t_dtype, r * K + j), V))
      atomicOr(&bits[(id - rs.first) >> 5], 1u << ((id - rs.first) & 31));
  }
  __syncthreads();
  MaxSum a{-FLT_MAX, 0.f};
  for (int s = threadIdx.x; s < rs.n; s += 256) {
    RowVec<D> v = rs.load(p, s);
    const uint32_t named = bits[s * D::EPV >> 5] >> (s * D::EPV & 31);
    if (named & ((1u << D::EPV) - 1)) {
#pragma unroll
      for (int i = 0; i < D::EPV; ++i)
        if (named >> i & 1) v.e[i] = D::put(-INFINITY);
    }
    fold<D>(a, v, c);
  }
  const MaxSumD rest = block_max_sum<256>(a, c, red);
  if (SPLIT) {
    if (threadIdx.x == 0) parts[blockIdx.x] = rest;
  } else if (threadIdx.x < 64) {
    distill_finish<D>(r, rest, p, t, t_dtype, idx, K, lse_t, loss, stats, V, it, ids);
  }
}

// one wavefront per row joins the chunks
template <class D>
__global__ __launch_bounds__(64) void nast_top_distill_join_kernel(const typename D::store* __restrict__ x, nast_rows xr,
                                                                   const void* __restrict__ t, int t_dtype,
                                                                   const int64_t* __restrict__ idx, int K,
                                                                   const float* __restrict__ lse_t, float* __restrict__ loss,
                                                                   DistillStats* __restrict__ stats, const MaxSumD* __restrict__ parts,
                                                                   int V, int n_chunk, double it) {
  __shared__ uint32_t ids[DISTILL_MAX_K];
  const int64_t r = blockIdx.x;
  MaxSumD rest{-FLT_MAX, 0};
  double m = -FLT_MAX, s = 0;
  for (int i = threadIdx.x; i < n_chunk; i += 64) m = fmax(m, parts[r * n_chunk + i].m);
  rest.m = wave_max_d(m);
  for (int i = threadIdx.x; i < n_chunk; i += 64) {
    const MaxSumD q = parts[r * n_chunk + i];
    s += q.s * exp((q.m - rest.m) * it);
  }
  rest.s = wave_sum_d(s);
  distill_finish<D>(r, rest, x + row_offset(r, xr), t, t_dtype, idx, K, lse_t, loss, stats, V, it, ids);
}

// One workgroup per chunk of a row: the rest's gradient everywhere, then, behind a barrier, the value of each named token over it.
template <class D>
__global__ __launch_bounds__(256) void nast_top_distill_bwd_kernel(const float* __restrict__ g, const typename D::store* __restrict__ x,
                                                                   nast_rows xr, const void* __restrict__ t, int t_dtype,
                                                                   const int64_t* __restrict__ idx, int K,
                                                                   const DistillStats* __restrict__ stats,
                                                                   typename D::store* __restrict__ gx, nast_rows gxr, int V, int chunk,
                                                                   int n_chunk, double it, ExpScale c) {
  __shared__ uint32_t ids[DISTILL_MAX_K];
  __shared__ float ts[DISTILL_MAX_K];
  const int64_t r = blockIdx.x / n_chunk;
  const int lo = (int)(blockIdx.x % n_chunk) * chunk, hi = min(V, lo + chunk);
  const typename D::store* p = x + row_offset(r, xr);
  typename D::store* o = gx + row_offset(r, gxr);
  const DistillStats st = stats[r];
  const double gr = (double)g[r] * it;
  uint32_t id = DISTILL_NO_ID;
  float z = 0.f;
  if ((int)threadIdx.x < K) {
    const int64_t v = idx[r * K + threadIdx.x];
    const float tv = teacher_logit(t, t_dtype, r * K + threadIdx.x);
    if (slot_used(v, tv, V) && v >= lo && v < hi) {
      id = (uint32_t)v;
      z = D::get(p[v]);
    }
    ids[threadIdx.x] = id;
    ts[threadIdx.x] = tv;
  }
  // a factor of 0 (a row without a list, a row of no weight) writes zeros whatever the logits hold
  const float F = gr == 0 ? 0.f : (float)(gr * st.coef), m = (float)st.m_rest;
  const RowSlots<D> rs(o, lo, hi);
  const bool same = ((reinterpret_cast<uintptr_t>(p) ^ reinterpret_cast<uintptr_t>(o)) & 15) == 0;
  for (int s = threadIdx.x; s < rs.n; s += 256) {
    RowVec<D> v;
    if (same) {
      v = rs.load(p, s);
    } else {
#pragma unroll
      for (int i = 0; i < D::EPV; ++i) {
        const int e = rs.elem(s) + i;
        v.e[i] = e >= lo && e < hi ? p[e] : D::put(0.f);
      }
    }
#pragma unroll
    for (int i = 0; i < D::EPV; ++i) v.e[i] = D::put(F == 0.f ? 0.f : exp_t(D::get(v.e[i]) - m, c) * F);
    if (rs.whole(s)) {
      *reinterpret_cast<uint4*>(o + rs.elem(s)) = v.raw;
    } else {
#pragma unroll
      for (int i = 0; i < D::EPV; ++i) {
        const int e = rs.elem(s) + i;
        if (e >= lo && e < hi) o[e] = v.e[i];
      }
    }
  }
  __syncthreads();
  if (id == DISTILL_NO_ID) return;
  double pj = 0;
  bool first = true;
  for (int j = 0; j < K; ++j) {
    if (ids[j] != id) continue;
    first = first && j >= (int)threadIdx.x;
    pj += exp(((double)ts[j] - st.C) * it - st.c);
  }
  if (first) o[id] = D::put(gr == 0 ? 0.f : (float)(gr * (exp(((double)z - st.M) * it - st.L) - pj)));
}

static int distill_check(const char* name, int dtype, int t_dtype, int K, int rows, int V, double temp) {
  NAST_REQUIRE(row_dtype_ok(dtype) && row_dtype_ok(t_dtype), "%s: unknown dtype", name);
  NAST_REQUIRE(rows >= 0 && V >= 1 && V < (1 << 24), "%s: bad sizes rows=%d V=%d", name, rows, V);
  NAST_REQUIRE(K >= 1 && K <= DISTILL_MAX_K, "%s: a list has 1 to %d slots, not %d", name, DISTILL_MAX_K, K);
  NAST_REQUIRE(temp > 0 && temp < 1e30, "%s: temperature must be > 0 and finite", name);
  return NAST_OK;
}
static int distill_chunk(int rows, int V) { return V < DISTILL_CHUNK - 8 ? V : DISTILL_CHUNK - 8; }

extern "C" int64_t nast_top_distill_workspace_bytes(int rows, int V, int dtype) {
  const int chunk = distill_chunk(rows, V), n = (V + chunk - 1) / chunk;
  return n > 1 ? (int64_t)rows * n * (int64_t)sizeof(MaxSumD) : 0;
}

extern "C" int nast_top_distill_fwd(const void* x, int dtype, nast_rows xr, const void* t, int t_dtype, const int64_t* idx, int K,
                                    const float* lse_t, float* loss, double* stats, int rows, int V, double temp, void* workspace,
                                    void* stream) {
  if (int rc = distill_check("nast_top_distill_fwd", dtype, t_dtype, K, rows, V, temp)) return rc;
  if (rows == 0) return NAST_OK;
  NAST_REQUIRE(x && t && idx && loss && stats, "nast_top_distill_fwd: NULL pointer");
  NAST_REQUIRE(row_aligned(x, dtype) && row_aligned(t, t_dtype), "nast_top_distill_fwd: misaligned pointer");
  const int chunk = distill_chunk(rows, V), n = (V + chunk - 1) / chunk;
  NAST_REQUIRE(n == 1 || workspace, "nast_top_distill_fwd: NULL workspace");
  NAST_REQUIRE((int64_t)rows * n < (1 << 24), "nast_top_distill_fwd: too many rows (%d)", rows);
  hipStream_t s = (hipStream_t)stream;
  DistillStats* st = (DistillStats*)stats;
  MaxSumD* parts = (MaxSumD*)workspace;
  const ExpScale c = exp_scale(temp);
  nast_prof_before(2, s);
  NAST_ROW_DTYPE(dtype, {
    const typename D::store* xp = (const typename D::store*)x;
    if (n == 1) {
      hipLaunchKernelGGL((nast_top_distill_fwd_kernel<D, false>), dim3(rows), dim3(256), 0, s, xp, xr, t, t_dtype, idx, K, lse_t, loss, st,
                         parts, V, chunk, n, 1.0 / temp, c);
    } else {
      hipLaunchKernelGGL((nast_top_distill_fwd_kernel<D, true>), dim3(rows * n), dim3(256), 0, s, xp, xr, t, t_dtype, idx, K, lse_t, loss,
                         st, parts, V, chunk, n, 1.0 / temp, c);
      hipLaunchKernelGGL((nast_top_distill_join_kernel<D>), dim3(rows), dim3(64), 0, s, xp, xr, t, t_dtype, idx, K, lse_t, loss, st, parts,
                         V, n, 1.0 / temp);
    }
  });
  nast_prof_after(2, s, (double)row_size(dtype) * rows * (double)V);
  NAST_CHECK_LAUNCH("nast_top_distill_fwd");
  return NAST_OK;
}

extern "C" int nast_top_distill_bwd(const float* g, const void* x, int dtype, nast_rows xr, const void* t, int t_dtype,
                                    const int64_t* idx, int K, const double* stats, void* gx, nast_rows gxr, int rows, int V, double temp,
                                    void* stream) {
  if (int rc = distill_check("nast_top_distill_bwd", dtype, t_dtype, K, rows, V, temp)) return rc;
  if (rows == 0) return NAST_OK;
  NAST_REQUIRE(g && x && t && idx && stats && gx, "nast_top_distill_bwd: NULL pointer");
  NAST_REQUIRE(x != gx, "nast_top_distill_bwd: in-place not supported");
  NAST_REQUIRE(row_aligned(x, dtype) && row_aligned(gx, dtype) && row_aligned(t, t_dtype), "nast_top_distill_bwd: misaligned pointer");
  const int chunk = V < 8192 ? V : 8192, n = (V + chunk - 1) / chunk;
  NAST_REQUIRE((int64_t)rows * n < (1 << 24), "nast_top_distill_bwd: too many rows (%d)", rows);
  nast_prof_before(2, (hipStream_t)stream);
  NAST_ROW_DTYPE(dtype, hipLaunchKernelGGL((nast_top_distill_bwd_kernel<D>), dim3(rows * n), dim3(256), 0, (hipStream_t)stream, g,
                                           (const typename D::store*)x, xr, t, t_dtype, idx, K, (const DistillStats*)stats,
                                           (typename D::store*)gx, gxr, V, chunk, n, 1.0 / temp, exp_scale(temp)));
  nast_prof_after(2, (hipStream_t)stream, 2.0 * row_size(dtype) * rows * (double)V);
  NAST_CHECK_LAUNCH("nast_top_distill_bwd");
  return NAST_OK;
}
