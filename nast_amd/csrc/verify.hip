// Verification of drafted tokens (speculative sampling) from given random numbers.
//
// Sequence b has drafts d_0 .. d_{n-1}, drawn from q_i = softmax(draft[b, i] / T) (or given without probabilities: q_i is one at d_i),
// and target rows p_i = softmax(target[b, i] / T), i = 0 .. n.  d_i is accepted while  q_i(d_i) > 0 and u_i * q_i(d_i) < p_i(d_i).  At the
// first refusal i the token is drawn from (p_i - q_i)+, behind the last draft from p_n: argmax_v w_v / E_v with Exp(1) draws E_v is a
// draw from w / sum(w), needs no sum and no prefix, and hardly ever depends on a rounding.  The tokens so drawn follow p.
//
// A decision is a comparison, so its rounding decides which token comes out.  The fp32 arithmetic carries bounds of its error; where a
// comparison is closer than they are, it is made again in double over the whole row.
#include "rowvec.h"

#define VERIFY_CHUNK 32768
#define VERIFY_MAX_DRAFTS 1024
#define VERIFY_REL 1e-5           // fp32 exponentials, sums and products here are within this, relative (see exp_t: ~1e-6)

struct VerifyRows {               // rows [.., V] of a [B, n, V] tensor
  int64_t bs, rs;
};

struct VerifyArgs {
  const void *target, *draft;     // draft NULL: no probabilities
  VerifyRows tr, qr;
  const int64_t *tokens, *lengths;
  const float *u, *E;
  int64_t u_bs, E_bs, tok_bs;
  int64_t *out, *accepted;
  int B, N, V, chunk, n_chunk;
  double it;                      // 1 / T
  float c;
  MaxSumD* parts;                 // [B * (2 N + 1)][n_chunk]: target rows first, then draft rows
  struct VerifyBest* best;        // [B][n_chunk]
};

// the running argmax of the race: score, bounds of the exact score, the largest upper bound of any other, where
struct VerifyBest {
  float score, lower, upper, other;
  int at;
};
__device__ __forceinline__ void best_merge(VerifyBest& a, const VerifyBest& b) {
  const float other = fmaxf(a.other, b.other);
  if (b.score > a.score || (b.score == a.score && b.at < a.at)) {
    const float beaten = a.upper;
    a = b;
    a.other = fmaxf(other, beaten);
  } else {
    a.other = fmaxf(other, b.upper);
  }
}

template <class D>
__device__ __forceinline__ const typename D::store* target_row(const VerifyArgs& A, int b, int i) {
  return (const typename D::store*)A.target + b * A.tr.bs + i * A.tr.rs;
}
template <class D>
__device__ __forceinline__ const typename D::store* draft_row(const VerifyArgs& A, int b, int i) {
  return (const typename D::store*)A.draft + b * A.qr.bs + i * A.qr.rs;
}
__device__ __forceinline__ int draft_length(const VerifyArgs& A, int b) {
  if (!A.lengths) return A.N;
  const int64_t n = A.lengths[b];
  return n < 0 ? 0 : n > A.N ? A.N : (int)n;
}

// ---- (max, sum of exponentials) of every row that can be asked for ------------------------------------------------------
template <class D>
__global__ __launch_bounds__(256) void nast_verify_lse_kernel(VerifyArgs A) {
  __shared__ double red[8];
  const int row = blockIdx.x / A.n_chunk, lo = (int)(blockIdx.x % A.n_chunk) * A.chunk, hi = min(A.V, lo + A.chunk);
  const int n_target = A.B * (A.N + 1);
  const bool is_target = row < n_target;
  const int b = is_target ? row / (A.N + 1) : (row - n_target) / A.N, i = is_target ? row % (A.N + 1) : (row - n_target) % A.N;
  const int len = draft_length(A, b);
  if (is_target ? i > len : i >= len) return;
  const typename D::store* p = is_target ? target_row<D>(A, b, i) : draft_row<D>(A, b, i);
  const MaxSum a = span_max_sum<D, 256>(p, lo, hi, A.c);
  const MaxSumD t = block_max_sum<256>(a, A.c, red);
  if (threadIdx.x == 0) A.parts[blockIdx.x] = t;
}

// a row's pair; a row without a distribution (a NaN, a +inf, nothing but -inf) has s = 0
__device__ __forceinline__ MaxSumD row_pair(const VerifyArgs& A, int row) {
  const MaxSumD* q = A.parts + (int64_t)row * A.n_chunk;
  MaxSumD t = q[0];
  for (int i = 1; i < A.n_chunk; ++i) {
    const MaxSumD o = q[i];
    const double m = fmax(t.m, o.m);
    t.s = t.s * exp((t.m - m) * A.it) + o.s * exp((o.m - m) * A.it);
    t.m = m;
  }
  if (!(t.s > 0 && t.m <= (double)FLT_MAX)) t.s = 0;
  return t;
}

// the same sum in double, by the whole workgroup of 256
template <class D>
__device__ double row_sum_exact(const VerifyArgs& A, const typename D::store* p, double m, double* red) {
  double s = 0;
  for (int e = threadIdx.x; e < A.V; e += 256) s += exp(((double)D::get(p[e]) - m) * A.it);
  s = wave_sum_d(s);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

struct VerifyDecision {
  int accepted, len;
};
// p_i(d_i) and q_i(d_i); a token that is not one, or a row without a distribution: 0
struct VerifyPair {
  double p, q;
};
template <class D>
__device__ __forceinline__ VerifyPair drafted(const VerifyArgs& A, int b, int i, const MaxSumD& p, const MaxSumD& q) {
  const int64_t d = A.tokens[b * A.tok_bs + i];
  if (d < 0 || d >= A.V || p.s == 0 || q.s == 0) return {0, 0};
  VerifyPair r;
  r.p = exp(((double)D::get(target_row<D>(A, b, i)[d]) - p.m) * A.it) / p.s;
  r.q = A.draft ? exp(((double)D::get(draft_row<D>(A, b, i)[d]) - q.m) * A.it) / q.s : 1.0;
  return r;
}
__device__ __forceinline__ bool stands(const VerifyPair& r, float u) { return r.q > 0 && (double)u * r.q < r.p; }

// How many drafts of sequence b stand, by the whole workgroup.  Each wavefront does the same: lane = position.
template <class D>
__device__ VerifyDecision decide(const VerifyArgs& A, int b, double* red) {
  const int len = draft_length(A, b), lane = threadIdx.x & 63;
  const int q0 = A.B * (A.N + 1) + b * A.N;
  for (int base = 0; base < len; base += 64) {
    const int i = base + lane;
    bool ok = true, near = false;
    if (i < len) {
      const MaxSumD p = row_pair(A, b * (A.N + 1) + i);
      const MaxSumD q = A.draft ? row_pair(A, q0 + i) : MaxSumD{0, 1};
      const VerifyPair r = drafted<D>(A, b, i, p, q);
      const float u = A.u[b * A.u_bs + i];
      ok = stands(r, u);
      near = r.p > 0 && r.q > 0 && fabs((double)u * r.q - r.p) <= VERIFY_REL * r.p;
    }
    uint64_t no = __ballot(!ok), close = __ballot(near);
    while (close) {
      const int at = __ffsll((unsigned long long)close) - 1;
      if (no & ((1ull << at) - 1)) break;                  // a clear refusal comes first
      close &= close - 1;
      const int j = base + at;
      MaxSumD p = row_pair(A, b * (A.N + 1) + j), q = A.draft ? row_pair(A, q0 + j) : MaxSumD{0, 1};
      p.s = row_sum_exact<D>(A, target_row<D>(A, b, j), p.m, red);
      if (A.draft) q.s = row_sum_exact<D>(A, draft_row<D>(A, b, j), q.m, red);
      const bool yes = stands(drafted<D>(A, b, j, p, q), A.u[b * A.u_bs + j]);
      no = yes ? no & ~(1ull << at) : no | (1ull << at);
    }
    if (no) return {base + __ffsll((unsigned long long)no) - 1, len};
  }
  return {len, len};
}

// the row drawn from: p = exp((z - m) / T) / s, less q where the draft at that place was refused
struct VerifyDraw {
  MaxSumD p, q;
  int64_t one;                    // the refused draft's token where it came without probabilities, else -1
  bool minus_q;
};
template <class D>
__device__ __forceinline__ VerifyDraw draw_of(const VerifyArgs& A, int b, const VerifyDecision& d) {
  VerifyDraw w;
  w.p = row_pair(A, b * (A.N + 1) + d.accepted);
  w.q = {0, 0};
  w.one = -1;
  w.minus_q = false;
  if (d.accepted < d.len) {
    if (A.draft) {
      w.q = row_pair(A, A.B * (A.N + 1) + b * A.N + d.accepted);
      w.minus_q = w.q.s > 0;
    } else {
      w.one = A.tokens[b * A.tok_bs + d.accepted];
    }
  }
  return w;
}

// argmax of w / E over [lo, hi) in fp32 with error bounds, by the whole workgroup
template <class D>
__device__ VerifyBest race(const VerifyArgs& A, int b, int place, const VerifyDraw& w, int lo, int hi, VerifyBest* lds) {
  VerifyBest a{0.f, 0.f, 0.f, 0.f, 0x7fffffff};
  if (w.p.s > 0) {
    const typename D::store* p = target_row<D>(A, b, place);
    const typename D::store* q = w.minus_q ? draft_row<D>(A, b, place) : nullptr;
    const float* E = A.E + b * A.E_bs;
    const float pm = (float)w.p.m, ps = (float)(1.0 / w.p.s), qm = (float)w.q.m, qs = w.minus_q ? (float)(1.0 / w.q.s) : 0.f;
    for (int e = lo + threadIdx.x; e < hi; e += 256) {
      if (e == w.one) continue;
      const float pv = exp_t(D::get(p[e]) - pm, A.c) * ps, qv = q ? exp_t(D::get(q[e]) - qm, A.c) * qs : 0.f;
      const float inv = 1.0f / E[e], d = pv - qv, err = (pv + qv) * (float)VERIFY_REL + 1e-37f;
      best_merge(a, {d * inv, (d - err) * inv, (d + err) * inv, 0.f, e});
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    VerifyBest x;
    x.score = __shfl_xor(a.score, o, 64);
    x.lower = __shfl_xor(a.lower, o, 64);
    x.upper = __shfl_xor(a.upper, o, 64);
    x.other = __shfl_xor(a.other, o, 64);
    x.at = __shfl_xor(a.at, o, 64);
    best_merge(a, x);
  }
  const int wv = threadIdx.x >> 6;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[wv] = a;
  __syncthreads();
  VerifyBest r = lds[0];
  for (int i = 1; i < 4; ++i) best_merge(r, lds[i]);
  return r;
}

// The draw in double, ties to the lowest id.  Where nothing is left of p - q (rounding, u >= 1) it is made from p.
template <class D>
__device__ int race_exact(const VerifyArgs& A, int b, int place, VerifyDraw w, double* red, int* ired) {
  if (w.p.s == 0) return -1;
  const typename D::store* p = target_row<D>(A, b, place);
  const typename D::store* q = w.minus_q ? draft_row<D>(A, b, place) : nullptr;
  const double ps = row_sum_exact<D>(A, p, w.p.m, red), qs = q ? row_sum_exact<D>(A, q, w.q.m, red) : 1;
  for (int whole = 0; whole < 2; ++whole) {
    double best = 0;
    int at = 0x7fffffff;
    for (int e = threadIdx.x; e < A.V; e += 256) {
      double v = exp(((double)D::get(p[e]) - w.p.m) * A.it) / ps;
      if (!whole) {
        if (q) v -= exp(((double)D::get(q[e]) - w.q.m) * A.it) / qs;
        if (e == w.one) v = 0;
      }
      if (!(v > 0)) continue;
      const double score = v / (double)A.E[b * A.E_bs + e];
      if (score > best) {
        best = score;
        at = e;
      }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const double s2 = __shfl_xor(best, o, 64);
      const int a2 = __shfl_xor(at, o, 64);
      if (s2 > best || (s2 == best && a2 < at)) {
        best = s2;
        at = a2;
      }
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
      red[threadIdx.x >> 6] = best;
      ired[threadIdx.x >> 6] = at;
    }
    __syncthreads();
    for (int i = 0; i < 4; ++i)
      if (red[i] > best || (red[i] == best && ired[i] < at)) {
        best = red[i];
        at = ired[i];
      }
    __syncthreads();
    if (best > 0) return at;
  }
  return -1;
}

template <class D>
__global__ __launch_bounds__(256) void nast_verify_race_kernel(VerifyArgs A) {
  __shared__ double red[4];
  __shared__ VerifyBest lds[4];
  const int b = blockIdx.x / A.n_chunk, lo = (int)(blockIdx.x % A.n_chunk) * A.chunk, hi = min(A.V, lo + A.chunk);
  const VerifyDecision d = decide<D>(A, b, red);
  const VerifyBest a = race<D>(A, b, d.accepted, draw_of<D>(A, b, d), lo, hi, lds);
  if (threadIdx.x == 0) {
    A.best[blockIdx.x] = a;
    if (lo == 0) A.accepted[b] = d.accepted;
  }
}

template <class D>
__global__ __launch_bounds__(256) void nast_verify_join_kernel(VerifyArgs A) {
  __shared__ double red[4];
  __shared__ int ired[4];
  const int b = blockIdx.x;
  const VerifyDecision d{(int)A.accepted[b], draft_length(A, b)};
  VerifyBest a = A.best[(int64_t)b * A.n_chunk];
  for (int i = 1; i < A.n_chunk; ++i) best_merge(a, A.best[(int64_t)b * A.n_chunk + i]);
  int token = a.at;
  if (!(a.lower > a.other)) token = race_exact<D>(A, b, d.accepted, draw_of<D>(A, b, d), red, ired);
  for (int i = threadIdx.x; i <= A.N; i += 256)
    A.out[(int64_t)b * (A.N + 1) + i] = i < d.accepted ? A.tokens[b * A.tok_bs + i] : i == d.accepted ? token : -1;
}

static int verify_chunks(int V) { return (V + VERIFY_CHUNK - 1) / VERIFY_CHUNK; }

extern "C" int64_t nast_verify_draft_workspace_bytes(int B, int N, int V, int dtype) {
  const int64_t n = verify_chunks(V);
  return ((int64_t)B * (2 * N + 1) * (int64_t)sizeof(MaxSumD) + (int64_t)B * (int64_t)sizeof(VerifyBest)) * n;
}

extern "C" int nast_verify_draft(const void* target, int64_t target_bs, int64_t target_rs, const void* draft, int64_t draft_bs,
                                 int64_t draft_rs, int dtype, const int64_t* tokens, const float* u, const float* E,
                                 const int64_t* lengths, int64_t* out, int64_t* accepted, int B, int N, int V, double temp,
                                 void* workspace, void* stream) {
  NAST_REQUIRE(row_dtype_ok(dtype), "nast_verify_draft: unknown dtype %d", dtype);
  NAST_REQUIRE(B >= 0 && N >= 0 && N <= VERIFY_MAX_DRAFTS && V >= 1 && V < (1 << 24), "nast_verify_draft: bad sizes B=%d N=%d V=%d", B, N, V);
  NAST_REQUIRE(temp > 0 && temp < 1e30, "nast_verify_draft: temperature must be > 0 and finite");
  if (B == 0) return NAST_OK;
  NAST_REQUIRE(target && E && out && accepted && workspace && (N == 0 || (tokens && u)), "nast_verify_draft: NULL pointer");
  NAST_REQUIRE(row_aligned(target, dtype) && row_aligned(draft, dtype), "nast_verify_draft: misaligned pointer");
  VerifyArgs A;
  A.target = target;
  A.draft = N ? draft : nullptr;
  A.tr = {target_bs, target_rs};
  A.qr = {draft_bs, draft_rs};
  A.tokens = tokens;
  A.lengths = lengths;
  A.u = u;
  A.E = E;
  A.u_bs = A.tok_bs = N;
  A.E_bs = V;
  A.out = out;
  A.accepted = accepted;
  A.B = B;
  A.N = N;
  A.V = V;
  A.chunk = VERIFY_CHUNK;
  A.n_chunk = verify_chunks(V);
  A.it = 1.0 / temp;
  A.c = exp_scale(temp);
  A.parts = (MaxSumD*)workspace;
  const int64_t rows = (int64_t)B * (A.draft ? 2 * N + 1 : N + 1);
  A.best = (VerifyBest*)(A.parts + (int64_t)B * (2 * N + 1) * A.n_chunk);
  NAST_REQUIRE(rows * A.n_chunk < (1 << 24), "nast_verify_draft: too many rows (%lld)", (long long)rows);
  hipStream_t s = (hipStream_t)stream;
  nast_prof_before(2, s);
  NAST_ROW_DTYPE(dtype, {
    hipLaunchKernelGGL((nast_verify_lse_kernel<D>), dim3((unsigned)(rows * A.n_chunk)), dim3(256), 0, s, A);
    hipLaunchKernelGGL((nast_verify_race_kernel<D>), dim3(B * A.n_chunk), dim3(256), 0, s, A);
    hipLaunchKernelGGL((nast_verify_join_kernel<D>), dim3(B), dim3(256), 0, s, A);
  });
  nast_prof_after(2, s, (double)V * (row_size(dtype) * (double)rows + 4.0 * B));
  NAST_CHECK_LAUNCH("nast_verify_draft");
  return NAST_OK;
}
