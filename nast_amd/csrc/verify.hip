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

#define VERIFY_MAX_V (1 << 20)
#define VERIFY_MAX_DRAFTS 1024
// Sums are off by ROW_SUM_REL each (see MaxSum): a draft's two probabilities are told apart where they differ by more than both, and by
// what doubles add.
#define VERIFY_CLOSE 1.1e-5
// What the fp32 probabilities of the draw are off by, relative: the row's sum 5e-6, an exponent of -a before and of up to a + 20 after the
// sum's logarithm is added ln 2 * 2^-24 * (4 a + 40) = 1.65e-7 a + 1.65e-6, the instruction 1.2e-7; a score's difference, sum with its bound,
// reciprocal and product 3e-7.  7.1e-6 in all, and 1.65e-7 a.
#define VERIFY_REL 7.5e-6f
#define VERIFY_REL_EXP 2e-7f

struct VerifyArgs {
  const void *target, *draft;     // draft NULL: no probabilities
  int64_t t_bs, t_rs, q_bs, q_rs; // strides of batch and row
  const int64_t *tokens, *lengths;
  const float *u, *E;
  int64_t *out, *accepted;
  int B, N, V;
  double it;                      // 1 / T
  float c;
  int chunk, n_chunk;             // of the rows' sums
  int race_chunk, n_race;         // of the draw
  MaxSumD* parts;                 // [B * (2 N + 1)][n_chunk]: target rows first, then draft rows
  struct VerifyBest* best;        // [B][n_race]
  int* ended;                     // [B]
};

// the running argmax of the draw: score, bounds of the exact score, the largest upper bound of any other, where
struct VerifyBest {
  float score, lower, upper, other;
  int at;
};
__device__ __forceinline__ void best_merge(VerifyBest& a, const VerifyBest b) {
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
  return (const typename D::store*)A.target + b * A.t_bs + i * A.t_rs;
}
template <class D>
__device__ __forceinline__ const typename D::store* draft_row(const VerifyArgs& A, int b, int i) {
  return (const typename D::store*)A.draft + b * A.q_bs + i * A.q_rs;
}
__device__ __forceinline__ int draft_length(const VerifyArgs& A, int b) {
  if (!A.lengths) return A.N;
  const int64_t n = A.lengths[b];
  return n < 0 ? 0 : n > A.N ? A.N : (int)n;
}
// a row without a distribution (a NaN, a +inf, nothing but -inf) has s = 0
__device__ __forceinline__ MaxSumD proper(MaxSumD t) {
  if (!(t.s > 0 && t.m <= (double)FLT_MAX)) t.s = 0;
  return t;
}

// a row's sum in double, by the whole workgroup; U loads in flight
template <class D, int NT, int U>
__device__ double row_sum_exact(const VerifyArgs& A, const typename D::store* p, double m, double* red) {
  double s = 0;
  for (int e = threadIdx.x; e < A.V; e += U * NT) {
    float z[U];
#pragma unroll
    for (int i = 0; i < U; ++i) z[i] = D::get(p[min(e + i * NT, A.V - 1)]);
#pragma unroll
    for (int i = 0; i < U; ++i) s += e + i * NT < A.V ? exp(((double)z[i] - m) * A.it) : 0.0;
  }
  s = wave_sum_d(s);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  s = 0;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) s += red[i];
  return s;
}

// p_i(d_i) and q_i(d_i); a token that is not one, or a row without a distribution: 0
struct VerifyPair {
  double p, q;
};
template <class D>
__device__ __forceinline__ VerifyPair drafted(const VerifyArgs& A, int b, int i, const MaxSumD& p, const MaxSumD& q) {
  const int64_t d = A.tokens[(int64_t)b * A.N + i];
  if (d < 0 || d >= A.V || p.s == 0 || q.s == 0) return {0, 0};
  VerifyPair r;
  r.p = exp(((double)D::get(target_row<D>(A, b, i)[d]) - p.m) * A.it) / p.s;
  r.q = A.draft ? exp(((double)D::get(draft_row<D>(A, b, i)[d]) - q.m) * A.it) / q.s : 1.0;
  return r;
}
__device__ __forceinline__ bool stands(const VerifyPair& r, float u) { return r.q > 0 && (double)u * r.q < r.p; }
__device__ __forceinline__ bool too_close(const VerifyPair& r, float u) {
  return r.p > 0 && r.q > 0 && fabs((double)u * r.q - r.p) <= VERIFY_CLOSE * r.p;
}
// the same decision with sums in double, by the whole workgroup
template <class D, int NT, int U>
__device__ bool stands_exact(const VerifyArgs& A, int b, int i, MaxSumD p, MaxSumD q, double* red) {
  p.s = row_sum_exact<D, NT, U>(A, target_row<D>(A, b, i), p.m, red);
  if (A.draft) q.s = row_sum_exact<D, NT, U>(A, draft_row<D>(A, b, i), q.m, red);
  return stands(drafted<D>(A, b, i, p, q), A.u[(int64_t)b * A.N + i]);
}

// What the token at place `place` is drawn from: p = exp((z - m) / T) / s, less q where the draft at that place was refused
struct VerifyDraw {
  MaxSumD p, q;
  int place, one;                 // one: the refused draft's token where it came without probabilities, else -1
  bool minus_q;
};
__device__ __forceinline__ VerifyDraw draw_of(const VerifyArgs& A, int b, int place, int len, const MaxSumD& p, const MaxSumD& q) {
  VerifyDraw w{p, q, place, -1, false};
  if (place < len) {
    if (A.draft) {
      w.minus_q = q.s > 0;
    } else {
      const int64_t d = A.tokens[(int64_t)b * A.N + place];
      w.one = d >= 0 && d < A.V ? (int)d : -1;
    }
  }
  return w;
}

// the best of the wavefront's, in every lane.  (Of equal scores any: neither is certain then.)
__device__ __forceinline__ VerifyBest best_of_wave(const VerifyBest& a) {
  VerifyBest r;
  r.score = wave_max(a.score);
  const int l = __ffsll((unsigned long long)__ballot(a.score == r.score)) - 1;
  r.lower = __shfl(a.lower, l, 64);
  r.upper = __shfl(a.upper, l, 64);
  r.at = __shfl(a.at, l, 64);
  r.other = wave_max((threadIdx.x & 63) == l ? a.other : fmaxf(a.other, a.upper));
  return r;
}

// Argmax of w / E over [lo, hi) in fp32 with error bounds, by the whole workgroup.  Most elements are told apart by one logarithm:
// log2(p / E), not less than the logarithm of their score, against that of the best lower bound their wavefront has seen (less 0.01, a
// thousand times what the two are off by).  Only what passes is looked at closer, and of the first vectors, where nothing has been seen
// yet, each lane's most promising element before the others.
template <class D, int NT>
__device__ VerifyBest race(const VerifyArgs& A, int b, const VerifyDraw& w, int lo, int hi, VerifyBest* lds) {
  VerifyBest a{0.f, 0.f, 0.f, 0.f, 0x7fffffff};
  if (w.p.s > 0) {
    const typename D::store* p = target_row<D>(A, b, w.place);
    const typename D::store* q = w.minus_q ? draft_row<D>(A, b, w.place) : nullptr;
    const float* E = A.E + (int64_t)b * A.V;
    const float pm = (float)w.p.m, qm = (float)w.q.m, ps = -(float)log2(w.p.s), qs = w.minus_q ? -(float)log2(w.q.s) : 0.f;
    const float slope = -VERIFY_REL_EXP * A.c, far = -200.f / A.c;
    float seen = 0.f;
    float seen_log = -INFINITY;
    auto log_score = [&](float zp, float en) { return __builtin_fmaf(zp - pm, A.c, ps) - __builtin_amdgcn_logf(en); };
    auto look = [&](float zp, float zq, float en, int e) {
      const float tp = zp - pm, tq = zq - qm, pv = __builtin_amdgcn_exp2f(__builtin_fmaf(tp, A.c, ps));
      const float qv = q ? __builtin_amdgcn_exp2f(__builtin_fmaf(tq, A.c, qs)) : 0.f;
      const float d = pv - qv, inv = __builtin_amdgcn_rcpf(en);
      // (below 2^-150 the bound is the absolute one; an exponent of -inf would make it 0 * inf)
      const float ep = pv * __builtin_fmaf(fmaxf(tp, far), slope, VERIFY_REL), eq = q ? qv * __builtin_fmaf(fmaxf(tq, far), slope, VERIFY_REL) : 0.f;
      const float err = 1e-37f + (ep + eq);
      const float upper = (d + err) * inv;
      if (upper > seen && e != w.one) {
        if (en >= FLT_MIN) best_merge(a, {d * inv, (d - err) * inv, upper, 0.f, e});
        else a.other = INFINITY;                                  // no reciprocal in fp32: left to the draw in double
      }
    };
    const RowSpan16<D> rs(p, lo, hi);
    const int edge = rs.edge(threadIdx.x), at_edge = edge >= 0 ? edge : lo;
    const float edge_p = D::get(p[at_edge]), edge_q = D::get((q ? q : p)[at_edge]), edge_E = E[at_edge];
    constexpr int W = D::EPV / 4;                               // vectors of draws to one of logits
    struct Slot {
      RowVec<D> p, q;
      RowVec<RowF32> E[W];
    };
    auto load = [&](int s) {
      const int at = rs.elem(min(s, rs.n - 1));
      Slot v;
      v.p = vec_load<D>(p + at);
      v.q = vec_load_any<D>((q ? q : p) + at);
#pragma unroll
      for (int j = 0; j < W; ++j) v.E[j] = vec_load_any<RowF32>(E + at + 4 * j);
      return v;
    };
    if (rs.n > 0) {
      Slot v = load(threadIdx.x);
#pragma unroll 1
      for (int b0 = 0; b0 < rs.n; b0 += NT) {
        const int s = b0 + (int)threadIdx.x;
        const Slot next = load(s + NT);
        float sc[D::EPV];
#pragma unroll
        for (int j = 0; j < D::EPV; ++j) {                      // (a draw of 0: +inf; NaN for one that never wins)
          sc[j] = log_score(v.p.get(j), v.E[j / 4].get(j % 4));
          if (s >= rs.n) sc[j] = -INFINITY;
        }
#pragma unroll 1
        while (true) {                                          // each lane's most promising element, as long as any lane has one
          float top = sc[0];
#pragma unroll
          for (int j = 1; j < D::EPV; ++j) top = fmaxf(top, sc[j]);
          const bool hit = top > -INFINITY && top >= seen_log;
          if (!__ballot(hit)) break;
          float zp = 0.f, zq = 0.f, en = 1.f;
          int first = -1;
#pragma unroll
          for (int j = 0; j < D::EPV; ++j) {
            const bool is = first < 0 && sc[j] == top;
            zp = is ? v.p.get(j) : zp;
            zq = is ? v.q.get(j) : zq;
            en = is ? v.E[j / 4].get(j % 4) : en;
            first = is ? j : first;
            sc[j] = is ? -INFINITY : sc[j];
          }
          if (hit) look(zp, zq, en, rs.elem(s) + first);
          seen = wave_max(fmaxf(seen, a.lower));
          seen_log = __builtin_amdgcn_logf(seen) - 0.01f;
        }
        v = next;
      }
    }
    if (edge >= 0 && log_score(edge_p, edge_E) >= seen_log) look(edge_p, edge_q, edge_E, edge);
  }
  a = best_of_wave(a);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = a;
  __syncthreads();
  return best_of_wave((threadIdx.x & 63) < NT / 64 ? lds[threadIdx.x & 63] : VerifyBest{0.f, 0.f, 0.f, 0.f, 0x7fffffff});
}

// The draw in double, ties to the lowest id.  Where nothing is left of p - q (rounding, u >= 1) it is made from p.  `lower`: what the
// best score reaches for certain; elements that fall short of it by the measure of race() are passed over.
template <class D, int NT, int U>
__device__ int race_exact(const VerifyArgs& A, int b, const VerifyDraw& w, float lower, double* red, int* ired) {
  if (w.p.s == 0) return -1;
  const typename D::store* p = target_row<D>(A, b, w.place);
  const typename D::store* q = w.minus_q ? draft_row<D>(A, b, w.place) : nullptr;
  const float* E = A.E + (int64_t)b * A.V;
  // (scores of p alone are compared without its sum)
  const double ps = q ? row_sum_exact<D, NT, U>(A, p, w.p.m, red) : w.p.s, qs = q ? row_sum_exact<D, NT, U>(A, q, w.q.m, red) : 1;
  const float pm = (float)w.p.m, log_s = -(float)log2(w.p.s);
  for (int whole = 0; whole < 2; ++whole) {
    const float least = whole || !(lower > 0) ? -INFINITY : __builtin_amdgcn_logf(lower) - 0.01f;
    double best = 0;
    int at = 0x7fffffff;
    auto look = [&](float z, float en, int e) {
      if (__builtin_fmaf(z - pm, A.c, log_s) - __builtin_amdgcn_logf(en) < least) return;
      double v = exp(((double)z - w.p.m) * A.it) / ps;
      if (!whole) {
        if (q) v -= exp(((double)D::get(q[e]) - w.q.m) * A.it) / qs;
        if (e == w.one) v = 0;
      }
      if (!(v > 0)) return;
      const double score = v / (double)en;
      if (score > best || (score == best && e < at)) {
        best = score;
        at = e;
      }
    };
    for (int e = threadIdx.x; e < A.V; e += U * NT) {
      float z[U], en[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int at = min(e + i * NT, A.V - 1);
        z[i] = D::get(p[at]);
        en[i] = E[at];
      }
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (e + i * NT < A.V) look(z[i], en[i], e + i * NT);
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
    for (int i = 0; i < NT / 64; ++i)
      if (red[i] > best || (red[i] == best && ired[i] < at)) {
        best = red[i];
        at = ired[i];
      }
    __syncthreads();
    if (best > 0) return at;
  }
  return -1;
}

// ---------------------------------------------------------------------------------------------
// Rows are read in rounds of places, each a launch over (sequence, row, chunk); a round leaves out the sequences that a clear refusal of
// an earlier one has ended, whose further rows nothing needs.  Then place and draw: by one workgroup a sequence, or in chunks, each
// workgroup finding the place for itself, and a launch that joins them.
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ MaxSumD row_pair(const VerifyArgs& A, int row) {
  const MaxSumD* q = A.parts + (int64_t)row * A.n_chunk;
  if (A.n_chunk == 1) return proper(q[0]);
  // the maximum first: each chunk's sum is then brought to it by one exponential, whatever order the maxima come in
  MaxSumD o[4], t;                                             // four loads in flight
#pragma unroll
  for (int j = 0; j < 4; ++j) o[j] = q[min(j, A.n_chunk - 1)];
  t.m = fmax(fmax(o[0].m, o[1].m), fmax(o[2].m, o[3].m));
  for (int i = 4; i < A.n_chunk; i += 4) {
    double m[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) m[j] = q[min(i + j, A.n_chunk - 1)].m;
    t.m = fmax(t.m, fmax(fmax(m[0], m[1]), fmax(m[2], m[3])));
  }
  t.s = 0;
  for (int i = 0; i < A.n_chunk; i += 4) {
    if (i) {
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = q[min(i + j, A.n_chunk - 1)];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i + j < A.n_chunk) t.s += o[j].s * (double)exp_t((float)(o[j].m - t.m), A.c);
  }
  return proper(t);
}

// the draft at place i of sequence b, from the rows' sums
template <class D>
__device__ __forceinline__ VerifyPair drafted_at(const VerifyArgs& A, int b, int i) {
  return drafted<D>(A, b, i, row_pair(A, b * (A.N + 1) + i), A.draft ? row_pair(A, A.B * (A.N + 1) + b * A.N + i) : MaxSumD{0, 1});
}

// Between two rounds, one wavefront a sequence: whether a draft before place i0 is clearly refused.  5 us, latency; without it each
// workgroup of the round would find that out for itself.
template <class D>
__global__ __launch_bounds__(64) void nast_verify_ended_kernel(VerifyArgs A, int i0) {
  const int b = blockIdx.x, len = draft_length(A, b);
  bool ended = false;
  for (int i = threadIdx.x; i < i0 && i < len; i += 64) {
    const VerifyPair r = drafted_at<D>(A, b, i);
    const float u = A.u[(int64_t)b * A.N + i];
    ended = ended || (!stands(r, u) && !too_close(r, u));
  }
  const uint64_t any = __ballot(ended);
  if (threadIdx.x == 0) A.ended[b] = any != 0 || len < i0;
}

// One workgroup a chunk of a row: maximum and exponential sum.  Bound by memory: 268 MB of 256 sequences' first two places x 131072 bf16 in
// 52 us (5.1 TB/s); sequences that have ended leave at once.
template <class D>
__global__ __launch_bounds__(256) void nast_verify_rows_kernel(VerifyArgs A, int i0, int n_target, int n_draft) {
  __shared__ double red[8];
  const int k = blockIdx.x / A.n_chunk, ch = blockIdx.x % A.n_chunk, lo = ch * A.chunk, hi = min(A.V, lo + A.chunk);
  const int b = k / (n_target + n_draft), j = k % (n_target + n_draft), len = draft_length(A, b);
  const bool is_target = j < n_target;
  const int i = i0 + (is_target ? j : j - n_target);
  if (is_target ? i > len : i >= len) return;
  if (i0 > 0 && A.ended[b]) return;
  const MaxSum a = span_max_sum<D, 256>(is_target ? target_row<D>(A, b, i) : draft_row<D>(A, b, i), lo, hi, A.c);
  const MaxSumD t = block_max_sum<256>(a, A.c, red);
  if (threadIdx.x == 0) A.parts[(int64_t)(is_target ? b * (A.N + 1) + i : A.B * (A.N + 1) + b * A.N + i) * A.n_chunk + ch] = t;
}

// How many drafts of sequence b stand, by the whole workgroup.  Each wavefront does the same: lane = place.  (Sums behind a clear refusal
// may never have been written; what is made of them is not looked at.)  A decision that comes too close is made in double, or, with
// U = 0, the answer is -1.
template <class D, int NT, int U>
__device__ int places(const VerifyArgs& A, int b, int len, double* red) {
  const int lane = threadIdx.x & 63;
  for (int base = 0; base < len; base += 64) {
    const int i = base + lane;
    bool ok = true, near = false;
    if (i < len) {
      const VerifyPair r = drafted_at<D>(A, b, i);
      const float u = A.u[(int64_t)b * A.N + i];
      ok = stands(r, u);
      near = too_close(r, u);
    }
    uint64_t no = __ballot(!ok), close = __ballot(near);
    while (close) {
      const int at = __ffsll((unsigned long long)close) - 1;
      if (no & ((1ull << at) - 1)) break;                  // a clear refusal comes first
      if constexpr (U == 0) {
        return -1;
      } else {
        close &= close - 1;
        const int j = base + at;
        const MaxSumD p = row_pair(A, b * (A.N + 1) + j), q = A.draft ? row_pair(A, A.B * (A.N + 1) + b * A.N + j) : MaxSumD{0, 1};
        const bool yes = stands_exact<D, NT, U>(A, b, j, p, q, red);
        no = yes ? no & ~(1ull << at) : no | (1ull << at);
      }
    }
    if (no) return base + __ffsll((unsigned long long)no) - 1;
  }
  return len;
}

template <class D>
__device__ __forceinline__ VerifyDraw draw_at(const VerifyArgs& A, int b, int place, int len) {
  return draw_of(A, b, place, len, row_pair(A, b * (A.N + 1) + place),
                 A.draft && place < len ? row_pair(A, A.B * (A.N + 1) + b * A.N + place) : MaxSumD{0, 0});
}

// the end of a sequence, by the whole workgroup
template <class D, int NT, int U>
__device__ void finish(const VerifyArgs& A, int b, int place, int len, const VerifyBest& a, double* red, int* ired) {
  const int token = a.lower > a.other ? a.at : race_exact<D, NT, U>(A, b, draw_at<D>(A, b, place, len), a.lower, red, ired);
  for (int i = threadIdx.x; i <= A.N; i += NT)
    A.out[(int64_t)b * (A.N + 1) + i] = i < place ? A.tokens[(int64_t)b * A.N + i] : i == place ? token : -1;
  if (threadIdx.x == 0) A.accepted[b] = place;
}

// One workgroup a sequence does everything behind the sums.  A chain of latencies: draft, its logits, place, p, q and E at that place,
// scores, maxima; 13 us at 1 x 32000 bf16, 10 at 128 x 9600 fp32, of which 4 go before the place is known.
template <class D, int NT>
__global__ __launch_bounds__(NT) void nast_verify_draw_kernel(VerifyArgs A) {
  __shared__ double red[NT / 64];
  __shared__ int ired[NT / 64];
  __shared__ VerifyBest lds[NT / 64];
  const int b = blockIdx.x, len = draft_length(A, b), place = places<D, NT, 1>(A, b, len, red);
  finish<D, NT, 1>(A, b, place, len, race<D, NT>(A, b, draw_at<D>(A, b, place, len), 0, A.V, lds), red, ired);
}

// One workgroup a chunk of a sequence.  Decisions that are too close are left to the join: the arithmetic in double would cost this
// kernel, which has to fill the card, 22 registers.  (Where one of 256 x 131072 comes too close, about one call in a hundred, the call
// takes 130 us more.)  Bound by memory where there are rows enough: 256 x 131072 bf16, 268 MB of p, q and E in 48 us (5.6 TB/s).
template <class D>
__global__ __launch_bounds__(256) void nast_verify_chunk_kernel(VerifyArgs A) {
  __shared__ VerifyBest lds[4];
  const int b = blockIdx.x / A.n_race, lo = (int)(blockIdx.x % A.n_race) * A.race_chunk, hi = min(A.V, lo + A.race_chunk);
  const int len = draft_length(A, b), place = places<D, 256, 0>(A, b, len, nullptr);
  if (place >= 0) {
    const VerifyBest a = race<D, 256>(A, b, draw_at<D>(A, b, place, len), lo, hi, lds);
    if (threadIdx.x == 0) A.best[blockIdx.x] = a;
  }
  if (lo == 0 && threadIdx.x == 0) A.accepted[b] = place;
}

template <class D>
__global__ __launch_bounds__(1024) void nast_verify_join_kernel(VerifyArgs A) {
  __shared__ double red[16];
  __shared__ int ired[16];
  __shared__ VerifyBest lds[16];
  const int b = blockIdx.x, len = draft_length(A, b);
  int place = (int)A.accepted[b];
  VerifyBest a{0.f, 0.f, 0.f, 0.f, 0x7fffffff};
  if (place >= 0) {
    for (int i = 0; i < A.n_race; ++i) {
      const VerifyBest o = A.best[(int64_t)b * A.n_race + i];
      best_merge(a, o);
    }
  } else {
    place = places<D, 1024, 4>(A, b, len, red);
    a = race<D, 1024>(A, b, draw_at<D>(A, b, place, len), 0, A.V, lds);
  }
  finish<D, 1024, 4>(A, b, place, len, a, red, ired);
}

// A further round costs two launches (10 us) and saves the rows of the sequences that have ended, half of them perhaps: it has to have
// 128 MB of rows (20 us).  So many places at least has each, the first two or more, the next ones twice as many as the one before; where
// less is left than that it is taken along.  256 x 8 drafts x 131072 bf16 in rounds of 2, 4, 3 places 196 us, at once 244; 512 x 32 x 9600
// fp32 120 and 234; 64 x 8 x 131072 in rounds of 4 and 5 74, at once 80, in the three rounds 83.
#define VERIFY_ROUND_BYTES (128 << 20)
static int verify_round(const VerifyArgs& A, int dtype, int i0, int last) {
  const int64_t place = (int64_t)A.B * A.V * row_size(dtype) * (A.draft ? 2 : 1), least = (VERIFY_ROUND_BYTES + place - 1) / place;
  const int left = A.N + 1 - i0;
  const int64_t n = least > 2 * last ? least : 2 * last;
  return n + least >= left ? left : (int)n;
}
// Chunks: rows at most 2^15 elements, the draw up to there in one workgroup (a join of its own costs more than chunks save: 1 x 4 drafts x
// 32000 bf16 17.8 us in one workgroup, 20.3 in chunks; 100 x 2 x 30000 22 either way).
static void verify_plan(VerifyArgs& A, int dtype) {
  const int most = 1 << 15, first = verify_round(A, dtype, 0, 1);
  A.n_chunk = row_chunks((int64_t)A.B * first * (A.draft ? 2 : 1), A.V, most, 1 << 13);
  A.chunk = (A.V + A.n_chunk - 1) / A.n_chunk;
  A.n_race = A.V <= most ? 1 : row_chunks(A.B, A.V, most, 1 << 13);
  A.race_chunk = (A.V + A.n_race - 1) / A.n_race;
}

extern "C" int64_t nast_verify_draft_workspace_bytes(int B, int N, int V, int dtype) {
  if (B < 1 || N < 0 || N > VERIFY_MAX_DRAFTS || V < 1 || V > VERIFY_MAX_V || !row_dtype_ok(dtype)) return 0;
  int64_t most = 0;
  for (int draft = 0; draft < 2; ++draft) {                   // (with and without draft logits)
    VerifyArgs A;
    A.B = B;
    A.N = N;
    A.V = V;
    A.draft = draft ? &A : nullptr;
    verify_plan(A, dtype);
    const int64_t n = (int64_t)B * (2 * N + 1) * A.n_chunk * (int64_t)sizeof(MaxSumD) + (int64_t)B * A.n_race * (int64_t)sizeof(VerifyBest) +
                      (int64_t)B * (int64_t)sizeof(int);
    most = n > most ? n : most;
  }
  return most;
}

extern "C" int nast_verify_draft(const void* target, int64_t target_bs, int64_t target_rs, const void* draft, int64_t draft_bs,
                                 int64_t draft_rs, int dtype, const int64_t* tokens, const float* u, const float* E,
                                 const int64_t* lengths, int64_t* out, int64_t* accepted, int B, int N, int V, double temp,
                                 void* workspace, void* stream) {
  NAST_REQUIRE(row_dtype_ok(dtype), "nast_verify_draft: unknown dtype %d", dtype);
  NAST_REQUIRE(B >= 0 && B < (1 << 20) && N >= 0 && N <= VERIFY_MAX_DRAFTS && V >= 1 && V <= VERIFY_MAX_V,
               "nast_verify_draft: bad sizes B=%d N=%d V=%d", B, N, V);
  NAST_REQUIRE(temp > 1e-30 && temp < 1e30, "nast_verify_draft: temperature must lie between 1e-30 and 1e30");
  if (B == 0) return NAST_OK;
  NAST_REQUIRE(target && E && out && accepted && workspace && (N == 0 || (tokens && u)),
               "nast_verify_draft: NULL pointer");
  NAST_REQUIRE(row_aligned(target, dtype) && row_aligned(draft, dtype), "nast_verify_draft: misaligned pointer");
  VerifyArgs A;
  A.target = target;
  A.draft = N ? draft : nullptr;
  A.t_bs = target_bs;
  A.t_rs = target_rs;
  A.q_bs = draft_bs;
  A.q_rs = draft_rs;
  A.tokens = tokens;
  A.lengths = lengths;
  A.u = u;
  A.E = E;
  A.out = out;
  A.accepted = accepted;
  A.B = B;
  A.N = N;
  A.V = V;
  A.it = 1.0 / temp;
  A.c = exp_scale(temp);
  hipStream_t s = (hipStream_t)stream;
  verify_plan(A, dtype);
  NAST_REQUIRE((int64_t)B * (2 * N + 1) * A.n_chunk < (1 << 24) && (int64_t)B * A.n_race < (1 << 22), "nast_verify_draft: too many rows (%d)", B);
  nast_prof_before(2, s);
  A.parts = (MaxSumD*)workspace;
  A.best = (VerifyBest*)(A.parts + (int64_t)B * (2 * N + 1) * A.n_chunk);
  A.ended = (int*)(A.best + (int64_t)B * A.n_race);
  NAST_ROW_DTYPE(dtype, {
    for (int i0 = 0, n = 1; i0 <= N; i0 += n) {
      n = verify_round(A, dtype, i0, n);
      if (i0) hipLaunchKernelGGL((nast_verify_ended_kernel<D>), dim3(B), dim3(64), 0, s, A, i0);
      const int n_draft = !A.draft ? 0 : n < N - i0 ? n : N - i0;
      hipLaunchKernelGGL((nast_verify_rows_kernel<D>), dim3(B * (n + n_draft) * A.n_chunk), dim3(256), 0, s, A, i0, n, n_draft);
    }
    if (A.n_race == 1) {
      // (512 threads where the workgroups do not fill the card twice: 128 x 9600 fp32 27 us, with 256 threads 29; 600 x 30000 bf16 67 and 60)
      if (B <= 512) hipLaunchKernelGGL((nast_verify_draw_kernel<D, 512>), dim3(B), dim3(512), 0, s, A);
      else hipLaunchKernelGGL((nast_verify_draw_kernel<D, 256>), dim3(B), dim3(256), 0, s, A);
    } else {
      hipLaunchKernelGGL((nast_verify_chunk_kernel<D>), dim3(B * A.n_race), dim3(256), 0, s, A);
      hipLaunchKernelGGL((nast_verify_join_kernel<D>), dim3(B), dim3(1024), 0, s, A);
    }
  });
  nast_prof_after(2, s, (double)V * B * (row_size(dtype) * (A.draft ? 2.0 * N + 1 : N + 1.0) + 4.0));
  NAST_CHECK_LAUNCH("nast_verify_draft");
  return NAST_OK;
}
