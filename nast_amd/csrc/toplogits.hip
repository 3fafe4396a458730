// A teacher's top logits and the distillation loss of a student against them (forward and backward).
//
//   top:      the k largest logits of a row with their ids, and lse = log sum_v exp(x_v / T)
//   distill:  p_j = exp(t_j / T - c) over the used slots j of the teacher's list, q = softmax(z / T),
//             loss = sum_j p_j (log p_j - log q_{id_j})  [+ p_r (log p_r - log q_r)]
//             dz_v = g / T * (w q_v - [rest] p_r q_v / q_r - sum_{j: id_j = v} p_j)
//             p_r = max(0, 1 - sum p_j) and q_r = sum of q over the tokens no used slot names: the rest bucket (only with the teacher's
//             lse, and only where q_r > 0);  w = sum p_j + p_r of the bucket kept: every term holds the normaliser of log q once.  w is 1
//             but where the list is more than one (its logits rounded, its lse not; an id in two slots) or the bucket has nothing
#include "rowvec.h"

// ---------------------------------------------------------------------------------------------
// top logits
// ---------------------------------------------------------------------------------------------
#define TOP_MAX_K 256
#define TOP_MAX_V (1 << 20)
#define TOP_MAX_LIST 16384        // entries the join of a row's chunks takes

// Elements are ordered by value, ties to the lower id: entry = key << 32 | ~id is one 64-bit number per element, no two alike, 0 is
// no element.
__device__ __forceinline__ uint64_t top_entry(float f, int e) { return ((uint64_t)order_key(f) << 32) | (uint32_t)~e; }
__device__ __forceinline__ int entry_id(uint64_t o) { return (int)~(uint32_t)o; }

// n distinct entries in LDS: each goes to out(rank among all, entry) where the rank is below k.  A rank is a count of larger entries.
// In workgroups of 1024, which few rows take, as many as 16 threads share an entry's comparisons (256 x 32000 fp32 k 256 17.4 -> 15.5 us);
// with 256, which fill the card, one makes them all (4096 x 9600 fp16 k 200 60 us, shared 76).
template <int NT, class F>
__device__ __forceinline__ void rank_out(const uint64_t* cand, int n, int k, F&& out) {
  if constexpr (NT == 1024) {
    int shift = 0;
    while (shift < 4 && n << (shift + 1) <= NT) ++shift;
    const int share = 1 << shift, part = threadIdx.x & (share - 1);
    for (int i = threadIdx.x >> shift; i < n; i += NT >> shift) {
      const uint64_t o = cand[i];
      int rank = 0;
#pragma unroll 8
      for (int j = part; j < n; j += share) rank += cand[j] > o ? 1 : 0;
      for (int m = 1; m < share; m <<= 1) rank += __shfl_xor(rank, m, 64);
      if (part == 0 && rank < k) out(rank, o);
    }
  } else {
    for (int i = threadIdx.x; i < n; i += NT) {
      const uint64_t o = cand[i];
      int rank = 0;
#pragma unroll 8
      for (int j = 0; j < n; ++j) rank += cand[j] > o ? 1 : 0;
      if (rank < k) out(rank, o);
    }
  }
}

template <int NT>
__device__ __forceinline__ int block_count(int n, int* cnt) {   // n <= 2^16 a thread; two barriers
  n = (int)wave_sum((float)n);                                  // <= 2^22: exact in fp32
  __syncthreads();
  if ((threadIdx.x & 63) == 0) cnt[threadIdx.x >> 6] = n;
  __syncthreads();
  int t = 0;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) t += cnt[i];
  return t;
}

// By one wavefront: bound[0] = a value that at least kk of the 64 * N group maxima reach (and, where one is found, not more than
// 9/8 kk + 8), bound[1] = the largest.  Bisection on the upper half of the order key.
template <int N>
__device__ __forceinline__ void group_bound(const float* gmax, int kk, float* bound) {
  const int lane = threadIdx.x & 63;
  float m = -INFINITY, least = INFINITY;
  uint32_t key[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float f = gmax[i * 64 + lane];
    m = fmaxf(m, f);
    least = fminf(least, f);
    key[i] = order_key(f) >> 16;
  }
  m = wave_max(m);
  least = -wave_max(-least);
  uint32_t b0 = order_key(least) >> 16, b1 = (order_key(m) >> 16) + 1;
  while (b0 + 1 < b1) {                                        // (false at once where nothing but signalling NaNs came: least > m)
    const uint32_t mid = (b0 + b1) >> 1;
    int n = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) n += __popcll(__ballot(key[i] >= mid));
    if (n >= kk) {
      b0 = mid;
      if (n <= kk + kk / 8 + 8) break;
    } else {
      b1 = mid;
    }
  }
  b0 <<= 16;
  if (lane == 0) {
    bound[0] = b0 < 0x00800000u ? -INFINITY : key_value(b0);   // (keys below that of -inf are of no number)
    bound[1] = fmaxf(m, -FLT_MAX);
  }
}

// What a chunk leaves beside its list: maximum and exponential sum, and a bound that at least k of its elements reach (-inf: unknown).
struct TopPart {
  double m, s;
  float bound;
};

// One workgroup of NT threads per chunk of a row, the chunk in registers: NV vectors a thread (and an edge element), read from memory
// once.
//
// The k-th largest of the maxima of disjoint groups of elements is a lower bound of the k-th largest element.  Each thread keeps the
// maximum of each of its vectors; their maxima over a thread (or, for k > 64, over a quarter of its vectors, with up to two of them of
// its elements) are the groups, and one wavefront finds a bound among them (group_bound).  Vectors whose maximum reaches the bound go to
// LDS, each wavefront's to a place of its own, where its lanes look at their elements one by one; what reaches the bound (a little more
// than k elements where they lie at random: 350 +- 19 of a large chunk for k = 256, a quarter of them to a wavefront) is ranked by
// counting.  Where more than `cap` elements of a wavefront reach it (many equal values, e.g. a constant row), or the row holds a NaN, the
// k-th key is found exactly instead, by bisection with a count over the chunk, and equal elements are taken in the order of their ids.
//
// Bound by memory on long rows in numbers (16384 x 9600 fp32 105 us, 6.0 TB/s; 2048 x 131072 bf16 113 us with the join, 4.8 TB/s, where
// the unpacking and exponentials of 16-bit elements take as long as their load), by latency below: 8 x 32000 fp32 9 us.
template <class D, int NT, int NV>
__global__ __launch_bounds__(NT, 4) void nast_top_chunk_kernel(const typename D::store* __restrict__ x, nast_rows xr,
                                                             typename D::store* __restrict__ values, int64_t* __restrict__ index,
                                                             float* __restrict__ lse, uint64_t* __restrict__ lists,
                                                             TopPart* __restrict__ parts, int V, int k, int cap, int len, int chunk, int n_chunk,
                                                             double inv_temp, float c) {
  constexpr int W = NT / 64, G = NT == 256 ? 4 : 1;
  __shared__ float gmax[NT * G];
  extern __shared__ uint4 vec_data[];                           // for `cap` candidates a wavefront: vector, entry, slot
  uint64_t* cand = (uint64_t*)(vec_data + W * cap);
  int* vec_slot = (int*)(cand + W * cap);
  __shared__ double red[W];
  __shared__ int cnt[W];
  __shared__ float bound[2];
  __shared__ int n_cand;
  const int64_t r = blockIdx.x / n_chunk;
  const int tid = threadIdx.x, lane = tid & 63, lo = (int)(blockIdx.x % n_chunk) * chunk, hi = min(V, lo + chunk);
  const typename D::store* p = x + row_offset(r, xr);
  const RowSpan16<D> rs(p, lo, hi);
  const int kk = min(k, hi - lo);
  const int ee = rs.edge(tid);
  const typename D::store edge = p[ee >= 0 ? ee : lo];
  RowVec<D> v[NV];
  // (no branch around a single load: the compiler would wait for each before the next)
  if (rs.n > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] = rs.load(p, min(i * NT + tid, rs.n - 1));
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] = vec_of<D>(-INFINITY);
  }
  if (rs.n < NV * NT) {                                          // (a branch: whole chunks are spared the selects)
    asm volatile("");
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if ((i + 1) * NT > rs.n && i * NT + tid >= rs.n) v[i] = vec_of<D>(-INFINITY);
  }
  const float ef = ee >= 0 ? D::get(edge) : -INFINITY;

  float vm[NV], g[G];
#pragma unroll
  for (int i = 0; i < G; ++i) g[i] = -INFINITY;
  g[0] = fmaxf(g[0], ef);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    vm[i] = -INFINITY;
#pragma unroll
    for (int j = 0; j < D::EPV; ++j) {
      const float f = v[i].get(j);
      vm[i] = fmaxf(vm[i], f);
      if (NV < G) g[j % G] = fmaxf(g[j % G], f);
    }
    if (NV >= G) g[i % G] = fmaxf(g[i % G], vm[i]);
    __builtin_amdgcn_sched_barrier(0);
  }
  // from here the vectors are unpacked once more for the sum: the compiler must not keep what it has unpacked (half the kernel's
  // occupancy at 16-bit types)
#pragma unroll
  for (int i = 0; i < NV; ++i) asm volatile("" : "+v"(v[i].w[0]), "+v"(v[i].w[1]), "+v"(v[i].w[2]), "+v"(v[i].w[3]));
  const int groups = G > 1 && k > 64 ? G : 1;
  if (groups > 1) {
#pragma unroll
    for (int i = 0; i < G; ++i) gmax[i * NT + tid] = g[i];
  } else {
#pragma unroll
    for (int i = 1; i < G; ++i) g[0] = fmaxf(g[0], g[i]);
    gmax[tid] = g[0];
  }
  __syncthreads();

  if (tid < 64) {
    if (groups > 1) group_bound<W * G>(gmax, kk, bound);
    else group_bound<W>(gmax, kk, bound);
  }
  __syncthreads();
  const float thr = bound[0], m = bound[1];

  // the wavefront's vectors that reach the bound, from registers into LDS
  const int w0 = (tid >> 6) * cap;
  int n_vec = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const bool hit = vm[i] >= thr && i * NT + tid < rs.n;
    const uint64_t all = __ballot(hit);
    if (all) {
      const int at = n_vec + lanes_below(all);
      if (hit && at < cap) {
        vec_slot[w0 + at] = i * NT + tid;
        vec_data[w0 + at] = make_uint4(v[i].w[0], v[i].w[1], v[i].w[2], v[i].w[3]);
      }
      n_vec += __popcll(all);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  // 2^(x c - M) with one rounding and one instruction less than 2^((x - m) c); M is m c rounded, what that is off by is made good below.
  // Beyond 2^24 that could be any power of two (and an infinite m has none): there the differences are taken, from memory once more.
  const float M = m * c;
  float sum = __builtin_amdgcn_exp2f(__builtin_fmaf(ef, c, -M));
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (i * NT < rs.n) {
      float t = 0.f;
#pragma unroll
      for (int j = 0; j < D::EPV; ++j) t += __builtin_amdgcn_exp2f(__builtin_fmaf(v[i].get(j), c, -M));
      sum += t;
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  if (!(fabsf(M) < 16777216.f)) {
    sum = exp_t(ef - m, c);
    for (int s = tid; s < rs.n; s += NT) {
      const RowVec<D> w = rs.load(p, s);
#pragma unroll
      for (int j = 0; j < D::EPV; ++j) sum += exp_t(w.get(j) - m, c);
    }
  } else {
    sum *= __builtin_amdgcn_exp2f(-__builtin_fmaf(m, c, -M));
  }
  const double ws = wave_sum_d((double)sum);
  // their elements, one to a lane
  wave_lds_fence();
  int n_own = 0;
  {
    const bool hit = ef >= thr && ee >= 0;
    const uint64_t all = __ballot(hit);
    if (hit) cand[w0 + lanes_below(all)] = top_entry(ef, ee);
    n_own = __popcll(all);
  }
  const uint32_t* words = (const uint32_t*)(vec_data + w0);
  for (int base = 0; base < min(n_vec, cap) * D::EPV; base += 64) {
    const int q = base + lane;
    bool hit = q < min(n_vec, cap) * D::EPV;
    float f = 0.f;
    if (hit) {
      f = D::unpack(words[q / RowVec<D>::PER], q % RowVec<D>::PER);
      hit = f >= thr;
    }
    const uint64_t all = __ballot(hit);
    const int at = n_own + lanes_below(all);
    if (hit && at < cap) cand[w0 + at] = top_entry(f, rs.elem(vec_slot[w0 + q / D::EPV]) + q % D::EPV);
    n_own += __popcll(all);
  }
  if (lane == 0) {
    red[tid >> 6] = ws;
    cnt[tid >> 6] = max(n_own, n_vec);                          // (a vector that does not fit has an element that does not)
  }
  __syncthreads();
  double s = 0;
  int all = 0, before_wave = 0, most = 0;
#pragma unroll
  for (int i = 0; i < W; ++i) {
    s += red[i];
    before_wave += i < tid >> 6 ? cnt[i] : 0;
    all += cnt[i];
    most = max(most, cnt[i]);
  }

  uint64_t* flat = (uint64_t*)vec_data;                         // the candidates without gaps
  const bool exact = s != s || most > cap;
  if (exact) {                                 // (from memory again: a copy in registers would cost every row its place)
    constexpr int SHIFT = D::KEY_ZEROS;
    auto count = [&](uint64_t at_least) {                       // elements with key >> SHIFT at or above
      int q = ee >= 0 && (order_key(ef) >> SHIFT) >= at_least ? 1 : 0;
      for (int s = tid; s < rs.n; s += NT) {
        const RowVec<D> w = rs.load(p, s);
#pragma unroll
        for (int j = 0; j < D::EPV; ++j) q += (order_key(w.get(j)) >> SHIFT) >= at_least ? 1 : 0;
      }
      return block_count<NT>(q, cnt);
    };
    uint64_t b0 = 0, b1 = 1ull << (32 - SHIFT);
    while (b0 + 1 < b1) {
      const uint64_t mid = (b0 + b1) >> 1;
      if (count(mid) >= kk) b0 = mid;
      else b1 = mid;
    }
    const int need = kk - count(b0 + 1);                        // of those equal to the k-th
    if (tid == 0) n_cand = 0;
    __syncthreads();
    int before = 0;
    // pieces of ascending ids: head, the vectors one row of slots after the other, tail
    const int pieces = (rs.n + NT - 1) / NT;
    for (int piece = -1; piece <= pieces; ++piece) {
      const int s = piece * NT + tid;
      uint32_t same = 0, more = 0;
      RowVec<D> w = vec_of<D>(ef);                              // an edge element stands first
      if (piece == -1 || piece == pieces) {
        const bool here = ee >= 0 && (piece == -1) == (ee < rs.body);
        const uint32_t key = order_key(ef) >> SHIFT;
        same = here && key == b0 ? 1 : 0;
        more = here && key > b0 ? 1 : 0;
      } else if (s < rs.n) {
        w = rs.load(p, s);
#pragma unroll
        for (int j = 0; j < D::EPV; ++j) {
          const uint32_t key = order_key(w.get(j)) >> SHIFT;
          same |= (key == b0 ? 1u : 0u) << j;
          more |= (key > b0 ? 1u : 0u) << j;
        }
      }
      int scan = __popc(same);                                  // inclusive over the wavefront
      const int own = scan;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int q = __shfl_up(scan, o, 64);
        if (lane >= o) scan += q;
      }
      __syncthreads();
      if (lane == 63) cnt[tid >> 6] = scan;
      __syncthreads();
      int place = before + scan - own;
#pragma unroll
      for (int i = 0; i < W; ++i) {
        if (i < tid >> 6) place += cnt[i];
        before += cnt[i];
      }
#pragma unroll
      for (int j = 0; j < D::EPV; ++j) {
        const bool eq = same >> j & 1;
        if ((eq && place < need) || (more >> j & 1))
          flat[atomicAdd(&n_cand, 1)] = top_entry(w.get(j), piece == -1 || piece == pieces ? ee : rs.elem(s) + j);
        place += eq ? 1 : 0;
      }
    }
    all = kk;
    __syncthreads();
  } else if (n_chunk == 1 || all > len) {
    for (int i = lane; i < n_own; i += 64) flat[before_wave + i] = cand[w0 + i];
    __syncthreads();
  }

  if (n_chunk == 1) {
    rank_out<NT>(flat, all, k, [&](int rank, uint64_t o) {
      index[r * k + rank] = entry_id(o);
      values[r * k + rank] = D::put(key_value((uint32_t)(o >> 32)));
    });
    if (tid == NT - 1) lse[r] = (float)((double)m * inv_temp + logf((float)s));
  } else {                                                      // unordered, all of them where they fit
    uint64_t* l = lists + (int64_t)blockIdx.x * len;
    if (exact) {
      for (int i = tid; i < kk; i += NT) l[i] = flat[i];
    } else if (all <= len) {
      for (int i = lane; i < n_own; i += 64) l[before_wave + i] = cand[w0 + i];
    } else {
      rank_out<NT>(flat, all, k, [&](int rank, uint64_t o) { l[rank] = o; });
      all = kk;
    }
    for (int i = all + tid; i < len; i += NT) l[i] = 0;
    if (tid == 0) parts[blockIdx.x] = {(double)m, s, exact || kk < k ? -INFINITY : thr};
  }
}

// The lists of a row's chunks joined (a few KB, 8 to 13 us, latency): 16 entries a thread, bisection until between k and 5 k / 4 + 32 of
// them are left, ranks by counting.
template <class D, int NT>
__global__ __launch_bounds__(NT) void nast_top_join_kernel(const uint64_t* __restrict__ lists, const TopPart* __restrict__ parts,
                                                           typename D::store* __restrict__ values, int64_t* __restrict__ index,
                                                           float* __restrict__ lse, int k, int len, int n_chunk, double inv_temp) {
  __shared__ uint64_t cand[TOP_MAX_K + TOP_MAX_K / 4 + 32];
  __shared__ int cnt[NT / 64];
  __shared__ int n_cand;
  const int64_t r = blockIdx.x;
  const int n = n_chunk * len;
  uint64_t o[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) o[i] = i * NT + (int)threadIdx.x < n ? lists[r * n + i * NT + threadIdx.x] : 0;
  if (threadIdx.x == 0) n_cand = 0;
  // At least k entries reach the largest of the chunks' bounds, none lies above the largest maximum: where every chunk has a bound.
  // Else (a NaN somewhere, many equal values) b0 = 1 is below all entries and b1 not below the largest.
  float bound = -INFINITY, top = -INFINITY;
  bool known = true;
  for (int i = threadIdx.x & 63; i < n_chunk; i += 64) {
    const TopPart q = parts[r * n_chunk + i];
    known = known && q.bound > -INFINITY;
    bound = fmaxf(bound, q.bound);
    top = fmaxf(top, (float)q.m);
  }
  bound = wave_max(bound);
  top = wave_max(top);
  known = __ballot(!known) == 0;
  uint64_t b0 = known ? (uint64_t)order_key(bound) << 32 : 1;
  if (n > k + k / 4 + 32) {
    uint64_t b1 = known ? ((uint64_t)order_key(top) + 1) << 32 : ~0ull;
    while (b0 + 1 < b1) {
      const uint64_t mid = b0 + ((b1 - b0) >> 1);
      int q = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (i * NT < n) q += __popcll(__ballot(o[i] >= mid));
      __syncthreads();
      if ((threadIdx.x & 63) == 0) cnt[threadIdx.x >> 6] = q;
      __syncthreads();
      q = 0;
#pragma unroll
      for (int i = 0; i < NT / 64; ++i) q += cnt[i];
      if (q >= k) {
        b0 = mid;
        if (q <= k + k / 4 + 32) break;
      } else {
        b1 = mid;
      }
    }
  }
  __syncthreads();
  int own = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (i * NT < n) own += __popcll(__ballot(o[i] >= b0));
  int at = 0;                                                  // (each wavefront's place: in any order, they are ranked)
  if ((threadIdx.x & 63) == 0 && own) at = atomicAdd(&n_cand, own);
  at = __shfl(at, 0, 64);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    if (i * NT < n) {
      const uint64_t all = __ballot(o[i] >= b0);
      if (o[i] >= b0) cand[at + lanes_below(all)] = o[i];
      at += __popcll(all);
    }
  }
  __syncthreads();
  rank_out<NT>(cand, n_cand, k, [&](int rank, uint64_t q) {
    index[r * k + rank] = entry_id(q);
    values[r * k + rank] = D::put(key_value((uint32_t)(q >> 32)));
  });
  if (threadIdx.x >= NT - 64) {                                 // (the wavefront that ranks least)
    double m = -FLT_MAX, s = 0;
    for (int i = threadIdx.x & 63; i < n_chunk; i += 64) m = fmax(m, parts[r * n_chunk + i].m);
    m = wave_max_d(m);
    for (int i = threadIdx.x & 63; i < n_chunk; i += 64) s += parts[r * n_chunk + i].s * exp((parts[r * n_chunk + i].m - m) * inv_temp);
    s = wave_sum_d(s);
    if (threadIdx.x == NT - 1) lse[r] = (float)(m * inv_temp + log(s));
  }
}

// A chunk holds at most 16 vectors a thread, and not less than 16 k elements (or its list would be most of it).  Its list has room
// for the candidates that a bound met by 9/8 k + 8 groups lets through, and at least k entries.
// Few rows (no more than there are compute units) of up to 2^16 elements are taken by one workgroup of 1024 threads each, all in its
// registers, without a join: 8 x 32000 fp32 k 16 9.0 us on the device against 10.1 in chunks, k 256 15.4 and 24.9, 256 x 50021 fp16 k 100
// 13.5 and 18.4; but 400 x 32000 21.0 and 19.1, and 8 x 131072 bf16 k 64 16.9 and 14.1.
struct TopPlan {
  int n, chunk, len, threads, cap;
};
static TopPlan top_plan(int rows, int V, int k, int dtype) {
  const int most = 256 * 16 * (16 / row_size(dtype));
  TopPlan t;
  t.threads = 256;
  t.n = row_chunks(rows, V, most, 16 * k > 2048 ? 16 * k : 2048);
  if (t.n > 1 && rows <= 256 && V <= 1 << 16) {
    t.n = 1;
    t.threads = 1024;
  }
  if (t.n * k > TOP_MAX_LIST) t.n = row_chunks(512, V, most, V);
  t.chunk = (V + t.n - 1) / t.n;
  // Candidates a wavefront has room for: more take the place of workgroups (4096 x 5003 fp32 k 256 62 us with 160, 80 with 256), but a row
  // of two wavefronts' vectors has them all in those (4096 x 1000 fp16 k 256 98 and 76).
  t.cap = t.threads == 1024 || k <= 128 ? 128 : t.chunk * row_size(dtype) <= 128 * 16 ? 256 : 160;
  t.len = 2 * k + 32 < TOP_MAX_LIST / t.n ? 2 * k + 32 : TOP_MAX_LIST / t.n;
  return t;
}

extern "C" int64_t nast_top_logits_workspace_bytes(int rows, int V, int k, int dtype) {
  if (rows < 1 || V < 1 || V > TOP_MAX_V || k < 1 || k > TOP_MAX_K || !row_dtype_ok(dtype)) return 0;
  const TopPlan t = top_plan(rows, V, k, dtype);
  return t.n > 1 ? (int64_t)rows * t.n * (t.len * (int64_t)sizeof(uint64_t) + (int64_t)sizeof(TopPart)) : 0;
}

template <class D, int NT, int NV>
static void top_launch(const void* x, nast_rows xr, void* values, int64_t* index, float* lse, uint64_t* lists, TopPart* parts, int rows,
                       int V, int k, TopPlan t, double temp, hipStream_t s) {
  using T = typename D::store;
  hipLaunchKernelGGL((nast_top_chunk_kernel<D, NT, NV>), dim3(rows * t.n), dim3(NT),
                     NT / 64 * t.cap * (sizeof(uint4) + sizeof(uint64_t) + sizeof(int)), s, (const T*)x, xr, (T*)values, index, lse, lists, parts, V,
                     k, t.cap, t.len, t.chunk, t.n, 1.0 / temp, exp_scale(temp));
  if (t.n == 1) return;
  if (t.n * t.len <= 4096)
    hipLaunchKernelGGL((nast_top_join_kernel<D, 256>), dim3(rows), dim3(256), 0, s, lists, parts, (T*)values, index, lse, k, t.len, t.n,
                       1.0 / temp);
  else
    hipLaunchKernelGGL((nast_top_join_kernel<D, 1024>), dim3(rows), dim3(1024), 0, s, lists, parts, (T*)values, index, lse, k, t.len, t.n,
                       1.0 / temp);
}

extern "C" int nast_top_logits(const void* x, int dtype, nast_rows xr, void* values, int64_t* index, float* lse, int rows, int V,
                               int k, double temp, void* workspace, void* stream) {
  NAST_REQUIRE(row_dtype_ok(dtype), "nast_top_logits: unknown dtype %d", dtype);
  NAST_REQUIRE(rows >= 0 && V >= 1 && V <= TOP_MAX_V, "nast_top_logits: bad sizes rows=%d V=%d", rows, V);
  NAST_REQUIRE(k >= 1 && k <= TOP_MAX_K && k <= V, "nast_top_logits: k=%d must lie in [1, %d] and not exceed V=%d", k, TOP_MAX_K, V);
  NAST_REQUIRE(temp > 1e-30 && temp < 1e30, "nast_top_logits: temperature must lie between 1e-30 and 1e30");
  if (rows == 0) return NAST_OK;
  const TopPlan t = top_plan(rows, V, k, dtype);
  NAST_REQUIRE((int64_t)rows * t.n < (t.n == 1 ? 1 << 24 : 1 << 22), "nast_top_logits: too many rows (%d)", rows);
  NAST_REQUIRE(x && values && index && lse && (t.n == 1 || workspace), "nast_top_logits: NULL pointer");
  NAST_REQUIRE(row_aligned(x, dtype) && row_aligned(values, dtype), "nast_top_logits: misaligned pointer");
  hipStream_t s = (hipStream_t)stream;
  uint64_t* lists = (uint64_t*)workspace;
  TopPart* parts = t.n > 1 ? (TopPart*)(lists + (int64_t)rows * t.n * t.len) : nullptr;
  const int nv = (t.chunk / (16 / row_size(dtype)) + t.threads - 1) / t.threads;      // vectors a thread
  nast_prof_before(2, s);
  // Vectors a thread: the next even number up to 12, else 16; a wider kernel's spare vectors cost registers and selects.  Two or four too
  // many: 28086 x 5600 fp32, k 32, 121 us with 6, 140 with 8; 16384 x 9600 110 with 10, 128 with 12; 13355 x 11777 113 with 12, 121
  // with 16; halves and k 200 alike.  14 is left out: 11234 x 14000 fp32 112.4 us with 16, 110.6 with 14; 28000 bf16 124.9 and 120.8.
  // Workgroups of 1024, for calls of 9 to 20 us: powers of two; 12 for 16 and 6 for 8 would save 0.2 to 1 us (8 x 40001 fp32 11.4, 10.4).
#define NAST_TOP(NT, NV) NAST_ROW_DTYPE(dtype, (top_launch<D, NT, NV>(x, xr, values, index, lse, lists, parts, rows, V, k, t, temp, s)))
  if (t.threads == 1024) {
    if (nv <= 2) NAST_TOP(1024, 2);
    else if (nv <= 4) NAST_TOP(1024, 4);
    else if (nv <= 8) NAST_TOP(1024, 8);
    else top_launch<RowF32, 1024, 16>(x, xr, values, index, lse, lists, parts, rows, V, k, t, temp, s);   // (2^16 halves are 8)
  } else if (nv <= 2) NAST_TOP(256, 2);
  else if (nv <= 4) NAST_TOP(256, 4);
  else if (nv <= 6) NAST_TOP(256, 6);
  else if (nv <= 8) NAST_TOP(256, 8);
  else if (nv <= 10) NAST_TOP(256, 10);
  else if (nv <= 12) NAST_TOP(256, 12);
  else NAST_TOP(256, 16);
#undef NAST_TOP
  nast_prof_after(2, s, (double)row_size(dtype) * rows * (double)V);
  NAST_CHECK_LAUNCH("nast_top_logits");
  return NAST_OK;
}

// ---------------------------------------------------------------------------------------------
// distillation
// ---------------------------------------------------------------------------------------------
#define DISTILL_MAX_K 256
#define DISTILL_BWD_CHUNK 8192    // elements of a workgroup of the backward pass, up to twice as many
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
// log (w q_v) = (z_v - M) / T - L and log p_j = (t_j - C) / T - c (in two parts: next to a logit of -3e38 a logarithm of a sum would be
// lost).
struct DistillStats {
  double m_rest, coef, M, L, C, c;
};

// What a chunk leaves of its tokens; twice: some id of its part of the list stands in two slots.
struct DistillPart {
  double m, s;
  int twice;
};

// What the list alone contributes to a row: with d_j = log p_j - (z_j - zm) / T up to the normalisers not known yet,
//   S0 = sum e_j, S1 = sum e_j d_j, S2 = sum of exp((z - zm) / T) over the tokens named (each once), e_j = exp((t_j - C) / T - c0).
// In double throughout: the loss is a small difference of terms near 1 (with one slot of p = 0.01 and q = 0.0075 it is 3e-4, while
// p_r log p_r alone is rounded by 6e-8 in fp32), and it is a few slots per row.
struct SlotSums {
  double S0, S1, S2, C, c0, zm;
  bool any;
};

// By a workgroup of NT >= K threads, thread j = slot j; every thread gets the sums.  ids: LDS, NT words at a multiple of 16 bytes, holds
// the used slots' ids afterwards.  mark(id) is called for every used slot, twice() behind the barrier that follows: whether some id is
// named by two of them.
// Without TAIL no S2.
template <class D, int NT, bool TAIL, class M, class W2>
__device__ __forceinline__ SlotSums slot_sums(int64_t r, const typename D::store* p, const void* t, int t_dtype, const int64_t* idx, int K,
                                              const float* lse_t, int V, double it, uint32_t* ids, double* red, M&& mark, W2&& twice) {
  constexpr int W = NT / 64;
  const int j = threadIdx.x, w = threadIdx.x >> 6;
  uint32_t id = DISTILL_NO_ID;
  float tj = -INFINITY, zj = -INFINITY;
  if (j < K) {
    const int64_t v = idx[r * K + j];
    tj = teacher_logit(t, t_dtype, r * K + j);
    if (slot_used(v, tj, V)) {
      id = (uint32_t)v;
      zj = D::get(p[v]);
      mark((int)id);
    }
  }
  ids[j] = id;                               // (all NT: read in sixteens below)
  const bool used = id != DISTILL_NO_ID;
  float tm = wave_max(used ? tj : -FLT_MAX), zm = wave_max(used ? zj : -FLT_MAX);
  tm = fmaxf(tm, -FLT_MAX);
  zm = fmaxf(zm, -FLT_MAX);
  if ((j & 63) == 0) {
    red[2 * w] = tm;
    red[2 * w + 1] = zm;
  }
  __syncthreads();
  SlotSums q;
  double top = red[0];
  q.zm = red[1];
#pragma unroll
  for (int i = 1; i < W; ++i) {
    top = fmax(top, red[2 * i]);
    q.zm = fmax(q.zm, red[2 * i + 1]);
  }
  q.C = TAIL ? 0.0 : top;
  q.c0 = TAIL ? (double)lse_t[r] : 0.0;
  double e = 0, ed = 0, ez = 0;
  if (used) {
    const double a = ((double)tj - q.C) * it - q.c0, b = ((double)zj - q.zm) * it;
    e = exp(a);
    if (e != 0) ed = e * (a - b);
    if (TAIL) {
      int at = j;                            // an id named twice is one token of the student's: the first slot's
      if (twice()) {
#pragma unroll 1
        for (int i = (K - 1) & ~15; i >= 0; i -= 16) {           // (sixteen at a time: one wait for LDS)
          uint4 o[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) o[u] = *(const uint4*)(ids + i + 4 * u);
#pragma unroll
          for (int u = 3; u >= 0; --u) {
            at = o[u].w == id ? i + 4 * u + 3 : at;
            at = o[u].z == id ? i + 4 * u + 2 : at;
            at = o[u].y == id ? i + 4 * u + 1 : at;
            at = o[u].x == id ? i + 4 * u : at;
          }
        }
      }
      if (at == j) ez = exp(b);
    }
  }
  double any = __ballot(used) ? 1 : 0;
  if (any != 0) {
    e = wave_sum_d(e);
    ed = wave_sum_d(ed);
    if (TAIL) ez = wave_sum_d(ez);
  }
  __syncthreads();
  if ((j & 63) == 0) {
    red[4 * w] = e;
    red[4 * w + 1] = ed;
    red[4 * w + 2] = ez;
    red[4 * w + 3] = any;
  }
  __syncthreads();
  q.S0 = q.S1 = q.S2 = 0;
  q.any = false;
#pragma unroll
  for (int i = 0; i < W; ++i) {
    q.S0 += red[4 * i];
    q.S1 += red[4 * i + 1];
    q.S2 += red[4 * i + 2];
    q.any = q.any || red[4 * i + 3] != 0;
  }
  __syncthreads();
  return q;
}

// The end of a row's forward pass by one thread.  rest: maximum and exponential sum, with TAIL of the tokens that no used slot names,
// without of all.
template <bool TAIL>
__device__ __forceinline__ void distill_finish(int64_t r, const MaxSumD& rest, const SlotSums& q, float* loss, DistillStats* stats, double it) {
  DistillStats o;
  double l;
  o.m_rest = rest.m;
  o.C = q.C;
  if (TAIL) {
    o.M = fmax(rest.m, q.zm);
    const double below = (rest.m - o.M) * it;
    o.L = log(q.S2 * exp((q.zm - o.M) * it) + rest.s * exp(below));
    o.c = q.c0;
    l = q.S1 + q.S0 * ((o.M - q.zm) * it + o.L);
    const double log_qr = below + log(rest.s) - o.L;
    const double pr = rest.s == 0 ? 0.0 : fmax(1.0 - q.S0, 0.0);   // (no bucket where the student has no token left for it)
    if (pr > 0) l += pr * (log(pr) - log_qr);
    const double w = q.S0 + pr;
    // w q_v - p_r q_v / q_r = exp((z_v - m_r) / T) / s_r * (w q_r - p_r): no quotient of small numbers; 0 for a row without a rest, NaN
    // for a row of nothing but -inf
    o.coef = rest.s == 0 ? (o.L > -INFINITY ? 0.0 : NAN) : (w * exp(log_qr) - pr) / rest.s;
    o.L -= log(w);                           // (+inf where w is 0: such a row's gradient is 0)
  } else {
    o.M = rest.m;
    o.L = log(rest.s);
    o.c = log(q.S0);
    l = q.S1 / q.S0 - o.c + (o.M - q.zm) * it + o.L;
    o.coef = rest.s == 0 ? NAN : 1.0 / rest.s;
  }
  if (!q.any) o.coef = l = 0;
  stats[r] = o;
  loss[r] = (float)l;
}

// One workgroup per chunk of a row: (max, exponential sum) of its tokens; with TAIL of those that no used slot names.  The named ones are
// marked in LDS, one bit per element and one per vector, and left out: their terms are added in double at the end, so that q_r is a sum
// and no difference.
// Rows are taken from the last to the first: the backward pass, from the first to the last, then begins with what this pass has
// left in the last-level cache (256 MB), and this pass with what the product that made the logits has left there.
// Bound by memory: 16384 x 9600 fp32 with a tail 118 us (5.3 TB/s), 4096 x 131072 bf16 193 us (5.6 TB/s); 33 x 9600 fp32 6 us, latency.
template <class D, bool SPLIT, bool TAIL>
__global__ __launch_bounds__(256) void nast_top_distill_fwd_kernel(const typename D::store* __restrict__ x, nast_rows xr,
                                                                   const void* __restrict__ t, int t_dtype,
                                                                   const int64_t* __restrict__ idx, int K,
                                                                   const float* __restrict__ lse_t, float* __restrict__ loss,
                                                                   DistillStats* __restrict__ stats, DistillPart* __restrict__ parts, int V,
                                                                   int chunk, int n_chunk, double it, float c) {
  constexpr int U = 4;
  extern __shared__ uint32_t bits[];                           // bit EPV + i: element body + i
  __shared__ double red[16];
  __shared__ int twice;
  __shared__ alignas(16) uint32_t ids[256];
  const unsigned block = gridDim.x - 1 - blockIdx.x;
  const int64_t r = block / n_chunk;
  const int lo = (int)(block % n_chunk) * chunk, hi = min(V, lo + chunk);
  const typename D::store* p = x + row_offset(r, xr);
  MaxSum a{-FLT_MAX, 0.0};
  SlotSums q;
  if (!TAIL) {
    if (!SPLIT) q = slot_sums<D, 256, TAIL>(r, p, t, t_dtype, idx, K, lse_t, V, it, ids, red, [](int) {}, [] { return false; });
    a = span_max_sum<D, 256>(p, lo, hi, c);
  } else {
    const RowSpan16<D> rs(p, lo, hi);
    const int bit0 = rs.body - D::EPV, e = rs.edge(threadIdx.x), words = (hi - bit0 + 31) / 32;
    const typename D::store edge = p[e >= 0 ? e : lo];
    uint32_t* flags = bits + words;                            // byte (s / 1024) * 256 + s % 256, bit s / 256 % 4: vector s
    const int flag_words = (rs.n + 1023) / 1024 * 64;
    for (int w = threadIdx.x; w < words + flag_words; w += 256) bits[w] = 0;
    if (threadIdx.x == 0) twice = 0;
    __syncthreads();
    auto mark = [&](int id) {
      const int bit = id - bit0, s = (id - rs.body) / D::EPV;
      if (atomicOr(&bits[bit >> 5], 1u << (bit & 31)) >> (bit & 31) & 1) twice = 1;
      if (id >= rs.body && s < rs.n) atomicOr(&flags[(s >> 10) * 64 + ((s & 255) >> 2)], 1u << ((s & 3) * 8 + ((s >> 8) & 3)));
    };
    if (!SPLIT) {
      q = slot_sums<D, 256, TAIL>(r, p, t, t_dtype, idx, K, lse_t, V, it, ids, red, mark, [&] { return twice != 0; });
    } else {
      if ((int)threadIdx.x < K) {
        const int64_t v = idx[r * K + threadIdx.x];
        if (v >= lo && v < hi && slot_used(v, teacher_logit(t, t_dtype, r * K + threadIdx.x), V)) mark((int)v);
      }
      __syncthreads();
    }
    auto leave_out = [&](RowVec<D>& v, int slot) {
      const int at = (slot + 1) * D::EPV;
      const uint32_t named = bits[at >> 5] >> (at & 31);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float f[2];
#pragma unroll
        for (int j = 0; j < RowVec<D>::PER; ++j) f[j] = named >> (i * RowVec<D>::PER + j) & 1 ? -INFINITY : D::unpack(v.w[i], j);
        v.w[i] = D::pack(f);
      }
    };
    const uint8_t* flag = (const uint8_t*)flags;
    for_slots<D, 256, U>(rs, [&](int s) { return rs.load(p, s); },
                         [&](RowVec<D>(&v)[U], int s) {
                           const uint32_t f = flag[(s >> 10) * 256 + threadIdx.x];
                           if (f) {
#pragma unroll
                             for (int u = 0; u < U; ++u)
                               if (f >> u & 1) leave_out(v[u], s + 256 * u);
                           }
                           fold<D, U>(a, v, c);
                         },
                         [&](RowVec<D>& v, int s) {
                           leave_out(v, s);
                           const RowVec<D> one[1] = {v};
                           fold<D, 1>(a, one, c);
                         });
    if (e >= 0 && !(bits[(e - bit0) >> 5] >> ((e - bit0) & 31) & 1)) fold_one(a, D::get(edge), c);
  }
  const MaxSumD rest = block_max_sum<256>(a, c, red);
  if (threadIdx.x != 0) return;
  if (SPLIT) parts[block] = {rest.m, rest.s, TAIL ? twice : 0};
  else distill_finish<TAIL>(r, rest, q, loss, stats, it);
}

// one workgroup of NT >= K threads per row joins the chunks
template <class D, int NT, bool TAIL>
__global__ __launch_bounds__(NT) void nast_top_distill_join_kernel(const typename D::store* __restrict__ x, nast_rows xr,
                                                                   const void* __restrict__ t, int t_dtype,
                                                                   const int64_t* __restrict__ idx, int K,
                                                                   const float* __restrict__ lse_t, float* __restrict__ loss,
                                                                   DistillStats* __restrict__ stats, const DistillPart* __restrict__ parts,
                                                                   int V, int n_chunk, double it) {
  __shared__ double red[NT / 16];
  __shared__ alignas(16) uint32_t ids[NT];
  const int64_t r = blockIdx.x;
  MaxSumD rest{-FLT_MAX, 0};
  bool twice = false;
  for (int i = threadIdx.x & 63; i < n_chunk; i += 64) rest.m = fmax(rest.m, parts[r * n_chunk + i].m);
  rest.m = wave_max_d(rest.m);
  for (int i = threadIdx.x & 63; i < n_chunk; i += 64) {
    const DistillPart o = parts[r * n_chunk + i];
    rest.s += o.s * exp((o.m - rest.m) * it);
    twice = twice || o.twice;
  }
  rest.s = wave_sum_d(rest.s);
  twice = __ballot(twice) != 0;
  const SlotSums q = slot_sums<D, NT, TAIL>(r, x + row_offset(r, xr), t, t_dtype, idx, K, lse_t, V, it, ids, red,
                                              [](int) {}, [&] { return twice; });
  if (threadIdx.x == 0) distill_finish<TAIL>(r, rest, q, loss, stats, it);
}

// One workgroup per chunk of a row: the rest's gradient everywhere, then, behind a barrier, the value of each named token over it.
// AROUND: gradients of more than the last-level cache holds (256 MB) are stored around it, so that they do not drive out the logits the
// forward pass has left there: 4096 x 131072 bf16 577 -> 569 us for both passes, 16384 x 9600 fp32 388 -> 354; a smaller one stays there
// for the product that reads it.
// Bound by memory, one read and one write of the logits: 16384 x 9600 fp32 226 us (5.6 TB/s), 1021 x 50021 fp16 34 us (6.0 TB/s); 33 rows
// of 9600 take 5 us, latency.  A chunk has 8192 elements or more, so that the list, read by each, is a small part of it.
template <class D, bool AROUND>
__global__ __launch_bounds__(256) void nast_top_distill_bwd_kernel(const float* __restrict__ g, const typename D::store* __restrict__ x,
                                                                   nast_rows xr, const void* __restrict__ t, int t_dtype,
                                                                   const int64_t* __restrict__ idx, int K,
                                                                   const DistillStats* __restrict__ stats,
                                                                   typename D::store* __restrict__ gx, nast_rows gxr, int V, int chunk,
                                                                   int n_chunk, double it, float c) {
  constexpr int U = 4;
  __shared__ uint32_t ids[256];              // the slots in this chunk, each wavefront's without gaps from 64 * its number
  __shared__ double ps[256];
  __shared__ uint32_t bits[DISTILL_BWD_CHUNK / 16];           // which elements are named: a chunk is shorter than two of these
  __shared__ int cnt[4], twice;
  const int64_t r = blockIdx.x / n_chunk;
  const int lo = (int)(blockIdx.x % n_chunk) * chunk, hi = min(V, lo + chunk);
  const typename D::store* p = x + row_offset(r, xr);
  typename D::store* o = gx + row_offset(r, gxr);
  const DistillStats st = stats[r];
  const double gr = (double)g[r] * it;
  uint32_t id = DISTILL_NO_ID;
  float z = 0.f, tv = 0.f;
  if ((int)threadIdx.x < K) {
    const int64_t v = idx[r * K + threadIdx.x];
    tv = teacher_logit(t, t_dtype, r * K + threadIdx.x);
    if (slot_used(v, tv, V) && v >= lo && v < hi) {
      id = (uint32_t)v;
      z = D::get(p[v]);
    }
  }
  for (int w = threadIdx.x; w < DISTILL_BWD_CHUNK / 16; w += 256) bits[w] = 0;
  if (threadIdx.x == 0) twice = 0;
  __syncthreads();
  if (id != DISTILL_NO_ID && (atomicOr(&bits[((int)id - lo) >> 5], 1u << (((int)id - lo) & 31)) >> (((int)id - lo) & 31) & 1)) twice = 1;
  const uint64_t named = __ballot(id != DISTILL_NO_ID);
  const int own = (threadIdx.x & 192) + lanes_below(named);
  if (id != DISTILL_NO_ID) {
    ids[own] = id;
    ps[own] = exp(((double)tv - st.C) * it - st.c);
  }
  if ((threadIdx.x & 63) == 0) cnt[threadIdx.x >> 6] = __popcll(named);
  // a factor of 0 (a row without a list, a row of no weight) writes zeros whatever the logits hold
  const float F = gr == 0 ? 0.f : (float)(gr * st.coef), m = (float)st.m_rest;
  const RowSpan16<D> rs(o, lo, hi);
  const int e = rs.edge(threadIdx.x);
  const typename D::store edge = p[e >= 0 ? e : lo];
  auto put = [&](RowVec<D>& v, int slot) {
    float f[D::EPV];
#pragma unroll
    for (int i = 0; i < D::EPV; ++i) f[i] = F == 0.f ? 0.f : exp_t(v.get(i) - m, c) * F;
    v.put(f);
    if (AROUND) vec_store_around<D>(o + rs.elem(slot), v);
    else vec_store<D>(o + rs.elem(slot), v);
  };
  for_slots<D, 256, U>(rs, [&](int s) { return vec_load_any<D>(p + rs.elem(s)); },
                       [&](RowVec<D>(&v)[U], int s) {
#pragma unroll
                         for (int u = 0; u < U; ++u) put(v[u], s + 256 * u);
                       },
                       put);
  if (e >= 0) o[e] = D::put(F == 0.f ? 0.f : exp_t(D::get(edge) - m, c) * F);
  __syncthreads();
  if (id == DISTILL_NO_ID) return;
  double pj = ps[own];
  bool first = true;
  if (twice) {                               // an id in two slots: the sum of both, by the first of them
    pj = 0;
    for (int w = 0; w < 4; ++w) {
      for (int j = w * 64; j < w * 64 + cnt[w]; ++j) {
        const bool same = ids[j] == id;
        first = first && !(same && j < own);
        pj += same ? ps[j] : 0.0;
      }
    }
  }
  if (first) o[id] = D::put(gr == 0 ? 0.f : (float)(gr * (exp(((double)z - st.M) * it - st.L) - pj)));
}

static int distill_check(const char* name, int dtype, int t_dtype, int K, int rows, int V, double temp) {
  NAST_REQUIRE(row_dtype_ok(dtype) && row_dtype_ok(t_dtype), "%s: unknown dtype", name);
  NAST_REQUIRE(rows >= 0 && V >= 1 && V < (1 << 24), "%s: bad sizes rows=%d V=%d", name, rows, V);
  NAST_REQUIRE(K >= 1 && K <= DISTILL_MAX_K, "%s: a list has 1 to %d slots, not %d", name, DISTILL_MAX_K, K);
  NAST_REQUIRE(temp > 1e-30 && temp < 1e30, "%s: temperature must lie between 1e-30 and 1e30", name);
  return NAST_OK;
}
// One workgroup reads a whole row where there are rows enough to fill the card (512: two workgroups a compute unit); a chunk has at
// least 16 Ki elements and at most 2^15 vectors (the membership bits of 2^18 elements take 40 KB).
struct DistillPlan {
  int n, chunk;
};
static DistillPlan distill_plan(int rows, int V, int dtype) {
  DistillPlan d;
  d.n = row_chunks(rows, V, (16 / row_size(dtype)) << 15, 1 << 14);
  d.chunk = (V + d.n - 1) / d.n;
  return d;
}

extern "C" int64_t nast_top_distill_workspace_bytes(int rows, int V, int dtype) {
  if (rows < 1 || V < 1 || !row_dtype_ok(dtype)) return 0;
  const DistillPlan d = distill_plan(rows, V, dtype);
  return d.n > 1 ? (int64_t)rows * d.n * (int64_t)sizeof(DistillPart) : 0;
}

template <class D, bool TAIL>
static void distill_fwd(const void* x, nast_rows xr, const void* t, int t_dtype, const int64_t* idx, int K, const float* lse_t,
                        float* loss, DistillStats* st, DistillPart* parts, int rows, int V, DistillPlan d, double temp, hipStream_t s) {
  const typename D::store* xp = (const typename D::store*)x;
  const double it = 1.0 / temp;
  // bits of a chunk's elements, and of its vectors in fours of 256
  const unsigned lds = TAIL ? 4u * ((d.chunk + 16 + 31) / 32 + (d.chunk / D::EPV + 1023) / 1024 * 64) : 0;
  if (d.n == 1) {
    hipLaunchKernelGGL((nast_top_distill_fwd_kernel<D, false, TAIL>), dim3(rows), dim3(256), lds, s, xp, xr, t, t_dtype, idx, K, lse_t, loss,
                       st, parts, V, d.chunk, d.n, it, exp_scale(temp));
    return;
  }
  hipLaunchKernelGGL((nast_top_distill_fwd_kernel<D, true, TAIL>), dim3(rows * d.n), dim3(256), lds, s, xp, xr, t, t_dtype, idx, K, lse_t,
                     loss, st, parts, V, d.chunk, d.n, it, exp_scale(temp));
  if (K <= 64)
    hipLaunchKernelGGL((nast_top_distill_join_kernel<D, 64, TAIL>), dim3(rows), dim3(64), 0, s, xp, xr, t, t_dtype, idx, K, lse_t, loss, st,
                       parts, V, d.n, it);
  else
    hipLaunchKernelGGL((nast_top_distill_join_kernel<D, 256, TAIL>), dim3(rows), dim3(256), 0, s, xp, xr, t, t_dtype, idx, K, lse_t, loss, st,
                       parts, V, d.n, it);
}

extern "C" int nast_top_distill_fwd(const void* x, int dtype, nast_rows xr, const void* t, int t_dtype, const int64_t* idx, int K,
                                    const float* lse_t, float* loss, double* stats, int rows, int V, double temp, void* workspace,
                                    void* stream) {
  if (int rc = distill_check("nast_top_distill_fwd", dtype, t_dtype, K, rows, V, temp)) return rc;
  if (rows == 0) return NAST_OK;
  NAST_REQUIRE(x && t && idx && loss && stats, "nast_top_distill_fwd: NULL pointer");
  NAST_REQUIRE(row_aligned(x, dtype) && row_aligned(t, t_dtype), "nast_top_distill_fwd: misaligned pointer");
  const DistillPlan d = distill_plan(rows, V, dtype);
  NAST_REQUIRE((int64_t)rows * d.n < (1 << 24), "nast_top_distill_fwd: too many rows (%d)", rows);
  NAST_REQUIRE(d.n == 1 || workspace, "nast_top_distill_fwd: NULL workspace");
  hipStream_t s = (hipStream_t)stream;
  DistillStats* st = (DistillStats*)stats;
  DistillPart* parts = (DistillPart*)workspace;
  nast_prof_before(2, s);
  NAST_ROW_DTYPE(dtype, {
    if (lse_t) distill_fwd<D, true>(x, xr, t, t_dtype, idx, K, lse_t, loss, st, parts, rows, V, d, temp, s);
    else distill_fwd<D, false>(x, xr, t, t_dtype, idx, K, lse_t, loss, st, parts, rows, V, d, temp, s);
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
  const int n = V < 2 * DISTILL_BWD_CHUNK ? 1 : V / DISTILL_BWD_CHUNK, chunk = (V + n - 1) / n;
  NAST_REQUIRE((int64_t)rows * n < (1 << 24), "nast_top_distill_bwd: too many rows (%d)", rows);
  nast_prof_before(2, (hipStream_t)stream);
  const bool around = (int64_t)rows * V * row_size(dtype) > (256 << 20);
  NAST_ROW_DTYPE(dtype, {
    using T = typename D::store;
    auto kernel = around ? nast_top_distill_bwd_kernel<D, true> : nast_top_distill_bwd_kernel<D, false>;
    hipLaunchKernelGGL(kernel, dim3(rows * n), dim3(256), 0, (hipStream_t)stream, g, (const T*)x, xr, t, t_dtype, idx, K,
                       (const DistillStats*)stats, (T*)gx, gxr, V, chunk, n, 1.0 / temp, exp_scale(temp));
  });
  nast_prof_after(2, (hipStream_t)stream, 2.0 * row_size(dtype) * rows * (double)V);
  NAST_CHECK_LAUNCH("nast_top_distill_bwd");
  return NAST_OK;
}
