// The rest of a speculative step after kf_attn_tree (kf_tree.hip): the walk
// through the drafted tree against the target's logits, and the move of the
// accepted path's cache rows.
#include "kf_common.h"
#include "kf_internal.h"

#include <algorithm>
#include <climits>

namespace kf {

namespace {

constexpr int MAXN = KF_TREE_MAX_NODES;

// ------------------------------------------------------------------ verification
// Node 0 is the token emitted last; row i of the logits is the target's
// distribution p_i = softmax(logits_i / T) of the token after node i.  From node
// 0 the walk tries a node's children in index order and steps to the first one
// taken, until none is:
//   drafts without probabilities   child with token c is taken if u W < p(c), W
//       what its refused elder siblings left of the mass (1 less their p); a
//       token refused before is refused again
//   a chain drawn from q           taken if u q(c) < p(c)
// and the token after the path is the smallest v at which the running sum of
// the weights passes u_0 times their total: p without the refused tokens, or
// max(p - q, 0), or p itself where nothing was refused.  Either way the emitted
// tokens have the target's distribution.  T = 0: a child is taken if its token
// is the most likely one (the lowest of equals), and that token follows the
// path.
//
// Two ways to the path, then the draw.  A row's softmax costs a pass over V
// values, and the next row of a path is known only after the last:
//   all rows  (stats) the sums of every row at once, over the whole chip, then
//             (draw) the walk over them, which is short
//   walk      (walk) one workgroup per sequence, row by row down the path
// The first reads every row once at the chip's rate, the second only the path's,
// at one CU's; verify_drafts says which is taken.  The draw's weights are formed by
// all workgroups of a sequence, a slice of the row each, and the last one to
// arrive picks the token.
//
// Measured: a chain of 5 with drafts over 32000 float32 values 15 us (4 of sums, 11 of
// ten dependent round trips); 16 trees of 64 nodes over 131072 16-bit values 41 to 54
// us (268 MB of logits: 5.4 TB/s and more where they lie in the last-level cache, then
// 19 us of walk and draw).

// 16 bytes of a row as floats: granule k of the row's aligned granules, the
// row's first element at place `lead` of granule 0.  Places outside the row are
// -inf, and never read.
template <typename T>
struct Row {
  static constexpr int E = 16 / sizeof(T);
  const T* x;
  int lead, V;
  __device__ __forceinline__ Row(const T* p, int V_) : x(p), V(V_) {
    lead = (int)(((uintptr_t)p & 15) / sizeof(T));
  }
  __device__ __forceinline__ int granules() const { return (lead + V + E - 1) / E; }
  __device__ __forceinline__ int first(int k) const { return k * E - lead; }
  __device__ __forceinline__ u32x4 raw(int k) const {
    const int v0 = first(k);
    if (v0 >= 0 && v0 + E <= V) return *(const u32x4*)(x + v0);
    T t[E];
#pragma unroll
    for (int e = 0; e < E; ++e)
      t[e] = v0 + e >= 0 && v0 + e < V ? x[v0 + e] : from_f32<T>(-INFINITY);
    u32x4 u;
    __builtin_memcpy(&u, t, 16);
    return u;
  }
  static __device__ __forceinline__ void unpack(const u32x4& u, float* f) {
    if constexpr (sizeof(T) == 4)
      __builtin_memcpy(f, &u, 16);
    else
      unpack8<T>(u, f);
  }
};

// 2^x for x <= 0 in 64 bits: 2^round(x) times the Taylor polynomial of 2^r, |r| <=
// 1/2, whose first term left out is (ln 2 / 2)^12 / 12! = 6e-15.
__device__ __forceinline__ double exp2_64(double x) {
  const double n = __builtin_rint(x), r = x - n;
  constexpr double L = 0.69314718055994530942;
  constexpr double c2 = L * L / 2, c3 = c2 * L / 3, c4 = c3 * L / 4, c5 = c4 * L / 5,
                   c6 = c5 * L / 6, c7 = c6 * L / 7, c8 = c7 * L / 8, c9 = c8 * L / 9,
                   c10 = c9 * L / 10, c11 = c10 * L / 11;
  double p = c11;
  p = fma(p, r, c10);
  p = fma(p, r, c9);
  p = fma(p, r, c8);
  p = fma(p, r, c7);
  p = fma(p, r, c6);
  p = fma(p, r, c5);
  p = fma(p, r, c4);
  p = fma(p, r, c3);
  p = fma(p, r, c2);
  p = fma(p, r, L);
  p = fma(p, r, 1.0);
  // (below 2^-1070 nothing is left; -inf has no r)
  return x > -1070.0 ? __builtin_ldexp(p, (int)n) : x <= -1070.0 ? 0.0 : x;
}

struct Stat {
  float m;   // maximum
  int at;    // first place of the maximum
  double s;  // sum of 2^((x - m) c); not positive and finite: no distribution
};
__device__ __forceinline__ bool has_mass(double s) { return s > 0.0 && s < INFINITY; }
// Whether the row is a distribution.  greedy: only NaN shows in s, so the maximum has to
// be finite (+inf, or -inf throughout).
__device__ __forceinline__ bool is_distribution(const Stat& st, bool greedy) {
  return greedy ? st.s == st.s && fabsf(st.m) < INFINITY : has_mass(st.s);
}

// 2^((a - b) c) for two maxima, 1 where both are -inf
__device__ __forceinline__ double weight_of(float a, float b, double c) {
  return a == b ? 1.0 : (double)exp2f((a - b) * (float)c);
}

// Joins a statistic of other values of the row.  Equal maxima: the lower place.
__device__ __forceinline__ void join(Stat& x, const Stat& y, double c) {
  const float m = fmaxf(x.m, y.m);
  x.s = x.s * weight_of(x.m, m, c) + y.s * weight_of(y.m, m, c);
  x.at = x.m > y.m ? x.at : y.m > x.m ? y.at : min(x.at, y.at);
  x.m = m;
}

// Adds granules k, k + stride, ... (U of them, below `end`) to a thread's share:
// the maximum of the batch first, then (SUM) one exponential a value; without SUM
// the place of the maximum.  s becomes NaN where a value is NaN or (SUM) +inf.
// The exponentials are one float32 instruction each (in 64 bits a chain of 16 nodes
// with the draft's rows, 16 sequences of 131072 values, takes 108 us instead of 51) of
// the difference to the maximum: the maximum's own is 1 and a constant added to the
// row, or a low temperature, moves no other.  An argument x is off by 2^-23 of itself,
// its exponential by that times |x| ln 2 and by 2^-22, a batch's sum (16 or 32 values)
// by some 2^-22 more; the batches are summed in 64 bits.  The mean of |x| over a
// distribution of V values is below log2 V, so a row's sum, and with it every
// probability, is off by less than 2^-18.5 of itself at V = 2^20, by some 2^-22 where a few
// tokens hold most of it (measured at the border of acceptance: 1e-7, root mean square, 32000
// to 131072 values), and so is the chance of a token; max(p - q, 0) by that of p and of q.
template <typename T, int U>
__device__ __forceinline__ void load_batch(const Row<T>& r, int k, int stride, int end,
                                           u32x4* raw) {
  constexpr int E = Row<T>::E;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (k + u * stride < end) {
      raw[u] = r.raw(k + u * stride);
    } else {  // (the lowest value of every type: 2^-inf below)
      T t[E];
#pragma unroll
      for (int e = 0; e < E; ++e) t[e] = from_f32<T>(-INFINITY);
      __builtin_memcpy(&raw[u], t, 16);
    }
  }
}
template <typename T, bool SUM, int U>
__device__ __forceinline__ void add_batch(const Row<T>& r, int k, int stride, const u32x4* raw,
                                          double c, Stat& st) {
  constexpr int E = Row<T>::E;
  float m = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float f[E];
    Row<T>::unpack(raw[u], f);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (!SUM) nan |= f[e] != f[e];
      m = fmaxf(m, f[e]);
    }
  }
  if (m > st.m) {
    if (SUM) {
      st.s *= weight_of(st.m, m, c);
    } else {
#pragma unroll
      for (int u = U - 1; u >= 0; --u) {
        float f[E];
        Row<T>::unpack(raw[u], f);
#pragma unroll
        for (int e = E - 1; e >= 0; --e)
          if (f[e] == m) st.at = r.first(k + u * stride) + e;
      }
    }
    st.m = m;
  }
  if (!SUM) {
    if (nan) st.s = NAN;
    return;
  }
  const float ref = st.m == -INFINITY ? 0.f : st.m;
  const float cf = (float)c;
  float gs = 0.f;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float f[E];
    Row<T>::unpack(raw[u], f);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      gs += __builtin_amdgcn_exp2f((f[e] - ref) * cf);
    }
  }
  st.s += (double)gs;
}

// The workgroup's shares joined, in order; `x` is one Stat per wavefront.
template <int NT>
__device__ __forceinline__ Stat join_all(Stat st, double c, Stat* x) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    Stat y;
    y.m = __shfl_xor(st.m, o, 64);
    y.at = __shfl_xor(st.at, o, 64);
    y.s = __shfl_xor(st.s, o, 64);
    join(st, y, c);
  }
  __syncthreads();  // the previous use of x is over
  if (lane == 0) x[w] = st;
  __syncthreads();
  // every wavefront joins the wavefronts' by itself, a lane each
  st = x[lane % (NT / 64)];
#pragma unroll
  for (int o = NT / 128; o >= 1; o >>= 1) {
    Stat y;
    y.m = __shfl_xor(st.m, o, 64);
    y.at = __shfl_xor(st.at, o, 64);
    y.s = __shfl_xor(st.s, o, 64);
    join(st, y, c);
  }
  st.s = __shfl(st.s, 0, 64);  // (the lanes' orders differ in the last bit)
  return st;
}

constexpr int ST = 256, SU = 4;            // threads, granules of a thread
constexpr int SLICE = ST * SU;             // granules of a slice
// slices of a row of V values at any alignment
__host__ __device__ __forceinline__ int slices_of(int V, int E) {
  return ((V + 2 * E - 2) / E + SLICE - 1) / SLICE;
}

// Workgroup (slice, row, sequence): rows 0 .. N - 1 the target's, N .. 2N - 2 the
// draft's.  Rows of unused nodes are left out.  Bound by HBM: a thread's four
// granules are in flight before the first is used.
template <typename T, bool SUM>
__global__ __launch_bounds__(ST) void verify_stats_kernel(VerifyArgs a, Stat* __restrict__ out,
                                                          int* __restrict__ arrived) {
  __shared__ Stat x[ST / 64];
  const int b = blockIdx.z, i = blockIdx.y, t = threadIdx.x;
  const int n = a.counts ? a.counts[b] : a.N;
  if (t == 0 && i == 0 && blockIdx.x == 0) arrived[b] = 0;
  const bool draft = i >= a.N;
  const int at = draft ? i - a.N : i;
  if (draft ? at + 1 >= n : at >= n) return;
  const Row<T> r(draft ? (const T*)a.drafts + b * a.drafts_sb + at * a.drafts_sn
                       : (const T*)a.logits + b * a.logits_sb + at * a.logits_sn,
                 a.V);
  const double c = a.inv_t * 1.4426950408889634074;
  Stat st{-INFINITY, INT_MAX, 0.0};
  u32x4 raw[SU];
  const int k = blockIdx.x * SLICE + t;
  load_batch<T, SU>(r, k, ST, r.granules(), raw);
  add_batch<T, SUM, SU>(r, k, ST, raw, c, st);
  st = join_all<ST>(st, c, x);
  if (t == 0) out[((int64_t)b * gridDim.y + i) * gridDim.x + blockIdx.x] = st;
}

// What a workgroup knows of its sequence's nodes.  kids[i]: node i's children as
// bits, so that a node meets its elder siblings and no other (64 nodes, four children
// each: the walk 1.9 us less than over all nodes between).
struct Nodes {
  int par[MAXN], tok[MAXN];
  float u[MAXN];
  uint32_t kids[MAXN][MAXN / 32];
};
// Loads the nodes; whether the sequence is refused.
__device__ __forceinline__ bool load_nodes(const VerifyArgs& a, int b, int n, Nodes& nd) {
  bool bad = n < 0 || n > a.N;
  const int words = (a.N + 31) / 32;
  for (int x = threadIdx.x; x < a.N * words; x += blockDim.x) nd.kids[x / words][x % words] = 0;
  __syncthreads();
  for (int t = threadIdx.x; t < a.N; t += blockDim.x) {
    int par = t - 1;
    if (a.parents != nullptr) par = a.parents[(int64_t)b * a.parents_stride + t];
    const int64_t tok = a.tokens[(int64_t)b * a.N + t];
    nd.par[t] = par;
    nd.tok[t] = tok >= 0 && tok < a.V ? (int)tok : -1;
    nd.u[t] = a.uniforms[(int64_t)b * a.N + t];
    if (t < n && (t == 0 ? par != -1 : par < 0 || par >= t)) bad = true;
    if (t > 0 && t < n && par >= 0 && par < t) atomicOr(&nd.kids[par][t >> 5], 1u << (t & 31));
  }
  return __syncthreads_or(bad);
}

// f(j) for the elder siblings j of node t, in order.
template <typename F>
__device__ __forceinline__ void elder_siblings(const Nodes& nd, int t, F f) {
  const int par = nd.par[t];
  for (int k = par >> 5; k <= t >> 5; ++k) {
    uint32_t bits = nd.kids[par][k];
    if (k == t >> 5) bits &= (1u << (t & 31)) - 1u;
    for (; bits; bits &= bits - 1) f(32 * k + __builtin_ctz(bits));
  }
}

// Whether an elder sibling of node t has its token: refused again.
__device__ __forceinline__ bool repeated(const Nodes& nd, int t) {
  const int tok = nd.tok[t];
  bool found = false;
  elder_siblings(nd, t, [&](int j) { found |= nd.tok[j] == tok; });
  return found;
}

// Whether node t is taken once its elder siblings are refused; sp[]: the nodes'
// probabilities, -1 where refused whatever the rest (none, or repeated).
__device__ __forceinline__ bool taken(const VerifyArgs& a, const Nodes& nd, const double* sp,
                                      const double* sq, int t) {
  const double p = sp[t];
  if (!(p >= 0.0)) return false;
  if (a.greedy) return p > 0.0;
  if (a.drafts != nullptr) return (double)nd.u[t] * sq[t] < p;
  double left = 1.0;
  elder_siblings(nd, t, [&](int j) { left -= fmax(sp[j], 0.0); });
  return (double)nd.u[t] * left < p;
}

constexpr int WT = 1024;

// Row by row down the path, one workgroup per sequence.  A CU forms a row's sums
// at 64 values a clock at most (about 8 operations each): a row of 131072 takes 14 us,
// whatever its type.  Leaves the last node and its statistic for the draw; greedy:
// writes the token too.
template <typename T>
__global__ __launch_bounds__(WT) void verify_walk_kernel(VerifyArgs a, int* __restrict__ last,
                                                         Stat* __restrict__ out,
                                                         int* __restrict__ arrived) {
  __shared__ Nodes nd;
  __shared__ int path[MAXN];
  __shared__ double sp[MAXN];
  __shared__ Stat x[WT / 64];
  __shared__ int step;
  const int b = blockIdx.x, t = threadIdx.x;
  const int n = a.counts ? a.counts[b] : a.N;
  const bool bad = load_nodes(a, b, n, nd);
  const double c = a.inv_t * 1.4426950408889634074;
  int cur = 0, len = 0, end = -1;
  Stat st{-INFINITY, INT_MAX, 0.0};
  while (!bad && n > 0) {
    if (t == 0) {
      path[len] = cur;
      step = INT_MAX;
    }
    ++len;
    const Row<T> r((const T*)a.logits + b * a.logits_sb + cur * a.logits_sn, a.V);
    const int ng = r.granules();
    st = Stat{-INFINITY, INT_MAX, 0.0};
    // the next batch's loads run under this one's exponentials
    constexpr int U = sizeof(T) == 4 ? 4 : 2;  // (registers for 16 wavefronts)
    u32x4 raw[U], ahead[U];
    load_batch<T, U>(r, t, WT, ng, raw);
    for (int k = t; k < ng; k += U * WT) {
      load_batch<T, U>(r, k + U * WT, WT, ng, ahead);
      if (a.greedy)
        add_batch<T, false, U>(r, k, WT, raw, c, st);
      else
        add_batch<T, true, U>(r, k, WT, raw, c, st);
#pragma unroll
      for (int u = 0; u < U; ++u) raw[u] = ahead[u];
    }
    st = join_all<WT>(st, c, x);
    if (!is_distribution(st, a.greedy)) break;
    end = cur;
    const bool child = t > 0 && t < n && nd.par[t] == cur;
    if (child) {
      const int tok = nd.tok[t];
      sp[t] = tok < 0 || repeated(nd, t) ? -1.0
              : a.greedy ? (tok == st.at ? 1.0 : -1.0)
                         : exp2_64(((double)to_f32(r.x[tok]) - (double)st.m) * c) / st.s;
    }
    __syncthreads();
    if (child && taken(a, nd, sp, nullptr, t)) atomicMin(&step, t);
    __syncthreads();
    const int to = step;
    __syncthreads();  // read by all before it is written again
    if (to == INT_MAX) break;
    cur = to;
    end = -1;
  }
  __syncthreads();
  for (int j = t; j < a.N; j += WT) a.path[(int64_t)b * a.N + j] = j < len ? path[j] : -1;
  if (t == 0) {
    a.kept[b] = len;
    a.next[b] = a.greedy && end >= 0 ? st.at : -1;
    last[b] = end;
    out[b] = st;
    arrived[b] = 0;
  }
}

// A slice of the draw: U granules a thread; a segment is the 64 granules that a
// wavefront takes at a time.  The 64-bit exponentials (about 20 operations each)
// want many workgroups, the counter they all raise few: U = 1 while that leaves
// at most 256 (5 nodes, 32000 float32 values: 12.5 us, 16.4 with U = 4), else 4 (16
// sequences of 131072 values: 23 us with U = 1, 20 with 4).
constexpr int DT = 256;
__host__ __device__ __forceinline__ int draw_slices_of(int V, int E, int U) {
  return ((V + 2 * E - 2) / E + U * DT - 1) / (U * DT);
}

// The draw (and, ALL, the walk before it, over the statistics of all rows, by
// every workgroup of the sequence for itself).  Workgroup (slice, sequence): the
// weights of a slice's values in 64 bits, summed by segments in order; the last
// to arrive finds the slice, the segment and the value at which the running sum
// passes the point.  greedy: one workgroup per sequence, no draw.
template <typename T, bool ALL, int U>
__global__ __launch_bounds__(DT) void verify_draw_kernel(VerifyArgs a, const int* __restrict__ last,
                                                         const Stat* __restrict__ stats,
                                                         int nslices, int ndraw, double* sums,
                                                         int* __restrict__ arrived) {
  constexpr int E = Row<T>::E, DSEG = U * DT / 64;  // segments of a slice
  __shared__ Nodes nd;
  __shared__ Stat row[ALL ? 2 * MAXN : 1];  // nodes 0 .. n - 1, then the draft's
  __shared__ double sp[MAXN], sq[ALL ? MAXN : 1];
  __shared__ int pick[MAXN];  // the child taken of each node, then the path
  __shared__ int refused[MAXN];  // tokens of the last node's children
  __shared__ double seg[DSEG], wsum[DT / 64];
  __shared__ int sh[4];
  const int b = blockIdx.y, slice = blockIdx.x, t = threadIdx.x, lane = t & 63, w = t >> 6;
  const int N = a.N, V = a.V;
  const int n = a.counts ? a.counts[b] : N;
  const bool bad = load_nodes(a, b, n, nd);
  const double c = a.inv_t * 1.4426950408889634074;
  const T* logits = (const T*)a.logits + b * a.logits_sb;
  const T* drafts = (const T*)a.drafts + b * a.drafts_sb;
  const bool drafted = ALL && a.drafts != nullptr;
  int cur = -1;  // the node drawn after, -1 if its row is no distribution
  Stat st{}, dst{};
  if constexpr (ALL) {
    const int nrows = a.drafts != nullptr ? 2 * N - 1 : N;
    const bool node = !bad && t < n;
    static_assert(DT >= MAXN, "a thread per node");
    float x = 0.f, y = 0.f;
    if (node && t > 0 && nd.tok[t] >= 0) {
      x = to_f32(logits[nd.par[t] * a.logits_sn + nd.tok[t]]);
      if (drafted) y = to_f32(drafts[(t - 1) * a.drafts_sn + nd.tok[t]]);
    }
    // the rows' slices joined, 16 lanes a row, four rows' loads in flight
    const int nr = bad ? 0 : drafted ? 2 * n - 1 : n;
    for (int i0 = t / 16; i0 < nr; i0 += 4 * (DT / 16)) {
      Stat z[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int i = i0 + x * (DT / 16), j = t % 16;
        z[x] = Stat{-INFINITY, INT_MAX, 0.0};
        if (i < nr && j < nslices)
          z[x] = stats[((int64_t)b * nrows + (i < n ? i : N + i - n)) * nslices + j];
      }
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int i = i0 + x * (DT / 16);
        if (i >= nr) break;  // (a row's 16 lanes alike)
        for (int j = t % 16 + 16; j < nslices; j += 16)
          join(z[x], stats[((int64_t)b * nrows + (i < n ? i : N + i - n)) * nslices + j], c);
#pragma unroll
        for (int o = 8; o >= 1; o >>= 1) {
          Stat v;
          v.m = __shfl_xor(z[x].m, o, 16);
          v.at = __shfl_xor(z[x].at, o, 16);
          v.s = __shfl_xor(z[x].s, o, 16);
          join(z[x], v, c);
        }
        if (t % 16 == 0) row[i] = z[x];
      }
    }
    if (t < N) pick[t] = INT_MAX;
    __syncthreads();
    if (node && t > 0) {
      const Stat& r = row[nd.par[t]];
      const int tok = nd.tok[t];
      sp[t] = tok < 0 || repeated(nd, t) ? -1.0
              : !is_distribution(r, a.greedy) ? -1.0
              : a.greedy ? (tok == r.at ? 1.0 : -1.0)
                         : exp2_64(((double)x - (double)r.m) * c) / r.s;
      if (drafted) {
        const Stat& d = row[n + t - 1];
        sq[t] = exp2_64(((double)y - (double)d.m) * c) / d.s;
      }
    }
    __syncthreads();
    if (node && t > 0 && taken(a, nd, sp, sq, t)) atomicMin(&pick[nd.par[t]], t);
    __syncthreads();
    if (t == 0) {
      int len = 0, at = 0, lastn = -1;
      if (!bad && n > 0) {
        while (true) {
          const int to = pick[at];
          pick[len++] = at;  // len <= at: the picks of nodes behind are intact
          const bool ok = is_distribution(row[at], a.greedy);
          if (ok && to == INT_MAX) lastn = at;
          if (!ok || to == INT_MAX) break;
          at = to;
        }
      }
      sh[0] = lastn;
      sh[1] = len;
    }
    __syncthreads();
    cur = sh[0];
    if (cur >= 0) st = row[cur];
    if (slice == 0) {
      if (t < N) a.path[(int64_t)b * N + t] = t < sh[1] ? pick[t] : -1;
      if (t == 0) {
        a.kept[b] = sh[1];
        if (cur < 0 || a.greedy) a.next[b] = cur < 0 ? -1 : st.at;
      }
    }
    if (cur >= 0 && drafted && cur + 1 < n) dst = row[n + cur];
  } else {
    cur = last[b];
    if (cur >= 0) st = stats[b];
  }
  if (cur < 0 || a.greedy) return;
  if (t == 0) sh[3] = 0;
  __syncthreads();
  if (t > cur && t < n && nd.par[t] == cur) refused[atomicAdd(&sh[3], 1)] = nd.tok[t];
  __syncthreads();
  const int nref = sh[3];
  // weights, times the target's sum (with a draft: probabilities)
  const bool minus = drafted && cur + 1 < n && has_mass(dst.s);
  const double rp = minus ? 1.0 / st.s : 1.0, rq = minus ? 1.0 / dst.s : 0.0;
  const Row<T> r(logits + cur * a.logits_sn, V);
  const Row<T> dr(minus ? drafts + cur * a.drafts_sn : r.x, V);
  const bool alike = dr.lead == r.lead;  // granules of the two rows hold the same values
  const int ng = r.granules();
  auto weights = [&](int k, const u32x4& raw, bool all, double* wt) {
    float f[E];
    Row<T>::unpack(raw, f);
    const int v0 = r.first(k);
#pragma unroll
    for (int e = 0; e < E; ++e) wt[e] = exp2_64(((double)f[e] - (double)st.m) * c) * rp;
    if (all) return;
    if (minus) {
      if (alike) {
        Row<T>::unpack(dr.raw(k), f);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
          f[e] = v0 + e >= 0 && v0 + e < V ? to_f32(dr.x[v0 + e]) : -INFINITY;
      }
#pragma unroll
      for (int e = 0; e < E; ++e)
        wt[e] = fmax(wt[e] - exp2_64(((double)f[e] - (double)dst.m) * c) * rq, 0.0);
    } else if (!drafted) {  // (a refused child of probability 0 changes nothing)
      for (int i = 0; i < nref; ++i) {
        const int at = refused[i] - v0;  // (hardly ever in the granule)
        if (at >= 0 && at < E) {
#pragma unroll
          for (int e = 0; e < E; ++e)
            if (at == e) wt[e] = 0.0;
        }
      }
    }
  };
  // the sums of a slice's segments, to seg[0 .. DSEG)
  auto slice_sums = [&](int sl, bool all, double* seg) {
    u32x4 raw[U];
    const int k0 = sl * U * DT + t;
    load_batch<T, U>(r, k0, DT, ng, raw);
    double x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      double wt[E];
      x[u] = 0.0;
      if (k0 + u * DT < ng) {
        weights(k0 + u * DT, raw[u], all, wt);
#pragma unroll
        for (int e = 0; e < E; ++e) x[u] += wt[e];
      }
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1)
#pragma unroll
      for (int u = 0; u < U; ++u) x[u] += __shfl_xor(x[u], o, 64);
    if (lane == 0)
#pragma unroll
      for (int u = 0; u < U; ++u) seg[u * (DT / 64) + w] = x[u];
    __syncthreads();
  };
  double* sums_b = sums + (int64_t)b * ndraw * DSEG;
  slice_sums(slice, false, seg);
  if (w == 0) {
    // Device-scope accesses on both sides, past the caches, so the order is all
    // that is left to see to: the sums have arrived before the count is raised.
    // (A release here would write back the XCD's whole L2, an acquire empty it.)
    if (t < DSEG)
      __hip_atomic_store(sums_b + slice * DSEG + t, seg[t], __ATOMIC_RELAXED,
                         __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (t == 0)
      sh[2] = __hip_atomic_fetch_add(arrived + b, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (sh[2] != ndraw - 1) return;
  // The last of the sequence: every segment's sum is there.  Thread j's share of
  // them runs in order, then the shares' sums.
  const int nseg = ndraw * DSEG, share = (nseg + DT - 1) / DT;
  const int j0 = min(t * share, nseg), j1 = min(j0 + share, nseg);
  double part, incl, total;
  constexpr int BATCH = 4;  // sums loaded at once (131072 16-bit values: a share of 2)
  double x[BATCH];
  auto load_sums = [&](int j) {  // 0 behind the share
#pragma unroll
    for (int e = 0; e < BATCH; ++e)
      x[e] = j + e < j1 ? __hip_atomic_load(sums_b + j + e, __ATOMIC_RELAXED,
                                            __HIP_MEMORY_SCOPE_AGENT)
                        : 0.0;
  };
  auto running = [&]() {
    part = 0.0;
    for (int j = j0; j < j1; j += BATCH) {
      load_sums(j);
#pragma unroll
      for (int e = 0; e < BATCH; ++e) part += x[e];
    }
    incl = part;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double y = __shfl_up(incl, o, 64);
      if (lane >= o) incl += y;
    }
    __syncthreads();
    if (lane == 63) wsum[w] = incl;
    __syncthreads();
    double below = 0.0;
    total = 0.0;
#pragma unroll
    for (int j = 0; j < DT / 64; ++j) {
      if (j == w) below = total;
      total += wsum[j];
    }
    incl += below;
  };
  running();
  // rounding can leave no mass where all of it was on refused tokens: the draw is
  // then from the row itself
  const bool all = !(total > 0.0);
  if (all) {
    for (int j = 0; j < ndraw; ++j) {
      slice_sums(j, true, seg);
      if (t < DSEG)
        __hip_atomic_store(sums_b + j * DSEG + t, seg[t], __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_AGENT);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
    }
    running();
  }
  const double point = (double)nd.u[0] * total;
  // the first share that passes the point (the last one, where sums of two orders
  // leave the point behind them), then its first segment
  if (t == 0) sh[3] = (nseg - 1) / share;
  __syncthreads();
  if (incl > point) atomicMin(&sh[3], t);
  __syncthreads();
  if (t == sh[3]) {
    double before = incl - part;
    int pick = j0;
    double at = before;
    bool open = true;
    for (int g = j0; g < j1; g += BATCH) {
      if (share > BATCH) load_sums(g);  // (else they are still there)
#pragma unroll
      for (int e = 0; e < BATCH; ++e) {
        if (open && x[e] > 0.0) {  // (a segment of no weight is never picked)
          pick = g + e;
          at = before;
        }
        open = open && !(before + x[e] > point);
        before += x[e];
      }
    }
    sh[0] = pick;
    seg[0] = at;
  }
  __syncthreads();
  if (w != 0) return;
  const int k = 64 * sh[0] + lane;
  const double before = seg[0];
  double wt[E], sum = 0.0;
  int hit = INT_MAX, any = -1;
#pragma unroll
  for (int e = 0; e < E; ++e) wt[e] = 0.0;
  if (k < ng) weights(k, r.raw(k), all, wt);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    sum += wt[e];
    if (wt[e] > 0.0) any = r.first(k) + e;
  }
  double run = sum;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double y = __shfl_up(run, o, 64);
    if (lane >= o) run += y;
  }
  run = before + (run - sum);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    run += wt[e];
    if (hit == INT_MAX && wt[e] > 0.0 && run > point) hit = r.first(k) + e;
  }
  // The first value that passes the point; sums of two orders may leave the point
  // behind the segment's last value.
  const uint64_t hits = __ballot(hit != INT_MAX), some = __ballot(any >= 0);
  const int first = hits ? __shfl(hit, __ffsll((unsigned long long)hits) - 1, 64) : -1;
  const int end = some ? __shfl(any, 63 - __clzll((long long)some), 64) : -1;
  if (lane == 0) a.next[b] = hits ? first : end;
}

// ------------------------------------------------------------------ keep
// Row L + path[j] to row L + j for j < kept, in every cache.  path rises, so
// path[j] >= j: a row is overwritten only after the only move that reads it (an
// earlier j).  A thread moves the same 16 bytes of every row, in order of j, so
// its own program order is all the ordering that needs.  Bound by its launch: 32
// layers of 16 sequences 3.8 us.
struct KeepPtrs {
  char *k[KEEP_CACHES], *v[KEEP_CACHES];
  const int32_t* lens[KEEP_CACHES];
  int32_t* lens_out[KEEP_CACHES];
};

// One workgroup per (cache, sequence): nothing else reads or writes lens[b] of
// that cache, so lens_out may be lens itself.
template <typename U>
__global__ __launch_bounds__(256) void cache_keep_kernel(KeepPtrs p, const int32_t* __restrict__ path,
                                                         const int32_t* __restrict__ kept, int N,
                                                         int Hkv, int Smax, int row_units) {
  __shared__ int sp[MAXN];
  const int c = blockIdx.x, b = blockIdx.y, t = threadIdx.x;
  const int L = p.lens[c][b], n = kept[b];
  bool bad = n < 0 || n > N || L < 0;
  if (!bad && t < n) {
    const int x = path[(int64_t)b * N + t];
    sp[t] = x;
    const int before = t > 0 ? path[(int64_t)b * N + t - 1] : -1;
    bad = x <= before || x >= N || (int64_t)L + x >= Smax;
  }
  bad = __syncthreads_or(bad);
  if (t == 0) p.lens_out[c][b] = bad ? L : L + n;
  if (bad) return;
  constexpr int J = 8;  // rows in flight
  for (int i = t; i < 2 * Hkv * row_units; i += 256) {
    const int which = i / (Hkv * row_units), u = i % (Hkv * row_units);
    const int h = u / row_units, col = u % row_units;
    U* base = (U*)(which ? p.v[c] : p.k[c]) + (((int64_t)b * Hkv + h) * Smax + L) * row_units + col;
    for (int j0 = 0; j0 < n; j0 += J) {
      U x[J];
#pragma unroll
      for (int j = 0; j < J; ++j)
        if (j0 + j < n) x[j] = base[(int64_t)sp[j0 + j] * row_units];
#pragma unroll
      for (int j = 0; j < J; ++j)
        if (j0 + j < n && sp[j0 + j] != j0 + j) base[(int64_t)(j0 + j) * row_units] = x[j];
    }
  }
}

}  // namespace

namespace {

size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

struct VerifyWs {
  int* arrived;   // [B]
  int* last;      // [B]
  Stat* stats;    // all rows: [B][rows][slices]; walk: [B]
  double* sums;   // [B][segments of the draw]
  bool all_rows;
  int rows, slices, draw, unit;  // unit: granules a thread of the draw
  size_t bytes;
};
VerifyWs verify_carve(const VerifyArgs& a, void* p) {
  const int el = a.dtype == F32 ? 4 : 2;
  VerifyWs w;
  w.slices = slices_of(a.V, 16 / el);
  w.unit = (int64_t)a.B * draw_slices_of(a.V, 16 / el, 1) <= 256 ? 1 : 4;
  w.draw = draw_slices_of(a.V, 16 / el, w.unit);
  w.rows = a.drafts != nullptr ? 2 * a.N - 1 : a.N;
  // All rows take B N el / 5 TB/s per value of the vocabulary, a walk about 110 ps
  // per value and level of the longest path: equal at 2200 bytes a value for trees,
  // whose paths have some four levels (64 trees of 64 nodes, 131072 16-bit values: walk
  // 73 us, all rows 260; 16 of them 67 and 46).  A chain's can be as long as the chain
  // (64 of 18 nodes, wholly accepted: walk 264 us, all rows 97), and a draft's rows come
  // with chains.  A chain, or another deep tree, given by its parents is not known for one
  // here and takes the walk.
  w.all_rows = a.parents == nullptr || (int64_t)a.B * a.N * el <= 2200;
  char* c = (char*)p;
  w.arrived = (int*)c;
  c += up256((size_t)a.B * 4);
  w.last = (int*)c;
  c += up256((size_t)a.B * 4);
  w.stats = (Stat*)c;
  c += up256((size_t)a.B * (w.all_rows ? (size_t)w.rows * w.slices : 1) * sizeof(Stat));
  w.sums = (double*)c;
  c += up256((size_t)a.B * w.draw * w.unit * (DT / 64) * sizeof(double));
  w.bytes = (size_t)(c - (char*)p);
  return w;
}

template <typename T>
int verify_typed(const VerifyArgs& a, void* workspace) {
  const VerifyWs w = verify_carve(a, workspace);
  if (w.all_rows) {
    auto kernel = a.greedy ? verify_stats_kernel<T, false> : verify_stats_kernel<T, true>;
    KF_LAUNCH("verify_stats", kernel, dim3(w.slices, w.rows, a.B), dim3(ST), 0, a.stream, a,
              w.stats, w.arrived);
    KF_CHECK_LAUNCH();
    auto draw = w.unit == 1 ? verify_draw_kernel<T, true, 1> : verify_draw_kernel<T, true, 4>;
    KF_LAUNCH("verify_draw", draw, dim3(a.greedy ? 1 : w.draw, a.B), dim3(DT), 0, a.stream, a,
              w.last, w.stats, w.slices, w.draw, w.sums, w.arrived);
    KF_CHECK_LAUNCH();
    return KF_OK;
  }
  KF_LAUNCH("verify_walk", verify_walk_kernel<T>, dim3(a.B), dim3(WT), 0, a.stream, a, w.last,
            w.stats, w.arrived);
  KF_CHECK_LAUNCH();
  if (a.greedy) return KF_OK;
  KF_LAUNCH("verify_draw", (w.unit == 1 ? verify_draw_kernel<T, false, 1>
                                        : verify_draw_kernel<T, false, 4>),
            dim3(w.draw, a.B), dim3(DT), 0, a.stream, a, w.last, w.stats, w.slices, w.draw, w.sums,
            w.arrived);
  KF_CHECK_LAUNCH();
  return KF_OK;
}

}  // namespace

size_t verify_workspace(const VerifyArgs& a) { return verify_carve(a, nullptr).bytes; }

int verify_drafts(const VerifyArgs& a, void* workspace) {
  switch (a.dtype) {
    case F32: return verify_typed<float>(a, workspace);
    case BF16: return verify_typed<bf16>(a, workspace);
    case F16: return verify_typed<_Float16>(a, workspace);
  }
  set_error("unsupported dtype %d", a.dtype);
  return KF_ERR_UNSUPPORTED;
}

int cache_keep(void* const* k, void* const* v, const int32_t* const* lens,
               int32_t* const* lens_out, int n_caches, const int32_t* path, const int32_t* kept,
               int N, int B, int Hkv, int Smax, int D, int dtype, hipStream_t stream) {
  const int bytes = D * (dtype == F32 ? 4 : 2);
  for (int c0 = 0; c0 < n_caches; c0 += KEEP_CACHES) {
    const int nc = std::min(KEEP_CACHES, n_caches - c0);
    KeepPtrs p = {};
    uintptr_t low = (uintptr_t)bytes;
    for (int c = 0; c < nc; ++c) {
      p.k[c] = (char*)k[c0 + c];
      p.v[c] = (char*)v[c0 + c];
      p.lens[c] = lens[c0 + c];
      p.lens_out[c] = lens_out[c0 + c];
      low |= (uintptr_t)p.k[c] | (uintptr_t)p.v[c];
    }
    const dim3 grid(nc, B);
    if (low % 16 == 0)
      KF_LAUNCH("cache_keep", cache_keep_kernel<u32x4>, grid, dim3(256), 0, stream, p, path, kept,
                N, Hkv, Smax, bytes / 16);
    else
      KF_LAUNCH("cache_keep", cache_keep_kernel<uint16_t>, grid, dim3(256), 0, stream, p, path,
                kept, N, Hkv, Smax, bytes / 2);
    KF_CHECK_LAUNCH();
  }
  return KF_OK;
}

}  // namespace kf
