// Beam search after the model's forward: the selection over beams and vocabulary, and
// the caches' rows of the beams that go on.
//
// Selection: of W beams with scores s_w and logits x_w over V tokens, the K largest of
//   t_wv = s_w + x_wv - log sum_u exp x_wu,
// equals by the lowest w, then v.  Within a beam t rises with x, so a row's K largest
// logits are all that can be picked of it, and where a beam's score leaves no bits for
// their differences (equal t), x still has their order:
//  1. rows   a workgroup per slice of a row: the slice's maximum and sum of
//            exponentials, and its K largest logits
//  2. pick   a workgroup per group: the rows' sums joined, then the K largest of the
//            W x slices x K candidates, in 64 bits
// Every logit is read once.  HBM bounds the first (bfloat16 rows of 131072: 32 x 8 take
// 17.5 us, 3.8 TB/s; 128 x 8 60 with the pick), two dependent launches the smallest calls
// (4 rows of 32000: 5.8 and 5 us).
#include "kf_common.h"
#include "kf_internal.h"
#include "kf_mfma.h"
#include "kf_row.h"
#include "kf_stream.h"

#include <algorithm>
#include <limits>
#include <type_traits>

namespace kf {

namespace {

// ------------------------------------------------------------------ the K largest
// of values spread over a workgroup of 256, largest first, equals by the lowest index (of
// 64-bit values: the lowest key).
//
// The workgroup's values fall into 64 groups (lane l of the four wavefronts); the K-th
// largest of the groups' maxima is at most the K-th largest value, and few values are
// above it (64 ln(64 / (64 - K)) of independent ones), so those are gathered and ordered
// by counting.  Many of the 64 picked leave many above (all, at 64), which are ordered in
// their number's square: then the 256 threads are the groups.  More than CAP of them (values
// that are ordered against the groups, or mostly equal) are taken one at a time.
constexpr int NT = 256, CAP = 1024;

template <typename V>
struct TopLds {
  using Index = typename std::conditional<sizeof(V) == 4, int, unsigned long long>::type;
  V top[NT];
  V val[CAP];
  Index idx[CAP], best;
  int count;
  V edge, red[NT / 64];
  __device__ __forceinline__ void add(V x, Index i) {
    const int at = atomicAdd(&count, 1);
    if (at < CAP) {
      val[at] = x;
      idx[at] = i;
    }
  }
};

__device__ __forceinline__ float lane_of(float x, int j) {
  return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), j));
}
__device__ __forceinline__ double lane_of(double x, int j) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)u, j),
                 hi = __builtin_amdgcn_readlane((uint32_t)(u >> 32), j);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// A value that K of the workgroup's values reach, if there are as many above -inf, given
// each thread's largest in lds.top: by one wavefront, each lane gets it.
template <typename V>
__device__ __forceinline__ V top_bound(int K, const TopLds<V>& lds) {
  const int lane = threadIdx.x & 63;
  V g[NT / 64], edge = INFINITY;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) g[i] = lds.top[lane + 64 * i];
  // (The launches of 16 x 16 rows of 131072 in us, by 64 and by 256: rows at 32 21, 38, at 48
  // 25, 34, at 56 32, 35, at 63 2200, 42; pick at 32 9.5, 14, at 40 11, 15, at 48 23.6, 17.)
  if (K <= (sizeof(V) == 4 ? 48 : 40)) {
#pragma unroll
    for (int i = 1; i < NT / 64; ++i) g[0] = fmax(g[0], g[i]);
    int above = 0;
#pragma unroll
    for (int j = 0; j < 64; ++j) above += lane_of(g[0], j) > g[0];
    if (above < K) edge = g[0];
  } else {
    int above[NT / 64] = {};
#pragma unroll
    for (int i = 0; i < NT / 64; ++i)
#pragma unroll
      for (int j = 0; j < 64; ++j) {
        const V x = lane_of(g[i], j);
#pragma unroll
        for (int k = 0; k < NT / 64; ++k) above[k] += x > g[k];
      }
#pragma unroll
    for (int i = 0; i < NT / 64; ++i)
      if (above[i] < K) edge = fmin(edge, g[i]);
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) edge = fmin(edge, __shfl_xor(edge, o, 64));
  return edge;
}

// The K first of the n <= CAP gathered values, by out(place, value, index).
template <typename V, typename Out>
__device__ __forceinline__ void top_order(int K, int n, Out out, const TopLds<V>& lds) {
  for (int a = threadIdx.x; a < n; a += NT) {
    const V x = lds.val[a];
    const auto i = lds.idx[a];
    int place = 0;
#pragma unroll 4
    for (int b = 0; b < n; ++b) {
      const V y = lds.val[b];
      place += (y > x) | ((y == x) & (lds.idx[b] < i));
    }
    if (place < K) out(place, x, i);
  }
}

// The same, one at a time: each(f) gives f(value, index) for the thread's values (f says
// whether to go on, here always); there are K of them.
template <typename V, typename Each, typename Out>
__device__ __forceinline__ void top_one_by_one(int K, Each each, Out out, TopLds<V>& lds) {
  using Index = typename TopLds<V>::Index;
  const int t = threadIdx.x;
  V last = INFINITY;
  Index after = 0;  // (no value is as large)
  for (int place = 0; place < K; ++place) {
    // the largest value behind (last, after), then the lowest index that has it
    V x = -INFINITY;
    each([&](V v, Index i) __attribute__((always_inline)) {
      if (v < last || (v == last && i > after)) x = fmax(x, v);
      return true;
    });
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) x = fmax(x, __shfl_xor(x, o, 64));
    __syncthreads();
    if ((t & 63) == 0) lds.red[t >> 6] = x;
    if (t == 0) lds.best = std::numeric_limits<Index>::max();
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) x = fmax(x, lds.red[w]);
    Index mine = std::numeric_limits<Index>::max();
    each([&](V v, Index i) __attribute__((always_inline)) {
      if (v == x && (v < last || i > after)) mine = min(mine, i);
      return true;
    });
    if (mine != std::numeric_limits<Index>::max()) atomicMin(&lds.best, mine);
    __syncthreads();
    if (t == 0) out(place, x, lds.best);
    last = x;
    after = lds.best;
  }
}

// ------------------------------------------------------------------ rows
struct SliceSum {
  float m;   // maximum
  double s;  // sum of exp(x - m); not positive and finite: no distribution
};
struct Candidate {
  float x;
  int v;  // -1: none
};

constexpr int U = 8;  // granules of a thread
// Slices of a row of V values, in granules of E.
int slices_of(int V, int E) { return ((V + E - 1) / E + NT * U - 1) / (NT * U); }

// A granule of -inf, and one without its first k values.
template <typename T>
__device__ __forceinline__ u32x4 none_of() {
  const uint32_t n = sizeof(T) == 4                ? 0xff800000u
                     : std::is_same<T, bf16>::value ? 0xff80ff80u
                                                    : 0xfc00fc00u;
  return u32x4{n, n, n, n};
}
template <typename T>
__device__ __forceinline__ void drop_first(u32x4& x, int k) {
  constexpr int P = 4 / sizeof(T);  // values of a dword
  const u32x4 none = none_of<T>();
#pragma unroll
  for (int d = 0; d < 4; ++d)
    x[d] = k >= P * (d + 1)                ? none[d]
           : P == 2 && k == P * d + 1      ? (x[d] & 0xffff0000u) | (none[d] & 0xffffu)
                                           : x[d];
}

// Granules that hold a value of the bound or more, put aside to be looked through by all
// threads: eight tests and appends in each thread's own code would cost as much as the
// sums.
constexpr int GRANULES = 256;

// Workgroup (row, slice).  Exponentials are float32 instructions of (x - m) log2 e, m the
// thread's maximum so far, sums of a thread's values in 32 bits, of the threads' in 64.
// The difference is formed first: its rounding, the product's and log2 e's are 2.25 steps
// of 2^-24 of it, whatever x (one rounding of x log2 e - m log2 e is as fast, but is off by
// what m log2 e was rounded by: too much for an exponential from 1e9 on, and a sum that is
// 1 was not 1).  Of V <= 2^20 values |log2 p| is 21.5 on average at most, the instruction
// adds 2^-22, a thread's sums 24 steps: a row's log-sum is off by less than 4e-6 (measured
// 1.4e-7).  In 64 bits an exponential would take more than all else that a thread does for
// a value.
// A thread's granules are counted from the row's first value, whatever its alignment (the
// loads may be unaligned): rows of equal values have equal sums, to the last bit, and their
// beams' candidates are equals.
template <typename T>
__global__ __launch_bounds__(NT, 4) void select_rows_kernel(SelectArgs a,
                                                            SliceSum* __restrict__ sums,
                                                            Candidate* __restrict__ best) {
  __shared__ TopLds<float> lds;
  __shared__ u32x4 hot[GRANULES];
  __shared__ int hot_at[GRANULES], hots;
  __shared__ float parts[NT];
  constexpr int E = Row<T>::E, BATCH = 4;  // granules whose maximum is taken at once
  const int g = blockIdx.x / a.W, w = blockIdx.x % a.W, t = threadIdx.x, lane = t & 63;
  if (!(fabsf(a.scores[blockIdx.x]) < INFINITY)) return;  // a beam that is not in use
  const T* row = (const T*)a.logits + g * a.logits_sg + w * a.logits_sw;
  const int v0 = (blockIdx.y * (NT * U) + t) * E;  // the thread's first value
  // A granule that would pass the row's end begins E values before it, and leaves out those
  // that are another's.
  auto first = [&](int u) {
    const int v = v0 + u * NT * E;
    return a.V >= E ? min(v, a.V - E) : v;
  };
  u32x4 raw[U];
  if (a.V >= E) {
#pragma unroll
    for (int u = 0; u < U; ++u) __builtin_memcpy(&raw[u], row + first(u), 16);
  } else {
    T x[E];
#pragma unroll
    for (int e = 0; e < E; ++e)
      x[e] = t == 0 && e < a.V ? row[min(e, a.V - 1)] : from_f32<T>(-INFINITY);
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = none_of<T>();
    __builtin_memcpy(&raw[0], x, 16);
  }
  if ((blockIdx.y + 1) * (NT * U * E) > a.V && a.V >= E) {
#pragma unroll
    for (int u = 0; u < U; ++u) drop_first<T>(raw[u], v0 + u * NT * E - first(u));
  }
  float gm[U], m = -INFINITY, part = 0.f;
#pragma unroll
  for (int b = 0; b < U; b += BATCH) {
    const float old = m;
#pragma unroll
    for (int u = b; u < b + BATCH; ++u) {
      float f[E];
      Row<T>::unpack(raw[u], f);
      gm[u] = f[0];
#pragma unroll
      for (int e = 1; e < E; ++e) gm[u] = fmaxf(gm[u], f[e]);
      m = fmaxf(m, gm[u]);
      mfma::settle(raw[u]);  // (kept as they are: unpacked they would take twice the registers)
    }
    if (old != -INFINITY && m > old) part *= fast_exp2((old - m) * kLog2e);
    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int u = b; u < b + BATCH; ++u) {
      float f[E], x = 0.f;
      Row<T>::unpack(raw[u], f);
#pragma unroll
      for (int e = 0; e < E; ++e) x += fast_exp2((f[e] - ref) * kLog2e);
      part += x;
      mfma::settle(raw[u]);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  // One wavefront finds the bound, another the sum: all four would spend on them what they
  // spend on the values.
  lds.top[t] = m;
  parts[t] = part;
  if (t == 0) lds.count = hots = 0;
  __syncthreads();
  const int64_t at = (int64_t)blockIdx.x * gridDim.y + blockIdx.y;
  if (t >> 6 == 0) {
    const float x = top_bound(a.K, lds);
    if (lane == 0) lds.edge = x;
  } else if (t >> 6 == 1) {
    constexpr double L = 1.4426950408889634074;
    float M = -INFINITY;
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) M = fmaxf(M, lds.top[lane + 64 * i]);
    M = wave_max(M);
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) {
      const double x = lds.top[lane + 64 * i];
      const float p = parts[lane + 64 * i];
      if (x == -INFINITY)
        s += p != p ? p : 0.f;
      else
        s += (double)p * exp2_64((x - (double)M) * L);
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
    if (lane == 0) sums[at] = SliceSum{M, s};
  }
  __syncthreads();
  const float edge = lds.edge;
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (gm[u] >= edge && gm[u] > -INFINITY) {
      const int x = atomicAdd(&hots, 1);
      if (x < GRANULES) {
        hot[x] = raw[u];
        hot_at[x] = first(u);
      }
    }
  __syncthreads();
  Candidate* out = best + at * a.K;
  auto put = [&](int place, float x, int v) { out[place] = Candidate{x, v}; };
  const int nh = hots;
  for (int x = t; nh <= GRANULES && x < nh * E; x += NT) {
    const float f = to_f32(((const T*)hot)[x]);
    if (f >= edge && f > -INFINITY) lds.add(f, hot_at[x / E] + x % E);
  }
  __syncthreads();
  int n = lds.count;
  if (nh <= GRANULES && n <= CAP) {
    top_order(a.K, n, put, lds);
  } else {  // (of E values and more)
    auto granule = [&](int u, float* f) {
      u32x4 x;
      __builtin_memcpy(&x, row + first(u), 16);
      drop_first<T>(x, v0 + u * NT * E - first(u));
      Row<T>::unpack(x, f);
    };
    auto each = [&](auto g) {
#pragma unroll 1
      for (int u = 0; u < U; ++u) {
        float f[E];
        granule(u, f);
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (f[e] > -INFINITY) g(f[e], first(u) + e);
      }
    };
    // Mostly equal values (tokens masked by the type's lowest one): the bound is the K-th
    // largest value itself where fewer than K are above it, and the lowest tokens that have
    // it follow those.
    __syncthreads();
    if (t == 0) lds.count = 0;
    __syncthreads();
    each([&](float x, int v) {
      if (x > edge) lds.add(x, v);
    });
    __syncthreads();
    n = lds.count;
    if (n < a.K) {
      top_order(a.K, n, put, lds);
#pragma unroll 1
      for (int u = 0; u < U && n < a.K; ++u) {
        float f[E];
        granule(u, f);
        int mine = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) mine += f[e] == edge;
        const int end = wave_prefix(mine);
        __syncthreads();
        if (lane == 63) hot_at[t >> 6] = end;
        __syncthreads();
        int place = n + end - mine;
#pragma unroll
        for (int w = 0; w < NT / 64; ++w) {
          place += w < t >> 6 ? hot_at[w] : 0;
          n += hot_at[w];
        }
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (f[e] == edge) {
            if (place < a.K) put(place, edge, first(u) + e);
            ++place;
          }
      }
    } else {
      top_one_by_one(a.K, each, put, lds);
      n = a.K;
    }
  }
  for (int i = n + t; i < a.K; i += NT) put(i, -INFINITY, -1);
}

// ------------------------------------------------------------------ pick
// A candidate's key: its beam, then its logit from the largest down (equal totals of
// one beam are equal logits, or such as its score leaves no bits for), then its token.
using Key = TopLds<double>::Index;
constexpr int VBITS = 20;
static_assert(KF_VERIFY_MAX_VOCAB <= 1 << VBITS && KF_BEAM_MAX <= 1 << (32 - VBITS), "a key's bits");
__device__ __forceinline__ Key key_of(int w, float x, int v) {
  const uint32_t u = __float_as_uint(x + 0.f);  // (-0 and 0 are equals)
  const uint32_t down = u >> 31 ? u : u ^ 0x7fffffffu;
  return (Key)w << (32 + VBITS) | (Key)down << VBITS | (Key)v;
}

// A slice's candidates are a list in order.  `parts` threads take the list's places in turn
// (more than 256 lists: a thread takes several), and leave it at the first that is below the
// bound, so of slices x K candidates a beam little more than K in all are looked at (8 x 8
// slices of 16: 8.5 us with the call's launch, 14 when all were).  What a
// thread begins with is asked for before anything is waited for: each round trip to what
// other compute units wrote costs as much as the rest.
__global__ __launch_bounds__(NT) void select_pick_kernel(SelectArgs a,
                                                         const SliceSum* __restrict__ sums,
                                                         const Candidate* __restrict__ best,
                                                         int slices) {
  __shared__ TopLds<double> lds;
  __shared__ double score[KF_BEAM_MAX], lse[KF_BEAM_MAX];
  const int g = blockIdx.x, t = threadIdx.x, W = a.W;
  constexpr double L = 1.4426950408889634074;
  const int lists = W * slices, parts = max(NT / lists, 1);
  const Candidate* c = best + (int64_t)g * lists * a.K;
  // the thread's first list, and its first two places of it
  const int l0 = t % lists, r0 = t / lists;
  const Candidate *begin = c + (int64_t)l0 * a.K;
  const Candidate one = begin[min(r0, a.K - 1)], two = begin[min(r0 + parts, a.K - 1)];
  // a row per group of lanes, all rows at once
  const int lanes = W <= 4 ? 64 : W <= 8 ? 32 : W <= 16 ? 16 : W <= 32 ? 8 : 4;
  {
    const int w = min(t / lanes, W - 1), x = t % lanes;
    const SliceSum* row = sums + ((int64_t)g * W + w) * slices;
    const float sc = a.scores[(int64_t)g * W + w];
    const SliceSum y = row[min(x, slices - 1)];
    const bool live = fabsf(sc) < INFINITY;  // (else what the slices hold was not written)
    double s = 0.0;
    float M = -INFINITY;
    if (live) {
      M = x < slices ? y.m : -INFINITY;
      for (int i = x + lanes; i < slices; i += lanes) M = fmaxf(M, row[i].m);
    }
    for (int o = lanes / 2; o >= 1; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
    if (live) {
      float m = y.m;
      double e = y.s;
      for (int i = x; i < slices;) {
        s += m == M ? e : e * exp2_64(((double)m - (double)M) * L);
        i += lanes;
        m = row[min(i, slices - 1)].m;
        e = row[min(i, slices - 1)].s;
      }
    }
    for (int o = lanes / 2; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
    const bool ok = live && s > 0.0 && s < INFINITY;
    if (x == 0 && t / lanes < W) {
      score[w] = ok ? (double)sc : -INFINITY;
      lse[w] = ok ? (double)M + log(s) : 0.0;
    }
  }
  __syncthreads();
  // f(value, key) for the thread's candidates, list by list, in order; f says whether to
  // go on in the list.
  auto walk = [&](auto f) __attribute__((always_inline)) {
    // (in registers: a choice between the two as they are is made a choice of addresses)
    float x1 = one.x, x2 = two.x;
    int v1 = one.v, v2 = two.v;
    asm("" : "+v"(x1), "+v"(v1), "+v"(x2), "+v"(v2));
    if (r0 >= parts) return;  // (threads that are too few for another place of every list)
    for (int l = l0; l < lists; l += NT) {
      const int w = l / slices;
      const double sc = score[w], ls = lse[w];
      if (sc == -INFINITY) continue;  // (what its slices hold was not written)
      for (int r = r0; r < a.K; r += parts) {
        const bool again = r != r0;
        float y = again ? x2 : x1;
        int v = again ? v2 : v1;
        if (l != l0 || r > r0 + parts) {
          const Candidate z = c[(int64_t)l * a.K + r];
          y = z.x, v = z.v;
        }
        if (v < 0 || !f(sc + ((double)y - ls), key_of(w, y, v))) break;
      }
    }
  };
  double own = -INFINITY;
  walk([&](double x, Key) {
    own = fmax(own, x);
    return false;
  });
  lds.top[t] = own;
  if (t == 0) lds.count = 0;
  __syncthreads();
  double edge = top_bound(a.K, lds);  // (each wavefront by itself: no other barrier)
  auto gather = [&](double x, Key k) {
    if (x < edge) return false;
    lds.add(x, k);
    return true;
  };
  walk(gather);
  __syncthreads();
  // Where fewer lists than K hold the K largest (few beams' scores are far above the others'),
  // the lists' beginnings bound little, and up to K candidates of each of those lists pass
  // (16 x 16 rows of 131072, 128 picked: 3.4 ms, now 0.12).  Then all candidates are dealt
  // out, 256 at a time, each deal turned against the last, so that no thread has two of the
  // first places of a few lists.  (That takes less than ordering what passed, by its
  // square, unless there are many candidates: 64 lists of 16 that all pass 40 us for 173,
  // 512 lists of 128 81 for 67.)
  const int passed = lds.count;
  if (passed > CAP || (passed > NT && passed * passed > 16 * lists * a.K)) {
    own = -INFINITY;
#pragma unroll 1
    for (int r = 0; r * NT < lists * a.K; ++r) {
      const int i = r * NT + ((t + 79 * r) & (NT - 1));
      if (i >= lists * a.K) continue;
      const int w = i / a.K / slices;
      if (score[w] == -INFINITY) continue;
      const Candidate x = c[i];
      if (x.v >= 0) own = fmax(own, score[w] + ((double)x.x - lse[w]));
    }
    __syncthreads();
    lds.top[t] = own;
    if (t == 0) lds.count = 0;
    __syncthreads();
    edge = fmax(edge, top_bound(a.K, lds));
    walk(gather);
    __syncthreads();
  }
  const int64_t at = (int64_t)g * a.K;
  auto put = [&](int place, double x, Key k) {
    a.out_scores[at + place] = (float)x;
    a.parents[at + place] = (int)(k >> (32 + VBITS));
    a.tokens[at + place] = (int64_t)(k & ((1 << VBITS) - 1));
  };
  int m = lds.count;
  if (m <= CAP) {
    top_order(a.K, m, put, lds);
  } else {
    top_one_by_one(a.K, walk, put, lds);
    m = a.K;
  }
  for (int i = m + t; i < a.K; i += NT) {
    a.out_scores[at + i] = -INFINITY;
    a.parents[at + i] = -1;
    a.tokens[at + i] = -1;
  }
}

// ------------------------------------------------------------------ reorder
// Sequence w of a group takes the rows of sequence parents[w]: a thread moves the same
// 16 bytes of a row of all its group's sequences, and reads every one that is continued
// elsewhere before it writes any.  No other thread touches them, so the move needs no
// second buffer, whatever the parents (cycles, several children of one).
__device__ __forceinline__ uint64_t uniform64(uint64_t x) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)x),
                 hi = __builtin_amdgcn_readfirstlane((uint32_t)(x >> 32));
  return (uint64_t)hi << 32 | lo;
}

struct ReorderPtrs {
  char *k[KEEP_CACHES], *v[KEEP_CACHES];
};

template <typename U, int MW>
__global__ __launch_bounds__(256) void cache_reorder_kernel(
    ReorderPtrs p, const int32_t* __restrict__ lens, const int32_t* __restrict__ parents, int W,
    int Hkv, int Smax, int row_units) {
  const int gh = blockIdx.x, g = gh / Hkv, h = gh % Hkv, c = blockIdx.y >> 1;
  char* base = blockIdx.y & 1 ? p.v[c] : p.k[c];
  // sequence w's children other than itself as bits, and the units they take
  __shared__ uint64_t kids[KF_BEAM_MAX];
  __shared__ int64_t last[KF_BEAM_MAX];
  __shared__ int most;
  const int t = threadIdx.x;
  if (t < KF_BEAM_MAX) {
    kids[t] = 0;
    last[t] = 0;
  }
  if (t == 0) most = 0;
  __syncthreads();
  if (t < W) {
    const int from = parents[(int64_t)g * W + t];
    if (from >= 0 && from < W && from != t) {
      const int n = lens[(int64_t)g * W + from];
      if (n > 0 && n <= Smax) {
        atomicOr((unsigned long long*)&kids[from], 1ull << t);
        last[from] = (int64_t)n * row_units;
        atomicMax(&most, n);
      }
    }
  }
  __syncthreads();
  // (the same for all threads: in scalar registers)
  using Mask = typename std::conditional<MW <= 32, uint32_t, uint64_t>::type;
  Mask to[MW];
  int64_t end_of[MW];
#pragma unroll
  for (int w = 0; w < MW; ++w) {
    to[w] = (Mask)uniform64(kids[w]);
    end_of[w] = uniform64(last[w]);
  }
  const int64_t stride = (int64_t)Hkv * Smax * row_units;  // between two sequences
  U* at = (U*)base + ((int64_t)g * W * Hkv + h) * (int64_t)Smax * row_units;
  const int64_t end = uniform64((int64_t)most * row_units);
  for (int64_t i = (int64_t)blockIdx.z * 256 + t; i < end; i += (int64_t)gridDim.z * 256) {
    U x[MW];
#pragma unroll
    for (int w = 0; w < MW; ++w)
      if (to[w] && i < end_of[w]) x[w] = at[w * stride + i];
#pragma unroll
    for (int w = 0; w < MW; ++w)
      if (to[w] && i < end_of[w])
        for (Mask m = to[w]; m; m &= m - 1)
          at[__builtin_ctzll(m) * stride + i] = x[w];
  }
}

size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

int slices_of(const SelectArgs& a) { return slices_of(a.V, a.dtype == F32 ? 4 : 8); }

template <typename T>
int select_typed(const SelectArgs& a, void* workspace) {
  const int slices = slices_of(a);
  SliceSum* sums = (SliceSum*)workspace;
  Candidate* best =
      (Candidate*)((char*)workspace + up256((size_t)a.G * a.W * slices * sizeof(SliceSum)));
  KF_LAUNCH("select_rows", select_rows_kernel<T>, dim3(a.G * a.W, slices), dim3(NT), 0, a.stream,
            a, sums, best);
  KF_CHECK_LAUNCH();
  KF_LAUNCH("select_pick", select_pick_kernel, dim3(a.G), dim3(NT), 0, a.stream, a, sums, best,
            slices);
  KF_CHECK_LAUNCH();
  return KF_OK;
}

template <typename U>
int reorder_launch(const ReorderPtrs& p, int n, const int32_t* lens, const int32_t* parents, int W,
                   int B, int Hkv, int Smax, int row_units, hipStream_t stream) {
  // Rows are spread over 8192 workgroups and more, 32 a compute unit (32 layers of 8 x 4
  // beams of 2048 rows: 2.84 ms with 4096, 2.48, 2.41 with 65536).  The lengths are on the
  // device, so those behind the last row find nothing to do, which more of them would take
  // long over where a long cache holds few rows.
  const int64_t items = (int64_t)(B / W) * Hkv * 2 * n;
  const int64_t all = ((int64_t)Smax * row_units + 255) / 256;
  const int64_t split = std::max<int64_t>(1, std::min<int64_t>({all, 8192 / items + 1, 65535}));
  const dim3 grid((unsigned)(B / W * Hkv), 2 * n, (unsigned)split);
  auto kernel = W <= 4 ? cache_reorder_kernel<U, 4> : cache_reorder_kernel<U, 8>;
  if (W > 8) kernel = cache_reorder_kernel<U, 16>;
  if constexpr (sizeof(U) < 16) {
    if (W > 16) kernel = cache_reorder_kernel<U, 64>;
  }
  KF_LAUNCH("cache_reorder", kernel, grid, dim3(256), 0, stream, p, lens, parents, W, Hkv, Smax,
            row_units);
  KF_CHECK_LAUNCH();
  return KF_OK;
}

}  // namespace

size_t select_workspace(const SelectArgs& a) {
  const size_t n = (size_t)a.G * a.W * slices_of(a);
  return up256(n * sizeof(SliceSum)) + up256(n * a.K * sizeof(Candidate));
}

int beam_select(const SelectArgs& a, void* workspace) {
  switch (a.dtype) {
    case F32: return select_typed<float>(a, workspace);
    case BF16: return select_typed<bf16>(a, workspace);
    case F16: return select_typed<_Float16>(a, workspace);
  }
  set_error("unsupported dtype %d", a.dtype);
  return KF_ERR_UNSUPPORTED;
}

int cache_reorder(void* const* k, void* const* v, int n_caches, const int32_t* lens,
                  const int32_t* parents, int W, int B, int Hkv, int Smax, int D, int dtype,
                  hipStream_t stream) {
  const int bytes = D * (dtype == F32 ? 4 : 2);
  for (int c0 = 0; c0 < n_caches; c0 += KEEP_CACHES) {
    const int n = std::min(KEEP_CACHES, n_caches - c0);
    ReorderPtrs p = {};
    uintptr_t low = (uintptr_t)bytes;
    for (int c = 0; c < n; ++c) {
      p.k[c] = (char*)k[c0 + c];
      p.v[c] = (char*)v[c0 + c];
      low |= (uintptr_t)p.k[c] | (uintptr_t)p.v[c];
    }
    int rc;
    // (64 registers of 16 bytes are too many: halves of them for wide beams.  32 layers of 64
    // sequences of 256 rows in groups of 8 and 16 move at 4.5 and 4.3 TB/s, in groups of 17,
    // 32 and 64 at 2.5, 2.6 and 3.2)
    if (low % 16 == 0 && W <= 16)
      rc = reorder_launch<u32x4>(p, n, lens, parents, W, B, Hkv, Smax, bytes / 16, stream);
    else if (low % 8 == 0)
      rc = reorder_launch<u32x2>(p, n, lens, parents, W, B, Hkv, Smax, bytes / 8, stream);
    else
      rc = reorder_launch<uint16_t>(p, n, lens, parents, W, B, Hkv, Smax, bytes / 2, stream);
    if (rc) return rc;
  }
  return KF_OK;
}

}  // namespace kf
