// Beam search after the model's forward: the selection over beams and vocabulary, and
// the caches' rows of the beams that go on.
//
// Selection: of W beams with scores s_w and logits x_w over V tokens, the K largest of
//   t_wv = s_w + x_wv - log sum_u exp x_wu,
// equals by the lowest w, then v.  Within a beam t rises with x, so a row's K largest
// logits are all that can be picked of it:
//  1. rows   a workgroup per slice of a row: the slice's maximum and sum of
//            exponentials, and its K largest logits
//  2. pick   a workgroup per group: the rows' sums joined, then the K largest of the
//            W x slices x K candidates, in 64 bits
// Every logit is read once.  HBM bounds the first (32 x 8 rows of 131072), two dependent
// launches the smallest calls.
#include "kf_common.h"
#include "kf_internal.h"
#include "kf_row.h"

#include <algorithm>
#include <climits>

namespace kf {

namespace {

// ------------------------------------------------------------------ the K largest
// of values spread over a workgroup of 256, largest first, equals by the lowest index.
//
// The workgroup's values fall into 64 groups (lane l of the four wavefronts); the K-th
// largest of the groups' maxima is at most the K-th largest value, and few values are
// above it (64 ln(64 / (64 - K)) of independent ones), so those are gathered and ordered
// by counting.  From 48 on the 256 threads are the groups.  More than CAP of them (values
// that are ordered against the groups, or mostly equal) are taken one at a time.
constexpr int NT = 256, CAP = 1024;

template <typename V>
struct TopLds {
  V top[NT];
  V val[CAP];
  int idx[CAP];
  int count, best;
  V red[NT / 64];
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

// own: the thread's largest value (-inf: none).  some(T, f): f(value, index) for the
// thread's values >= T above -inf.  out(place, value, index), place < K; returns how many
// places there are values for.
template <typename V, typename Some, typename Out>
__device__ __forceinline__ int top_k(int K, V own, Some some, Out out, TopLds<V>& lds) {
  const int t = threadIdx.x, lane = t & 63;
  lds.top[t] = own;
  if (t == 0) lds.count = 0;
  __syncthreads();
  V edge = INFINITY;
  if (K <= 48) {
    V g = lds.top[lane];
#pragma unroll
    for (int i = 1; i < NT / 64; ++i) g = fmax(g, lds.top[lane + 64 * i]);
    int above = 0;
    for (int j = 0; j < 64; ++j) above += lane_of(g, j) > g;
    if (above < K) edge = g;
  } else {
    V g[NT / 64];
    int above[NT / 64] = {};
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) g[i] = lds.top[lane + 64 * i];
    for (int j = 0; j < NT; ++j) {
      const V x = lds.top[j];
#pragma unroll
      for (int i = 0; i < NT / 64; ++i) above[i] += x > g[i];
    }
#pragma unroll
    for (int i = 0; i < NT / 64; ++i)
      if (above[i] < K) edge = fmin(edge, g[i]);
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) edge = fmin(edge, __shfl_xor(edge, o, 64));
  if (own >= edge)
    some(edge, [&](V x, int i) {
      const int at = atomicAdd(&lds.count, 1);
      if (at < CAP) {
        lds.val[at] = x;
        lds.idx[at] = i;
      }
    });
  __syncthreads();
  const int n = lds.count;
  if (n <= CAP) {
    for (int a = t; a < n; a += NT) {
      const V x = lds.val[a];
      const int i = lds.idx[a];
      int place = 0;
      for (int b = 0; b < n; ++b) place += lds.val[b] > x || (lds.val[b] == x && lds.idx[b] < i);
      if (place < K) out(place, x, i);
    }
    return min(n, K);
  }
  V last = INFINITY;
  int after = -1;
  for (int place = 0; place < K; ++place) {
    // the largest value behind (last, after), then the lowest index that has it
    V x = -INFINITY;
    some(edge, [&](V v, int i) {
      if (v < last || (v == last && i > after)) x = fmax(x, v);
    });
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) x = fmax(x, __shfl_xor(x, o, 64));
    __syncthreads();
    if (lane == 0) lds.red[t >> 6] = x;
    if (t == 0) lds.best = INT_MAX;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) x = fmax(x, lds.red[w]);
    some(edge, [&](V v, int i) {
      if (v == x && (v < last || i > after)) atomicMin(&lds.best, i);
    });
    __syncthreads();
    if (t == 0) out(place, x, lds.best);
    last = x;
    after = lds.best;
  }
  return K;
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

// Slices of a row of V values, U granules of E a thread.
int slices_of(int V, int E, int U) { return ((V + E - 1) / E + NT * U - 1) / (NT * U); }

// Workgroup (row, slice).  Exponentials are float32 instructions of the difference to the
// thread's maximum, x log2 e - m log2 e in one rounding (2^-24 of it, so a term of weight
// p is off by 2^-24 |ln p|), sums of a thread's values in 32 bits, of the threads' in 64;
// what m log2 e was rounded by is taken back in 64 bits.  A thread's granules are counted
// from the row's first value, whatever its alignment (the loads may be unaligned): rows of
// equal values have equal sums, to the last bit, and their beams' candidates are equals.
template <typename T, int U>
__global__ __launch_bounds__(NT) void select_rows_kernel(SelectArgs a, SliceSum* __restrict__ sums,
                                                         Candidate* __restrict__ best) {
  __shared__ TopLds<float> lds;
  __shared__ float sm[NT / 64];
  __shared__ double ss[NT / 64];
  constexpr int E = Row<T>::E;
  const int g = blockIdx.x / a.W, w = blockIdx.x % a.W, t = threadIdx.x, lane = t & 63;
  if (!(fabsf(a.scores[blockIdx.x]) < INFINITY)) return;  // a beam that is not in use
  const T* row = (const T*)a.logits + g * a.logits_sg + w * a.logits_sw;
  const int v0 = (blockIdx.y * (NT * U) + t) * E;  // the thread's first value
  u32x4 raw[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int v = v0 + u * NT * E;
    if (v + E <= a.V) {
      __builtin_memcpy(&raw[u], row + v, 16);
    } else {
      T x[E];
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = v + e < a.V ? row[v + e] : from_f32<T>(-INFINITY);
      __builtin_memcpy(&raw[u], x, 16);
    }
  }
  float gm[U], m = -INFINITY;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float f[E];
    Row<T>::unpack(raw[u], f);
    gm[u] = f[0];
#pragma unroll
    for (int e = 1; e < E; ++e) gm[u] = fmaxf(gm[u], f[e]);
    m = fmaxf(m, gm[u]);
  }
  const float ref = m == -INFINITY ? 0.f : m, ml = ref * kLog2e;
  float part = 0.f;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float f[E], x = 0.f;
    Row<T>::unpack(raw[u], f);
#pragma unroll
    for (int e = 0; e < E; ++e) x += fast_exp2(__builtin_fmaf(f[e], kLog2e, -ml));
    part += x;
  }
  constexpr double L = 1.4426950408889634074;
  float M = m;
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
  if (lane == 0) sm[t >> 6] = M;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) M = fmaxf(M, sm[i]);
  double s = m == -INFINITY ? (double)(part != part ? part : 0.f)
                            : (double)part * exp2_64(((double)m - (double)M) * L +
                                                     (ml - (double)m * (double)kLog2e));
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
  if (lane == 0) ss[t >> 6] = s;
  __syncthreads();
  const int64_t at = (int64_t)blockIdx.x * gridDim.y + blockIdx.y;
  if (t == 0) {
    s = 0.0;
    for (int i = 0; i < NT / 64; ++i) s += ss[i];
    sums[at] = SliceSum{M, s};
  }
  Candidate* out = best + at * a.K;
  const int n = top_k(
      a.K, m,
      [&](float edge, auto f) {
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (gm[u] >= edge) {
            float x[E];
            Row<T>::unpack(raw[u], x);
#pragma unroll
            for (int e = 0; e < E; ++e)
              if (x[e] >= edge && x[e] > -INFINITY) f(x[e], v0 + u * NT * E + e);
          }
      },
      [&](int place, float x, int v) { out[place] = Candidate{x, v}; }, lds);
  for (int i = n + t; i < a.K; i += NT) out[i] = Candidate{-INFINITY, -1};
}

// ------------------------------------------------------------------ pick
__global__ __launch_bounds__(NT) void select_pick_kernel(SelectArgs a,
                                                         const SliceSum* __restrict__ sums,
                                                         const Candidate* __restrict__ best,
                                                         int slices) {
  __shared__ TopLds<double> lds;
  __shared__ double score[KF_BEAM_MAX], lse[KF_BEAM_MAX];
  const int g = blockIdx.x, t = threadIdx.x, lane = t & 63, W = a.W;
  constexpr double L = 1.4426950408889634074;
  for (int w = t >> 6; w < W; w += NT / 64) {
    const float sc = a.scores[(int64_t)g * W + w];
    bool ok = fabsf(sc) < INFINITY;
    double s = 0.0;
    float M = -INFINITY;
    if (ok) {
      const SliceSum* row = sums + ((int64_t)g * W + w) * slices;
      for (int i = lane; i < slices; i += 64) M = fmaxf(M, row[i].m);
      M = wave_max(M);
      for (int i = lane; i < slices; i += 64)
        s += row[i].m == M ? row[i].s : row[i].s * exp2_64(((double)row[i].m - (double)M) * L);
#pragma unroll
      for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
      ok = s > 0.0 && s < INFINITY;
    }
    if (lane == 0) {
      score[w] = ok ? (double)sc : -INFINITY;
      lse[w] = ok ? (double)M + log(s) : 0.0;
    }
  }
  __syncthreads();
  const int per = slices * a.K, n = W * per;
  const Candidate* c = best + (int64_t)g * n;
  auto each = [&](auto f) {
    for (int i = t; i < n; i += NT) {
      const int w = i / per;
      if (score[w] == -INFINITY) continue;  // (what its slices hold was not written)
      const Candidate x = c[i];
      if (x.v >= 0) f(score[w] + ((double)x.x - lse[w]), w * a.V + x.v);
    }
  };
  double own = -INFINITY;
  each([&](double x, int) { own = fmax(own, x); });
  const int64_t at = (int64_t)g * a.K;
  const int m = top_k(
      a.K, own,
      [&](double edge, auto f) {
        each([&](double x, int i) {
          if (x >= edge) f(x, i);
        });
      },
      [&](int place, double x, int i) {
        a.out_scores[at + place] = (float)x;
        a.parents[at + place] = i / a.V;
        a.tokens[at + place] = i % a.V;
      },
      lds);
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
  const int64_t stride = (int64_t)Hkv * Smax * row_units;  // between two sequences
  U* at = (U*)base + ((int64_t)g * W * Hkv + h) * (int64_t)Smax * row_units;
  const int64_t end = (int64_t)most * row_units;
  for (int64_t i = (int64_t)blockIdx.z * 256 + t; i < end; i += (int64_t)gridDim.z * 256) {
    U x[MW];
#pragma unroll
    for (int w = 0; w < MW; ++w)
      if (w < W && i < last[w]) x[w] = at[w * stride + i];
#pragma unroll
    for (int w = 0; w < MW; ++w)
      if (w < W && i < last[w])
        for (uint64_t m = kids[w]; m; m &= m - 1) at[__builtin_ctzll(m) * stride + i] = x[w];
  }
}

size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

// Granules a thread of the rows kernel: few where many would leave compute units without a
// workgroup.
int unit_of(const SelectArgs& a) {
  return (int64_t)a.G * a.W * slices_of(a.V, a.dtype == F32 ? 4 : 8, 16) >= 512 ? 16 : 4;
}
int slices_of(const SelectArgs& a) { return slices_of(a.V, a.dtype == F32 ? 4 : 8, unit_of(a)); }

template <typename T>
int select_typed(const SelectArgs& a, void* workspace) {
  const int unit = unit_of(a), slices = slices_of(a);
  SliceSum* sums = (SliceSum*)workspace;
  Candidate* best =
      (Candidate*)((char*)workspace + up256((size_t)a.G * a.W * slices * sizeof(SliceSum)));
  KF_LAUNCH("select_rows", (unit == 16 ? select_rows_kernel<T, 16> : select_rows_kernel<T, 4>),
            dim3(a.G * a.W, slices), dim3(NT), 0, a.stream, a, sums, best);
  KF_CHECK_LAUNCH();
  KF_LAUNCH("select_pick", select_pick_kernel, dim3(a.G), dim3(NT), 0, a.stream, a, sums, best,
            slices);
  KF_CHECK_LAUNCH();
  return KF_OK;
}

template <typename U>
int reorder_launch(const ReorderPtrs& p, int n, const int32_t* lens, const int32_t* parents, int W,
                   int B, int Hkv, int Smax, int row_units, hipStream_t stream) {
  // Rows are spread over workgroups until there are some 16 per compute unit; the
  // lengths are on the device, so those behind the last row find nothing to do.
  const int64_t items = (int64_t)(B / W) * Hkv * 2 * n;
  const int64_t all = ((int64_t)Smax * row_units + 255) / 256;
  const int64_t split = std::max<int64_t>(1, std::min<int64_t>({all, 4096 / items + 1, 65535}));
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
    // (64 registers of 16 bytes are too many: halves of them for wide beams)
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
