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
// One workgroup of 16 wavefronts per sequence: the walk reads only the rows on
// its path, and the next row is known only after the last.
constexpr int VT = 1024, VW = VT / 64;

// 16 bytes of a row as floats: granule k of the row's aligned granules, the
// row's first element at place `lead` of granule 0.  Places outside the row get
// -inf.
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
  __device__ __forceinline__ void load(int k, float* f) const {
    const int v0 = first(k);
    if (v0 >= 0 && v0 + E <= V) {
      T t[E];
      *(u32x4*)t = *(const u32x4*)(x + v0);
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] = to_f32(t[e]);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        f[e] = v0 + e >= 0 && v0 + e < V ? to_f32(x[v0 + e]) : -INFINITY;
    }
  }
};

struct Stat {
  float m;   // maximum
  double s;  // sum of exp((x - m) / T); not positive and finite: no distribution
  int at;    // first place of the maximum
};

// Maximum, its first place and (SUM) the sum of exp((x - m) / T) of a row, by
// the whole workgroup.  A row holding NaN gets s = NaN.
// Each exponential is one float32 instruction (relative error 2^-22 and that of
// its argument); their sum is kept in 64 bits.
template <typename T>
__device__ Stat row_stats(const Row<T>& r, double inv_t, float* sf, double* sd, int* si) {
  constexpr int E = Row<T>::E;
  const int t = threadIdx.x, lane = t & 63, w = t >> 6;
  const float c = (float)(inv_t * 1.4426950408889634);
  float m = -INFINITY;
  int at = INT_MAX;
  double s = 0.0;
  bool nan = false;
  for (int k = t; k < r.granules(); k += VT) {
    float f[E];
    r.load(k, f);
    float gm = f[0];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      nan |= f[e] != f[e];
      gm = fmaxf(gm, f[e]);
    }
    if (gm > m) {
      s *= (double)exp2f((m - gm) * c);  // (m = -inf: s is 0)
      m = gm;
#pragma unroll
      for (int e = E - 1; e >= 0; --e)
        if (f[e] == gm) at = r.first(k) + e;
    }
    const float ref = m == -INFINITY ? 0.f : m;
    float gs = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) gs += exp2f((f[e] - ref) * c);
    s += (double)gs;
  }
  if (at == INT_MAX && t < r.V) at = t;  // a share without a finite value
  if (nan) s = NAN;
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    const float m2 = __shfl_xor(m, o, 64);
    const double s2 = __shfl_xor(s, o, 64);
    const int a2 = __shfl_xor(at, o, 64);
    const float mn = fmaxf(m, m2), ref = mn == -INFINITY ? 0.f : mn;
    s = s * (double)exp2f((m - ref) * c) + s2 * (double)exp2f((m2 - ref) * c);
    at = m > m2 ? at : m2 > m ? a2 : min(at, a2);
    m = mn;
  }
  __syncthreads();  // the previous use of the exchange arrays is over
  if (lane == 0) {
    sf[w] = m;
    sd[w] = s;
    si[w] = at;
  }
  __syncthreads();
  Stat o{-INFINITY, 0.0, INT_MAX};
  for (int j = 0; j < VW; ++j) o.m = fmaxf(o.m, sf[j]);
  const float ref = o.m == -INFINITY ? 0.f : o.m;
  for (int j = 0; j < VW; ++j) {
    o.s += sd[j] * (double)exp2f((sf[j] - ref) * c);
    if (sf[j] == o.m) o.at = min(o.at, si[j]);
  }
  return o;
}

__device__ __forceinline__ bool has_mass(double s) { return s > 0.0 && s < INFINITY; }

// p(x) of a row in 64 bits.
__device__ __forceinline__ double prob(float x, const Stat& st, double inv_t) {
  return exp(((double)x - (double)st.m) * inv_t) / st.s;
}

// V <= KF_VERIFY_MAX_VOCAB: segments of 64 granules of at least 4 values
constexpr int MAXSEG = KF_VERIFY_MAX_VOCAB / 256 + 2;

template <typename T>
__global__ __launch_bounds__(VT) void verify_kernel(VerifyArgs a) {
  constexpr int E = Row<T>::E;
  __shared__ int spar[MAXN], stok[MAXN], spath[MAXN];
  __shared__ float su[MAXN];
  __shared__ double sp[MAXN];
  __shared__ int srefused[MAXN];  // tokens of the last node's refused children
  __shared__ float sf[VW];
  __shared__ double sd[VW];
  __shared__ int si[VW];
  __shared__ int step, token, nref;
  __shared__ double seg[MAXSEG];
  const int b = blockIdx.x, t = threadIdx.x, lane = t & 63, w = t >> 6;
  const int N = a.N, V = a.V;
  const int n = a.counts ? a.counts[b] : N;
  const bool greedy = !(a.temperature > 0.0);
  const double inv_t = greedy ? 1.0 : 1.0 / a.temperature;
  bool bad = n < 0 || n > N;
  if (t < N) {
    int par = t - 1;
    if (a.parents != nullptr) par = a.parents[(int64_t)b * a.parents_stride + t];
    const int64_t tok = a.tokens[(int64_t)b * N + t];
    spar[t] = par;
    stok[t] = tok >= 0 && tok < V ? (int)tok : -1;
    su[t] = a.uniforms[(int64_t)b * N + t];
    spath[t] = -1;
    if (t < n && (t == 0 ? par != -1 : par < 0 || par >= t)) bad = true;
  }
  bad = __syncthreads_or(bad);
  int cur = 0, len = 0;
  int64_t next = -1;
  if (!bad && n > 0) {
    while (true) {
      if (t == 0) {
        spath[len] = cur;
        step = -1;
        token = -1;
        nref = 0;
      }
      ++len;
      const Row<T> row((const T*)a.logits + b * a.logits_sb + cur * a.logits_sn, V);
      const Stat st = row_stats<T>(row, inv_t, sf, sd, si);
      if (greedy ? st.s != st.s : !has_mass(st.s)) break;  // no distribution: next stays -1
      const bool drafted = a.drafts != nullptr && cur + 1 < n;
      const Row<T> drow(drafted ? (const T*)a.drafts + b * a.drafts_sb + cur * a.drafts_sn : row.x,
                        V);
      Stat dst{0.f, 1.0, 0};
      if (drafted) dst = row_stats<T>(drow, inv_t, sf, sd, si);
      // every child's probability, then the children in order
      if (t < n && spar[t] == cur && t > 0) {
        const int c = stok[t];
        double p = -1.0;  // a token outside the vocabulary, or a sibling's: refused
        if (c >= 0) {
          if (greedy) {
            p = c == st.at;
          } else {
            p = prob(to_f32(row.x[c]), st, inv_t);
            if (!drafted)
              for (int j = cur + 1; j < t; ++j)
                if (spar[j] == cur && stok[j] == c) p = -1.0;
          }
        }
        sp[t] = p;
      }
      __syncthreads();
      if (t == 0) {
        double left = 1.0;
        for (int i = cur + 1; i < n; ++i) {
          if (spar[i] != cur) continue;
          const double p = sp[i];
          bool take;
          if (greedy)
            take = p > 0.0;
          else if (drafted)
            take = p >= 0.0 && (double)su[i] * prob(to_f32(drow.x[stok[i]]), dst, inv_t) < p;
          else
            take = p >= 0.0 && (double)su[i] * left < p;
          if (take) {
            step = i;
            break;
          }
          if (p > 0.0) {
            left -= p;
            srefused[nref++] = stok[i];
          }
        }
      }
      __syncthreads();
      const int to = step;
      if (to >= 0) {
        cur = to;
        __syncthreads();  // step is read before it is written again
        continue;
      }
      if (greedy) {
        next = st.at;
        break;
      }
      // The draw, in 64 bits: weights of the row's values in order, summed by
      // segments of 64 granules; then the segment that holds the point.
      const bool minus = drafted && has_mass(dst.s);
      // weights of granule k (the draft's row may be aligned differently: read
      // value by value)
      auto weights = [&](int k, bool all, double* wt) {
        float f[E];
        row.load(k, f);
        const int v0 = row.first(k);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int v = v0 + e;
          wt[e] = v < 0 || v >= V ? 0.0 : prob(f[e], st, inv_t);
          if (minus && !all && wt[e] > 0.0)
            wt[e] = fmax(wt[e] - prob(to_f32(drow.x[v]), dst, inv_t), 0.0);
        }
        if (!drafted && !all)
          for (int i = 0; i < nref; ++i)
#pragma unroll
            for (int e = 0; e < E; ++e)
              if (srefused[i] == v0 + e) wt[e] = 0.0;
      };
      const int nseg = (row.granules() + 63) / 64;
      double total = 0.0;
      bool all = false;
      for (int pass = 0; pass < 2; ++pass) {
        for (int g = w; g < nseg; g += VW) {
          double x = 0.0;
          const int k = 64 * g + lane;
          if (k < row.granules()) {
            double wt[E];
            weights(k, all, wt);
#pragma unroll
            for (int e = 0; e < E; ++e) x += wt[e];
          }
#pragma unroll
          for (int o = 32; o >= 1; o >>= 1) x += __shfl_xor(x, o, 64);
          if (lane == 0) seg[g] = x;
        }
        __syncthreads();
        total = 0.0;
        for (int g = 0; g < nseg; ++g) total += seg[g];
        // rounding can leave no mass where all of it was on refused tokens: the
        // draw is then from the row itself
        if (total > 0.0 || all) break;
        all = true;
        __syncthreads();
      }
      if (w == 0) {
        const double point = (double)su[0] * total;
        double before = 0.0;
        int g = 0;
        for (; g < nseg - 1; ++g) {
          if (before + seg[g] > point) break;
          before += seg[g];
        }
        const int k = 64 * g + lane;
        double wt[E], own = 0.0;
        int last = -1;
#pragma unroll
        for (int e = 0; e < E; ++e) wt[e] = 0.0;
        if (k < row.granules()) {
          weights(k, all, wt);
#pragma unroll
          for (int e = 0; e < E; ++e) {
            own += wt[e];
            if (wt[e] > 0.0) last = row.first(k) + e;
          }
        }
        double incl = own;
        for (int o = 1; o < 64; o <<= 1) {
          const double y = __shfl_up(incl, o, 64);
          if (lane >= o) incl += y;
        }
        double run = before + (incl - own);
        int hit = INT_MAX;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          run += wt[e];
          if (hit == INT_MAX && wt[e] > 0.0 && run > point) hit = row.first(k) + e;
        }
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) {
          hit = min(hit, __shfl_xor(hit, o, 64));
          last = max(last, __shfl_xor(last, o, 64));
        }
        // (sums of two orders may leave the point behind the segment's last value)
        if (lane == 0) token = hit != INT_MAX ? hit : last;
      }
      __syncthreads();
      next = token;
      break;
    }
  }
  __syncthreads();
  if (t < N) a.path[(int64_t)b * N + t] = t < len ? spath[t] : -1;
  if (t == 0) {
    a.kept[b] = len;
    a.next[b] = next;
  }
}

// ------------------------------------------------------------------ keep
// Row L + path[j] to row L + j for j < kept, in every cache.  path rises, so
// path[j] >= j: a row is overwritten only after the only move that reads it (an
// earlier j).  A thread moves the same 16 bytes of every row, in order of j, so
// its own program order is all the ordering that needs.
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

int verify_drafts(const VerifyArgs& a) {
  switch (a.dtype) {
    case F32:
      KF_LAUNCH("verify", verify_kernel<float>, dim3(a.B), dim3(VT), 0, a.stream, a);
      break;
    case BF16:
      KF_LAUNCH("verify", verify_kernel<bf16>, dim3(a.B), dim3(VT), 0, a.stream, a);
      break;
    case F16:
      KF_LAUNCH("verify", verify_kernel<_Float16>, dim3(a.B), dim3(VT), 0, a.stream, a);
      break;
    default:
      set_error("unsupported dtype %d", a.dtype);
      return KF_ERR_UNSUPPORTED;
  }
  KF_CHECK_LAUNCH();
  return KF_OK;
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
