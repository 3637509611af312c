// Attention of a tree of drafted tokens over a KV cache.
//
// Node i of sequence b sees the cached prefix (keys 0 .. lens[b] - 1), itself and
// its ancestors in the tree:
//   s_ij = q_i . k_j / sqrt(D),  j in prefix or anc(i);  o_i = softmax(s_i) V
// Its key is rotated at position lens[b] + depth(i) and stored in cache row
// lens[b] + i, so that the rows of all nodes lie behind the prefix in node order.
//
//  1. prep    the ancestors of every node (as bit masks), the rotated queries,
//             and the nodes' rows of the caches
//  2. rows    one wavefront per (node, query head)
#include "kf_common.h"
#include "kf_internal.h"

#include <climits>

namespace kf {

namespace {

constexpr int MAXN = KF_TREE_MAX_NODES;
constexpr int MAXW = MAXN / 32;  // 32-bit words of an ancestor mask

// RMSNorm of one element given its row's sum of squares (rms_scale of
// kf_decode.hip: float32, rounded to the storage type).
template <typename T>
__device__ __forceinline__ float rms_scale(float x, float ss, int D, float eps, float w) {
  const float r = rsqrtf(ss / (float)D + eps);
  return round_to<T>((x * r) * w);
}

template <typename T>
__device__ __forceinline__ bool finite(T x) {
  return fabsf(to_f32(x)) < INFINITY;  // false for NaN too
}

// One workgroup: sequence blockIdx.y, `per` of its N * (Hq + 2 Hkv) rows.
//
// The ancestor masks come from pointer doubling: after round r, mask[i] holds
// the 2^r nearest of i and its ancestors and ptr[i] the next one beyond, so 8
// rounds cover 256 nodes whatever their depth (a walk up a chain of 200 would
// take 200 dependent reads).  Every workgroup of a sequence forms them again
// (under a microsecond, no launch of its own); the first one stores them.
template <typename T>
__global__ __launch_bounds__(256) void tree_prep_kernel(TreeArgs a, T* __restrict__ qrot,
                                                        uint32_t* __restrict__ anc,
                                                        int2* __restrict__ seq,
                                                        uint8_t* __restrict__ vbad, int W,
                                                        int per) {
  __shared__ uint32_t smask[MAXN][MAXW + 1];
  __shared__ int sptr[MAXN], sdepth[MAXN];
  const int b = blockIdx.y, t = threadIdx.x, lane = t & 63, w = t >> 6;
  const int N = a.N, D = a.D, half = D / 2;
  const int L = a.lens[b], n = a.counts ? a.counts[b] : N;
  bool bad = n < 0 || n > N || L < 0 || (int64_t)L + n > a.max_len;
  const int used = bad ? 0 : n;
  int depth = t;
  if (a.parents != nullptr) {
    int par = -1;
    if (t < used) {
      par = a.parents[(int64_t)b * a.parents_stride + t];
      if (par < -1 || par >= t) {
        bad = true;
        par = -1;
      }
    }
    for (int k = 0; k < W; ++k) smask[t][k] = 0;
    smask[t][t >> 5] = 1u << (t & 31);
    sptr[t] = par;
    __syncthreads();
    for (int span = 1; span < used; span <<= 1) {
      const int p = sptr[t];
      uint32_t m[MAXW];
      int next = -1;
      if (p >= 0) {
        for (int k = 0; k < MAXW; ++k) m[k] = k < W ? smask[p][k] : 0u;
        next = sptr[p];
      }
      __syncthreads();
      if (p >= 0) {
        for (int k = 0; k < MAXW; ++k)
          if (k < W) smask[t][k] |= m[k];
        sptr[t] = next;
      }
      __syncthreads();
    }
    depth = -1;
    for (int k = 0; k < W; ++k) depth += __popc(smask[t][k]);
  } else {  // a chain: node i sees nodes 0 .. i
    for (int k = 0; k < W; ++k) {
      const int lo = t + 1 - 32 * k;
      smask[t][k] = lo <= 0 ? 0u : lo >= 32 ? ~0u : (1u << lo) - 1u;
    }
  }
  sdepth[t] = depth;
  const int64_t trow = (int64_t)L + depth - a.rope_row_offset;
  if (t < used && (trow < 0 || trow >= a.rope_rows)) bad = true;
  bad = __syncthreads_or(bad);
  if (blockIdx.x == 0) {
    if (t == 0) seq[b] = make_int2(bad ? -1 : n, bad ? 0 : L);
    if (t < N)
      for (int k = 0; k < W; ++k) anc[((int64_t)b * N + t) * W + k] = smask[t][k];
  }
  if (bad) return;
  const int heads = a.Hq + 2 * a.Hkv, n_rep = a.Hq / a.Hkv;
  const int64_t r1 = min((int64_t)n * heads, (int64_t)(blockIdx.x + 1) * per);
  for (int64_t r = (int64_t)blockIdx.x * per + w; r < r1; r += 4) {
    const int i = (int)(r / heads), h = (int)(r % heads);
    const int64_t node = (int64_t)b * N + i;
    if (h >= a.Hq + a.Hkv) {
      const int g = h - a.Hq - a.Hkv;
      const T* src = (const T*)a.v_new + (node * a.Hkv + g) * D;
      T* dst = (T*)a.v_cache + (((int64_t)b * a.Hkv + g) * a.Smax + L + i) * D;
      bool fin = true;
      for (int d = lane; d < D; d += 64) {
        const T x = src[d];
        dst[d] = x;
        fin = fin && finite(x);
      }
      const uint64_t all = __builtin_amdgcn_ballot_w64(!fin);
      if (lane == 0) vbad[((int64_t)b * a.Hkv + g) * N + i] = all != 0;
      continue;
    }
    const bool is_q = h < a.Hq;
    const int g = is_q ? h / n_rep : h - a.Hq;
    const T* src = is_q ? (const T*)a.q_new + (node * a.Hq + h) * D
                        : (const T*)a.k_new + (node * a.Hkv + g) * D;
    T* dst = is_q ? qrot + (((int64_t)b * a.Hkv + g) * N * n_rep + (int64_t)i * n_rep + h % n_rep) * D
                  : (T*)a.k_cache + (((int64_t)b * a.Hkv + g) * a.Smax + L + i) * D;
    const float* nw = is_q ? a.q_norm_w : a.k_norm_w;
    float ss = 0.f;
    if (nw != nullptr) {
      for (int d = lane; d < D; d += 64) ss += to_f32(src[d]) * to_f32(src[d]);
      ss = wave_sum(ss);
    }
    const int64_t row = ((int64_t)L + sdepth[i] - a.rope_row_offset) * half;
    for (int d = lane; d < half; d += 64) {
      float x1 = to_f32(src[d]), x2 = to_f32(src[d + half]), y1, y2;
      if (nw != nullptr) {
        x1 = rms_scale<T>(x1, ss, D, a.norm_eps, nw[d]);
        x2 = rms_scale<T>(x2, ss, D, a.norm_eps, nw[d + half]);
      }
      rope_pair<T>(x1, x2, a.cos[row + d], a.sin[row + d], y1, y2);
      dst[d] = from_f32<T>(y1);
      dst[d + half] = from_f32<T>(y2);
    }
  }
}

// One wavefront per (b, node, query head), any D <= 256: the prefix and the
// node's own row and ancestors, one key at a time.  Masked keys are not read.
template <typename T>
__global__ __launch_bounds__(256) void tree_rows_kernel(TreeArgs a, const T* __restrict__ qrot,
                                                        const uint32_t* __restrict__ anc,
                                                        const int2* __restrict__ seq, int W) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= (int64_t)a.B * a.N * a.Hq) return;
  const int hq = (int)(row % a.Hq), i = (int)(row / a.Hq % a.N), b = (int)(row / a.Hq / a.N);
  const int D = a.D, n_rep = a.Hq / a.Hkv, g = hq / n_rep;
  const int2 s = seq[b];
  T* out = (T*)a.out + row * D;
  if (s.x < 0 || i >= s.x) {  // a refused sequence, or an unused node
    for (int d = lane; d < D; d += 64) out[d] = from_f32<T>(s.x < 0 ? NAN : 0.f);
    return;
  }
  const int L = s.y;
  const T* q = qrot + (((int64_t)b * a.Hkv + g) * a.N * n_rep + (int64_t)i * n_rep + hq % n_rep) * D;
  const T* kb = (const T*)a.k_cache + ((int64_t)b * a.Hkv + g) * a.Smax * D;
  const T* vb = (const T*)a.v_cache + ((int64_t)b * a.Hkv + g) * a.Smax * D;
  float qv[4], acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int e = 0; e < 4; ++e) qv[e] = lane + 64 * e < D ? to_f32(q[lane + 64 * e]) : 0.f;
  float m = -INFINITY, l = 0.f;
  auto key = [&](int j) {
    float x = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (lane + 64 * e < D) x += qv[e] * to_f32(kb[(int64_t)j * D + lane + 64 * e]);
    x = wave_sum(x) * a.scale;
    const float mn = fmaxf(m, x);
    const float ref = mn == -INFINITY ? 0.f : mn;
    const float alpha = expf(m - ref), p = expf(x - ref);
    l = l * alpha + p;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      acc[e] = acc[e] * alpha +
               (lane + 64 * e < D ? p * to_f32(vb[(int64_t)j * D + lane + 64 * e]) : 0.f);
    m = mn;
  };
  for (int j = 0; j < L; ++j) key(j);
  const uint32_t* words = anc + ((int64_t)b * a.N + i) * W;
  for (int k = 0; k < W; ++k)
    for (uint32_t bits = words[k]; bits; bits &= bits - 1) key(L + 32 * k + __builtin_ctz(bits));
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (lane + 64 * e < D) out[lane + 64 * e] = from_f32<T>(acc[e] / l);
}

size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

// workspace: rotated queries, ancestor masks, per sequence (nodes in use or -1,
// prefix length), per (b, KV head, node) whether its V row holds Inf or NaN
struct Ws {
  void* qrot;
  uint32_t* anc;
  int2* seq;
  uint8_t* vbad;
  size_t bytes;
};
Ws carve(const TreeArgs& a, void* p) {
  const size_t el = a.dtype == F32 ? 4 : 2;
  const size_t W = (a.N + 31) / 32;
  char* c = (char*)p;
  Ws w;
  w.qrot = c;
  c += up256((size_t)a.B * a.N * a.Hq * a.D * el);
  w.anc = (uint32_t*)c;
  c += up256((size_t)a.B * a.N * W * 4);
  w.seq = (int2*)c;
  c += up256((size_t)a.B * sizeof(int2));
  w.vbad = (uint8_t*)c;
  c += up256((size_t)a.B * a.Hkv * a.N);
  w.bytes = (size_t)(c - (char*)p);
  return w;
}

template <typename T>
int tree_typed(const TreeArgs& a, void* workspace) {
  const Ws w = carve(a, workspace);
  const int W = (a.N + 31) / 32, per = 16;
  const int64_t rows = (int64_t)a.N * (a.Hq + 2 * a.Hkv);
  KF_LAUNCH("tree_prep", tree_prep_kernel<T>, dim3((unsigned)((rows + per - 1) / per), a.B),
            dim3(256), 0, a.stream, a, (T*)w.qrot, w.anc, w.seq, w.vbad, W, per);
  KF_CHECK_LAUNCH();
  KF_LAUNCH("tree_rows", tree_rows_kernel<T>,
            dim3((unsigned)(((int64_t)a.B * a.N * a.Hq + 3) / 4)), dim3(256), 0, a.stream, a,
            (const T*)w.qrot, w.anc, w.seq, W);
  KF_CHECK_LAUNCH();
  return KF_OK;
}

}  // namespace

size_t tree_workspace(const TreeArgs& a) { return carve(a, nullptr).bytes; }

int tree_attention(const TreeArgs& a, void* workspace) {
  switch (a.dtype) {
    case F32: return tree_typed<float>(a, workspace);
    case BF16: return tree_typed<bf16>(a, workspace);
    case F16: return tree_typed<_Float16>(a, workspace);
  }
  set_error("unsupported dtype %d", a.dtype);
  return KF_ERR_UNSUPPORTED;
}

}  // namespace kf
