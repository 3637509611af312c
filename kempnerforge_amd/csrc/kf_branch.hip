// Attention behind shared prefixes: B sequences in G groups of W, each group with one
// prefix in a KV cache of its own, each sequence with its own tokens behind it.
//
// New token i of sequence b (of its n_b) sees the P_g keys of its group's prefix, the
// L_b cached tokens of its own and the new tokens up to itself:
//   s_ij = q_i . k_j / sqrt(D);  o_i = softmax(s_i) V
// Its key is rotated at position P_g + L_b + i and stored in row L_b + i of its own
// cache.  Softmax statistics and sums are joined over the prefix and the own rows.
//
// Rounding: the norm and the rotation of q and k are formed in 32 bits, k is rounded
// once, where it is stored.
#include "kf_common.h"
#include "kf_internal.h"
#include "kf_mfma.h"
#include "kf_split.h"
#include "kf_stream.h"

#include <algorithm>
#include <atomic>
#include <climits>
#include <type_traits>

namespace kf {

namespace {

// A sequence's new tokens in use (-1: the sequence is refused), its own cached tokens
// and its prefix.
struct Seq {
  int n, L, P;
};
__device__ __forceinline__ Seq branch_seq(const BranchArgs& a, int b) {
  const int n = a.counts ? a.counts[b] : a.N, L = a.lens[b], P = a.prefix_lens[b / (a.B / a.G)];
  const int64_t low = (int64_t)P + L - a.rope_row_offset;  // table row of token 0
  const bool ok = n >= 0 && n <= a.N && L >= 0 && (int64_t)L + n <= a.max_len && P >= 0 &&
                  P <= a.max_prefix && (n == 0 || (low >= 0 && low + n <= a.rope_rows));
  return ok ? Seq{n, L, P} : Seq{-1, 0, 0};
}

// ---- other head sizes and misaligned buffers -----------------------------------
// One workgroup: sequence blockIdx.y, `per` of its N * (Hq + 2 Hkv) rows, a wavefront a
// row: the queries to `qrot`, float32 [B][N][Hq][D], rotated and scaled by D^-1/2 log2(e),
// the new keys and values to the cache.
template <typename T>
__global__ __launch_bounds__(256) void branch_prep_kernel(BranchArgs a, float* __restrict__ qrot,
                                                          int per) {
  const int b = blockIdx.y, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int D = a.D, half = D / 2, heads = a.Hq + 2 * a.Hkv;
  const Seq s = branch_seq(a, b);
  const int64_t r1 = min((int64_t)max(s.n, 0) * heads, (int64_t)(blockIdx.x + 1) * per);
  for (int64_t r = (int64_t)blockIdx.x * per + w; r < r1; r += 4) {
    const int i = (int)(r / heads), h = (int)(r % heads);
    const int64_t tok = (int64_t)b * a.N + i;
    if (h >= a.Hq + a.Hkv) {
      const int g = h - a.Hq - a.Hkv;
      const T* src = (const T*)a.v_new + (tok * a.Hkv + g) * D;
      T* dst = (T*)a.v_cache + (((int64_t)b * a.Hkv + g) * a.Smax + s.L + i) * D;
      for (int d = lane; d < D; d += 64) dst[d] = src[d];
      continue;
    }
    const bool is_q = h < a.Hq;
    const int g = h - a.Hq;
    const T* src = is_q ? (const T*)a.q_new + (tok * a.Hq + h) * D
                        : (const T*)a.k_new + (tok * a.Hkv + g) * D;
    float* qdst = qrot + (tok * a.Hq + h) * D;
    T* kdst = (T*)a.k_cache + (((int64_t)b * a.Hkv + g) * a.Smax + s.L + i) * D;
    const float* nw = is_q ? a.q_norm_w : a.k_norm_w;
    float rs = 1.f;
    if (nw != nullptr) {
      float ss = 0.f;
      for (int d = lane; d < D; d += 64) ss += to_f32(src[d]) * to_f32(src[d]);
      rs = rsqrtf(wave_sum(ss) / (float)D + a.norm_eps);
    }
    const int64_t row = ((int64_t)s.P + s.L + i - a.rope_row_offset) * half;
    for (int d = lane; d < half; d += 64) {
      float x1 = to_f32(src[d]), x2 = to_f32(src[d + half]);
      if (nw != nullptr) {
        x1 = x1 * rs * nw[d];
        x2 = x2 * rs * nw[d + half];
      }
      const float c = a.cos[row + d], sn = a.sin[row + d];
      const float y[2] = {x1 * c - x2 * sn, x2 * c + x1 * sn};
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int at = d + e * half;
        if (is_q)
          qdst[at] = y[e] * (a.scale * kLog2e);
        else
          kdst[at] = from_f32<T>(y[e]);
      }
    }
  }
}

// One wavefront per (b, token, query head), any D <= 256: the prefix, then the own rows
// up to the token's, one key at a time.
template <typename T>
__global__ __launch_bounds__(256) void branch_rows_kernel(BranchArgs a,
                                                          const float* __restrict__ qrot) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= (int64_t)a.B * a.N * a.Hq) return;
  const int hq = (int)(row % a.Hq), i = (int)(row / a.Hq % a.N), b = (int)(row / a.Hq / a.N);
  const int D = a.D, g = hq / (a.Hq / a.Hkv), grp = b / (a.B / a.G);
  const Seq s = branch_seq(a, b);
  T* out = (T*)a.out + row * D;
  if (i >= s.n) {  // a refused sequence, or an unused token
    for (int d = lane; d < D; d += 64) out[d] = from_f32<T>(s.n < 0 ? NAN : 0.f);
    return;
  }
  float qv[4], acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int e = 0; e < 4; ++e) qv[e] = lane + 64 * e < D ? qrot[row * D + lane + 64 * e] : 0.f;
  float m = -INFINITY, l = 0.f;
  auto keys = [&](const void* kc, const void* vc, int64_t pair, int rows, int n) {
    const T* kb = (const T*)kc + pair * rows * D;
    const T* vb = (const T*)vc + pair * rows * D;
    for (int j = 0; j < n; ++j) {
      float x = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (lane + 64 * e < D) x += qv[e] * to_f32(kb[(int64_t)j * D + lane + 64 * e]);
      x = wave_sum(x);
      const float mn = fmaxf(m, x);
      const float ref = mn == -INFINITY ? 0.f : mn;
      const float alpha = fast_exp2(m - ref), p = fast_exp2(x - ref);
      l = l * alpha + p;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        acc[e] = acc[e] * alpha +
                 (lane + 64 * e < D ? p * to_f32(vb[(int64_t)j * D + lane + 64 * e]) : 0.f);
      m = mn;
    }
  };
  keys(a.k_prefix, a.v_prefix, (int64_t)grp * a.Hkv + g, a.Pmax, s.P);
  keys(a.k_cache, a.v_cache, (int64_t)b * a.Hkv + g, a.Smax, s.L + i + 1);
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (lane + 64 * e < D) out[lane + 64 * e] = from_f32<T>(acc[e] / l);
}

size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

template <typename T>
int branch_typed(const BranchArgs& a, void* workspace) {
  float* qrot = (float*)workspace;
  const int per = 16;
  const int64_t rows = (int64_t)a.N * (a.Hq + 2 * a.Hkv);
  KF_LAUNCH("branch_prep", branch_prep_kernel<T>, dim3((unsigned)((rows + per - 1) / per), a.B),
            dim3(256), 0, a.stream, a, qrot, per);
  KF_CHECK_LAUNCH();
  KF_LAUNCH("branch_rows", branch_rows_kernel<T>,
            dim3((unsigned)(((int64_t)a.B * a.N * a.Hq + 3) / 4)), dim3(256), 0, a.stream, a, qrot);
  KF_CHECK_LAUNCH();
  return KF_OK;
}

}  // namespace

size_t branch_workspace(const BranchArgs& a) {
  return up256((size_t)a.B * a.N * a.Hq * a.D * 4);
}

int branch_attention(const BranchArgs& a, void* workspace) {
  switch (a.dtype) {
    case F32: return branch_typed<float>(a, workspace);
    case BF16: return branch_typed<bf16>(a, workspace);
    case F16: return branch_typed<_Float16>(a, workspace);
  }
  set_error("unsupported dtype %d", a.dtype);
  return KF_ERR_UNSUPPORTED;
}

}  // namespace kf
