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
// once, where it is stored; the products take q and P as two numbers of the type each
// (hi + lo: 16 bits of significand in bfloat16, 22 in float16), so that what is left is the
// rounding of the output: the error against 64 bits is its, to 0.1%.
//
// A prefix's keys are met once by the rows of all its sequences, each sequence's own keys
// by its rows; both lists of key chunks are shared out over one launch, and a second joins
// the partials.  Measured, in us (the stream's launch + the merge's), 128 a head:
//   4 sequences behind 1000 keys, 32 / 8 heads          9 + 5: latency
//   4 x 16 behind 8192, up to 512 own, 64 / 8 heads    51 .. 57 + 8: 3.2 TB/s
//   128 behind 4096, up to 2048 own, 32 / 8 heads     125 + 8: 5.2 TB/s, bound by HBM
//   8 x up to 200 tokens behind 4096, 32 / 8 heads    122 .. 158 + 17: a wavefront's scores,
//     exponentials and values in turn, two wavefronts a SIMD (matrix cores busy a third of it)
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
// up to the token's, one key at a time, each row the prefix again (4 sequences behind 1000
// keys, 32 / 8 heads of 96: 0.74 ms; 128 behind 4096 with up to 2048 own 9.7).
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

// ---- split-K attention on the matrix cores -------------------------------------
// New tokens in use of a group, where they are counted (compact rows), else W N.
__device__ __forceinline__ int group_tokens(const BranchArgs& a, int grp, bool compact) {
  const int W = a.B / a.G;
  if (!compact) return W * a.N;
  int n = 0;
#pragma unroll 4
  for (int w = 0; w < W; ++w) n += min(max(a.counts[grp * W + w], 0), a.N);
  return n;
}
__device__ __forceinline__ int prefix_keys(const BranchArgs& a, int grp) {
  const int P = a.prefix_lens[grp];
  return P >= 0 && P <= a.max_prefix ? P : 0;
}
// row of the tables, kept inside them (a refused sequence's may not be)
__device__ __forceinline__ int64_t table_row(const BranchArgs& a, int64_t pos) {
  return min(max(pos - a.rope_row_offset, (int64_t)0), a.rope_rows - 1) * (a.D / 2);
}

// What the stream kernel leaves for the merge.  A: the prefixes' items (group, KV head, row
// tile), B: the sequences' own (sequence, KV head, row tile).  A worker's partial of an
// item lies in slot worker + item: workers of one item and items of one worker are
// consecutive.
struct Lists {
  float *oa, *mla, *ob, *mlb;  // [slot][rows][D], [slot][rows] (m, l)
  int2 *sha, *shb;             // first and last worker of each item
  int rows_a, tiles_a, rows_b, tiles_b, item_b;  // item_b: the first of B's items
  int compact;                 // a group's rows leave out unused tokens
};

// ---- one wavefront a share: up to 16 rows
// A chunk is 32 keys (float32: 16).  Products on 16 x 16 tiles:
//   S^T (keys x rows) = K q^T: lane l supplies key (or row) l % 16, 16 bytes l / 16 of each
//       64 of the row
//   O^T (dims x rows) += V^T P^T: P^T straight from the S registers (lane l holds row l %
//       16, keys 4 (l / 16) .. of each 16); V through the wavefront's LDS and back
//       transposed, or (float32) loaded as the operand is: dim l % 16 of each 16 of keys
//       4 (l / 16) ..
// The next chunk's rows are loaded while one is computed.  Bound by the first round trips
// where shares are few chunks (4 sequences behind 1000 keys: one chunk each), by HBM where
// they are long: 32 sequences of 8192 own keys stream at 6.0 TB/s.
template <typename T>
constexpr int WK = sizeof(T) == 4 ? 16 : 32;  // keys of a chunk

// Entities of the list: (ALL) the groups' prefixes, then the sequences' own rows: the chunks
// of what is cached, then one of the new tokens (16 at most).
template <bool ALL, int WKEYS>
struct WaveSched {
  const BranchArgs& a;
  int G0, B, C;  // groups in front, entities, chunks
  // entity `lane`'s, all there are up to 64 of them: cached keys, new tokens (0: a prefix),
  // keys of the prefix
  int3 own{0, 0, 0};
  __device__ __forceinline__ WaveSched(const BranchArgs& a_, int lane)
      : a(a_), G0(ALL ? a_.G : 0), B(G0 + a_.B) {
    int n = 0;
    for (int e = lane; e < B; e += 64) {
      own = keys(e);
      n += nck(own) * a.Hkv;
    }
    C = __builtin_amdgcn_readlane(wave_prefix(n), 63);
  }
  __device__ __forceinline__ int3 keys(int e) const {
    if (ALL && e < G0) return make_int3(prefix_keys(a, e), 0, 0);
    const Seq s = branch_seq(a, e - G0);
    return s.n > 0 ? make_int3(s.L, s.n, s.P) : make_int3(0, 0, 0);
  }
  __device__ __forceinline__ int3 keys_of(int e) const {  // (uniform e)
    const int3 x = B <= 64 ? own : keys(e);
    const int at = B <= 64 ? e : 0;
    return make_int3(__builtin_amdgcn_readlane(x.x, at), __builtin_amdgcn_readlane(x.y, at),
                     __builtin_amdgcn_readlane(x.z, at));
  }
  static __device__ __forceinline__ int nck(int3 k) { return (k.x + WKEYS - 1) / WKEYS + (k.y > 0); }
  __device__ __forceinline__ int chunks(int e) const { return nck(keys(e)) * a.Hkv; }
  // the entity that holds a chunk, and its first one
  __device__ __forceinline__ void locate(int c, int lane, int& e, int& base) const {
    if (B > 64) {
      locate_chunk(*this, c, lane, e, base);
      return;
    }
    const int n = nck(own) * a.Hkv, end = wave_prefix(n);
    e = __builtin_ctzll(__builtin_amdgcn_ballot_w64(end - n <= c && c < end) | 1ull << 63);
    base = __builtin_amdgcn_readlane(end - n, e);
  }
};

template <typename T, int D>
struct WaveLds {
  T v[sizeof(T) == 4 ? 4 : WK<T> * D];
};

template <typename T, int D, bool ALL>
__device__ __forceinline__ void wave_role(const BranchArgs& a, const Lists& ls, char* lds,
                                          const WaveSched<ALL, WK<T>>& sched, int gw, int NW) {
  using namespace mfma;
  using P = Piece<T>;
  constexpr bool F32T = sizeof(T) == 4;
  constexpr int E = P::E, KEYS = WK<T>, NB = KEYS / 16;  // values of 16 bytes, blocks of 16 keys
  constexpr int KT = D / (4 * E), DB = D / 16, KR = D / E, HALF = D / 2;
  constexpr int VL = KEYS * KR / 64;
  // P = 2^(s - m + LIFT), m moved only when a score is 2^SLACK above it (as in the tiles below):
  // chunk after chunk nothing crosses lanes
  constexpr bool HALF_P = std::is_same<T, _Float16>::value;
  constexpr float SLACK = HALF_P ? 2.f : 8.f, LIFT = HALF_P ? 13.f : 0.f;
  if (gw >= NW) return;
  gw = __builtin_amdgcn_readfirstlane(gw);
  const int w = wave_id(), lane = threadIdx.x & 63, q4 = lane >> 4, c16 = lane & 15;
  T* lv = ((WaveLds<T, D>*)lds)[w].v;
  const int n_rep = a.Hq / a.Hkv, W = a.B / a.G, N = a.N;
  const int c_lo = range_start(gw, sched.C, NW), c_hi = range_start(gw + 1, sched.C, NW);

  struct Cursor {
    int e, g, lc, nck;
    int3 k;  // cached keys, new tokens (0: a prefix), keys of the prefix
  };
  auto enter = [&](Cursor& c, int e) {
    c.e = e;
    c.k = sched.keys_of(e);
    c.nck = sched.nck(c.k);
  };
  auto next = [&](Cursor& c) {
    if (++c.lc < c.nck) return;
    c.lc = 0;
    if (++c.g < a.Hkv) return;
    c.g = 0;
    do
      enter(c, c.e + 1);
    while (c.nck == 0 && c.e + 1 < sched.B);
  };
  auto is_prefix = [&](const Cursor& c) { return ALL && c.e < sched.G0; };
  auto is_new = [&](const Cursor& c) { return c.k.y > 0 && c.lc == c.nck - 1; };
  auto chunk_rows = [&](const Cursor& c) { return is_new(c) ? c.k.y : min(c.k.x - c.lc * KEYS, KEYS); };
  // A chunk's row r begins at base + r * stride; rows behind the last repeat it.  The caches
  // are read once a step: non-temporal loads.
  struct Rows {
    const T* base;
    uint32_t stride;
    int last;
  };
  // (the tensors by their distance from one of them: a choice of pointers would be kept
  // in memory)
  auto rows_of = [&](const Cursor& c, const void* pre, const void* own, const void* fresh) {
    const int64_t b = c.e - sched.G0;
    int64_t at = (((b * a.Hkv + c.g) * a.Smax + c.lc * KEYS) * D) * (int)sizeof(T);
    if (is_prefix(c))
      at = ((const char*)pre - (const char*)own) +
           ((((int64_t)c.e * a.Hkv + c.g) * a.Pmax + c.lc * KEYS) * D) * (int)sizeof(T);
    if (is_new(c))
      at = ((const char*)fresh - (const char*)own) + (b * N * a.Hkv + c.g) * D * (int)sizeof(T);
    Rows r;
    r.base = (const T*)((const char*)own + at);
    r.stride = is_new(c) ? a.Hkv * D : D;
    r.last = chunk_rows(c) - 1;
    return r;
  };
  u32x4 kreg[NB][KT];  // key 16 kb + c16 of the chunk, dims 4 E ks + E q4 ..
  // V row (64 j + lane) / KR, piece (64 j + lane) % KR; (float32) key 4 q4 + t, dim 16 blk + c16
  // at t * DB + blk
  u32x4 vreg[F32T ? 1 : VL];
  float vf[F32T ? 4 * DB : 1];
  auto load_k = [&](const Cursor& c) {
    const Rows r = rows_of(c, a.k_prefix, a.k_cache, a.k_new);
#pragma unroll
    for (int kb = 0; kb < NB; ++kb) {
      const uint32_t off = (uint32_t)min(16 * kb + c16, r.last) * r.stride + E * q4;
#pragma unroll
      for (int ks = 0; ks < KT; ++ks)
        kreg[kb][ks] = __builtin_nontemporal_load((const u32x4*)(r.base + off + 4 * E * ks));
    }
  };
  auto load_v = [&](const Cursor& c) {
    const Rows r = rows_of(c, a.v_prefix, a.v_cache, a.v_new);
    if constexpr (F32T) {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const uint32_t off = (uint32_t)min(4 * q4 + t, r.last) * r.stride + c16;
#pragma unroll
        for (int blk = 0; blk < DB; ++blk)
          vf[t * DB + blk] = __builtin_nontemporal_load(r.base + off + 16 * blk);
      }
    } else {
#pragma unroll
      for (int j = 0; j < VL; ++j) {
        const int li = 64 * j + lane;
        const uint32_t off = (uint32_t)min(li / KR, r.last) * r.stride + li % KR * 8;
        vreg[j] = __builtin_nontemporal_load((const u32x4*)(r.base + off));
      }
    }
  };
  // Pieces of a row (dims d ..) and of its other half, rotated, after the norm if there is one.
  struct Angles {
    float c[E], s[E];
  };
  auto angles = [&](int64_t trow, int d) {
    Angles g;
#pragma unroll
    for (int x = 0; x < E; x += 4) {
      *(f32x4*)(g.c + x) = *(const f32x4*)(a.cos + trow + d + x);
      *(f32x4*)(g.s + x) = *(const f32x4*)(a.sin + trow + d + x);
    }
    return g;
  };
  auto rotate = [&](float* f1, float* f2, const Angles& g, int d, const float* nw, float rs) {
    if (nw != nullptr) {
#pragma unroll
      for (int x = 0; x < E; ++x) {
        f1[x] = f1[x] * rs * nw[d + x];
        f2[x] = f2[x] * rs * nw[d + HALF + x];
      }
    }
#pragma unroll
    for (int x = 0; x < E; ++x) {
      const float y1 = f1[x] * g.c[x] - f2[x] * g.s[x];
      f2[x] = f2[x] * g.c[x] + f1[x] * g.s[x];
      f1[x] = y1;
    }
  };
  auto row_norm = [&](const u32x4* raw) {  // the row's four lanes hold its pieces
    float ss = 0.f;
#pragma unroll
    for (int ks = 0; ks < KT; ++ks) {
      float f[E];
      P::unpack(raw[ks], f);
#pragma unroll
      for (int x = 0; x < E; ++x) ss += f[x] * f[x];
    }
    ss += __shfl_xor(ss, 16, 64);
    ss += __shfl_xor(ss, 32, 64);
    return rsqrtf(ss / (float)D + a.norm_eps);
  };

  // transposed-read byte offsets of this lane in the V tile, per 16-dim block: address lane
  // c16 of group q4 reads row 4 q4 + c16 / 4, dims 16 blk + 4 (c16 % 4) .. + 3 (the second
  // read: row + 16, the same swizzle)
  const int tr_row = 4 * q4 + (c16 >> 2), tr_sw = swz<KR>(tr_row);
  const uint32_t tr_base = (uint32_t)((tr_row * KR + (((c16 & 3) >> 1) ^ (tr_sw & 1))) * 16 +
                                      (4 * (c16 & 1)) * 2);
  const int tr_hs = tr_sw >> 1;

  u32x4 qh[KT], ql[F32T ? 1 : KT];
  f32x4 acc[DB];
  float m = -INFINITY, lsum = 0.f;
  int token = 0;  // the lane's row's, of its sequence's new tokens
  Cursor cc;
  {
    int e, base;
    sched.locate(c_lo, lane, e, base);
    enter(cc, e);
    cc.g = __builtin_amdgcn_readfirstlane((c_lo - base) / max(cc.nck, 1));
    cc.lc = c_lo - base - cc.g * cc.nck;
  }
  // A pair's queries: the lane's row of them and of the tables, then rotated.
  auto pair_rows = [&](const Cursor& c) { return (is_prefix(c) ? W * N : c.k.y) * n_rep; };
  auto load_q = [&](const Cursor& c, u32x4* raw, Angles* ang) {
    int ln = lane;
    asm volatile("" : "+v"(ln));  // (nothing of this is kept across the loop)
    const int q4 = ln >> 4, c16 = ln & 15;
    const bool pre = is_prefix(c);
    const int r = min(c16, pair_rows(c) - 1), tok = r / n_rep;
    const int at = pre ? tok / N : 0;
    const int64_t b = pre ? c.e * W + at : c.e - sched.G0;
    token = pre ? tok - at * N : tok;
    const T* qr =
        (const T*)a.q_new + ((b * N + token) * a.Hq + (int64_t)c.g * n_rep + r % n_rep) * D + E * q4;
#pragma unroll
    for (int ks = 0; ks < KT; ++ks) raw[ks] = *(const u32x4*)(qr + 4 * E * ks);
    int64_t pos = (int64_t)c.k.z + c.k.x + token;
    if (pre)
      pos = (int64_t)c.k.x + token +
            (sched.B <= 64 ? __shfl(sched.own.x, (int)b + sched.G0, 64) : a.lens[b]);
    const int64_t trow = table_row(a, pos);
#pragma unroll
    for (int ks = 0; ks < KT / 2; ++ks) ang[ks] = angles(trow, 4 * E * ks + E * q4);
  };
  auto rotate_q = [&](const u32x4* raw, const Angles* ang) {
    int ln = lane;
    asm volatile("" : "+v"(ln));
    const int q4 = ln >> 4;
    const float rs = a.q_norm_w != nullptr ? row_norm(raw) : 1.f;
    const float sc = a.scale * kLog2e;
#pragma unroll
    for (int ks = 0; ks < KT / 2; ++ks) {
      float f[2][E];
      P::unpack(raw[ks], f[0]);
      P::unpack(raw[ks + KT / 2], f[1]);
      rotate(f[0], f[1], ang[ks], 4 * E * ks + E * q4, a.q_norm_w, rs);
      __builtin_amdgcn_sched_barrier(0);  // (registers)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
#pragma unroll
        for (int y = 0; y < E; ++y) f[x][y] *= sc;
        qh[ks + x * (KT / 2)] = P::pack(f[x]);
        if constexpr (!F32T) {
          float hi[E];
          P::unpack(qh[ks + x * (KT / 2)], hi);
#pragma unroll
          for (int y = 0; y < E; ++y) f[x][y] -= hi[y];
          ql[ks + x * (KT / 2)] = P::pack(f[x]);
        }
      }
    }
    m = -INFINITY;
    lsum = 0.f;
#pragma unroll
    for (int blk = 0; blk < DB; ++blk) acc[blk] = f32x4{0.f, 0.f, 0.f, 0.f};
  };
  {
    // (the queries first: loads return in order)
    u32x4 raw[KT];
    Angles ang[KT / 2];
    load_q(cc, raw, ang);
    __builtin_amdgcn_sched_barrier(0);
    load_k(cc);
    load_v(cc);
    __builtin_amdgcn_sched_barrier(0);
    rotate_q(raw, ang);
  }
  for (int i = c_lo; i < c_hi; ++i) {
    const bool pre = is_prefix(cc), fresh = is_new(cc), more = i + 1 < c_hi;
    const int keys = chunk_rows(cc);
    const int64_t b0 = cc.e - sched.G0;  // (own) the sequence
    if (i > c_lo && cc.lc == 0) {        // a pair begins
      u32x4 raw[KT];
      Angles ang[KT / 2];
      load_q(cc, raw, ang);
      rotate_q(raw, ang);
    }
    uint32_t bad = 0;  // V rows with Inf or NaN that not all rows see
    if (fresh) {       // (16 keys at most: kb = 0)
      int ln = lane;
      asm volatile("" : "+v"(ln));  // (nothing of this block is kept across the loop)
      const int q4 = ln >> 4, c16 = ln & 15;
      const int64_t at = (b0 * a.Hkv + cc.g) * a.Smax + cc.k.x;  // the first new row
      const float rs = a.k_norm_w != nullptr ? row_norm(kreg[0]) : 1.f;
      if (c16 < keys) {
        const int64_t trow = table_row(a, (int64_t)cc.k.z + cc.k.x + c16);
        T* dst = (T*)a.k_cache + (at + c16) * D + E * q4;
#pragma unroll
        for (int ks = 0; ks < KT / 2; ++ks) {
          float f[2][E];
          const int d = 4 * E * ks + E * q4;
          P::unpack(kreg[0][ks], f[0]);
          P::unpack(kreg[0][ks + KT / 2], f[1]);
          rotate(f[0], f[1], angles(trow, d), d, a.k_norm_w, rs);
          __builtin_amdgcn_sched_barrier(0);  // (registers)
          kreg[0][ks] = P::pack(f[0]);
          kreg[0][ks + KT / 2] = P::pack(f[1]);
          *(u32x4*)(dst + 4 * E * ks) = kreg[0][ks];
          *(u32x4*)(dst + 4 * E * ks + HALF) = kreg[0][ks + KT / 2];
        }
      }
      // (one new token: every row sees it)
      if constexpr (F32T) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const int row = 4 * q4 + t;
          T* dst = (T*)a.v_cache + (at + row) * D + c16;
          bool fin = true;
          if (row < keys)
#pragma unroll
            for (int blk = 0; blk < DB; ++blk) {
              dst[16 * blk] = vf[t * DB + blk];
              fin = fin && finite(vf[t * DB + blk]);
            }
          const uint64_t x = keys > 1 ? __builtin_amdgcn_ballot_w64(!fin) : 0;
#pragma unroll
          for (int y = 0; y < 4; ++y) bad |= (x >> (16 * y) & 0xffff ? 1u : 0u) << (4 * y + t);
        }
      } else {
#pragma unroll
        for (int j = 0; j < VL / 2; ++j) {
          const int li = 64 * j + ln, row = li / KR, pc = li % KR;
          bool fin = true;
          if (row < keys) {
            *(u32x4*)((T*)a.v_cache + (at + row) * D + 8 * pc) = vreg[j];
            float f[8];
            unpack8<T>(vreg[j], f);
#pragma unroll
            for (int x = 0; x < 8; ++x) fin = fin && finite(f[x]);
          }
          const uint64_t x = keys > 1 ? __builtin_amdgcn_ballot_w64(!fin) : 0;
#pragma unroll
          for (int y = 0; y < 64 / KR; ++y)
            bad |= (x >> (y * KR) & ((1ull << KR) - 1) ? 1u : 0u) << (64 / KR * j + y);
        }
      }
    }
    Cursor ic = cc;
    if (more) next(ic);
    f32x4 sc[NB], sl[NB];
#pragma unroll
    for (int kb = 0; kb < NB; ++kb) {
      sc[kb] = sl[kb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KT; ++ks) {
        if constexpr (F32T) {  // (two sums: each waits for its own last product)
          const f32x4 x = __builtin_bit_cast(f32x4, kreg[kb][ks]),
                      y = __builtin_bit_cast(f32x4, qh[ks]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            f32x4& s = e & 1 ? sl[kb] : sc[kb];
            s = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], s, 0, 0, 0);
          }
        } else {
          sc[kb] = mfma16<T>(as_bf16x8(kreg[kb][ks]), as_bf16x8(qh[ks]), sc[kb]);
          sl[kb] = mfma16<T>(as_bf16x8(kreg[kb][ks]), as_bf16x8(ql[ks]), sl[kb]);
        }
      }
    }
    if (more) load_k(ic);
    float tmax = -INFINITY;
#pragma unroll
    for (int kb = 0; kb < NB; ++kb) sc[kb] += sl[kb];
    // (a new token sees those before it and itself: 16 of them fill a chunk of float32)
    if (fresh || keys < KEYS) {
      const int limit = fresh ? token + 1 : keys;
#pragma unroll
      for (int t = 0; t < 4 * NB; ++t)
        sc[t / 4][t % 4] =
            16 * (t / 4) + 4 * q4 + t % 4 < limit ? sc[t / 4][t % 4] : -INFINITY;
    }
#pragma unroll
    for (int t = 0; t < 4 * NB; ++t) tmax = fmaxf(tmax, sc[t / 4][t % 4]);
    if (__builtin_amdgcn_ballot_w64(tmax > m + SLACK || m == -INFINITY)) {
      tmax = fmaxf(tmax, __shfl_xor(tmax, 16, 64));
      tmax = fmaxf(tmax, __shfl_xor(tmax, 32, 64));
      const float mnew = fmaxf(m, tmax);
      const float alpha = m == -INFINITY ? 0.f : fast_exp2(m - mnew);
      m = mnew;
      lsum *= alpha;
#pragma unroll
      for (int blk = 0; blk < DB; ++blk) acc[blk] *= alpha;
    }
    const float ref = (m == -INFINITY ? 0.f : m) - LIFT;  // (-inf: no key yet)
    float p[4 * NB];
#pragma unroll
    for (int t = 0; t < 4 * NB; ++t) {
      p[t] = fast_exp2(sc[t / 4][t % 4] - ref);
      lsum += p[t];
    }
    if constexpr (F32T) {
      if (keys < KEYS || bad)  // (rows behind the last, and those of `bad`: 0 x NaN)
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const bool drop = 4 * q4 + t >= keys || (bad >> (4 * q4 + t) & 1);
#pragma unroll
          for (int blk = 0; blk < DB; ++blk) vf[t * DB + blk] = drop ? 0.f : vf[t * DB + blk];
        }
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int blk = 0; blk < DB; ++blk)
          acc[blk] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf[t * DB + blk], p[t], acc[blk], 0, 0, 0);
      if (more) load_v(ic);
    } else {
      u32x4 ph, pl;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const uint2 u = Tile<T, D>::split2(p[2 * t], p[2 * t + 1]);
        ph[t] = u.x;
        pl[t] = u.y;
      }
      // V rows into the tile (rows behind the last, and those of `bad`, as zeros)
#pragma unroll
      for (int j = 0; j < VL; ++j) {
        const int li = 64 * j + lane, row = li / KR, pc = li % KR;
        const bool drop = row >= keys || (bad >> row & 1);
        *(u32x4*)(lv + (row * KR + (pc ^ swz<KR>(row))) * 8) = drop ? u32x4{0u, 0u, 0u, 0u} : vreg[j];
      }
      if (more) load_v(ic);
#pragma unroll
      for (int blk = 0; blk < DB; ++blk) {
        const char* base = (const char*)lv + tr_base + (uint32_t)((blk ^ tr_hs) * 32);
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)base);
        const s16x4 hi =
            __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(base + 16 * KR * 16));
        const bf16x8 vt =
            __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        acc[blk] = mfma16<T>(vt, as_bf16x8(ph), acc[blk]);
        acc[blk] = mfma16<T>(vt, as_bf16x8(pl), acc[blk]);
      }
    }
    for (uint32_t x = bad; x; x &= x - 1) {  // one by one, for the rows that see them
      const int r = __builtin_ctz(x);
      float pr = 0.f;
#pragma unroll
      for (int t = 0; t < 4; ++t)
        if (t == (r & 3)) pr = p[t];
      pr = __shfl(pr, c16 + 16 * (r >> 2), 64);
      if (r <= token) {
        const T* vr = (const T*)a.v_new + ((b0 * N + r) * a.Hkv + cc.g) * D + 4 * q4;
#pragma unroll
        for (int blk = 0; blk < DB; ++blk)
#pragma unroll
          for (int y = 0; y < 4; ++y) acc[blk][y] += pr * to_f32(vr[16 * blk + y]);
      }
    }
    const bool last = cc.lc == cc.nck - 1;
    const int item = cc.e * a.Hkv + cc.g;
    if (lane == 0 && (cc.lc == 0 || last)) {
      int2* sh = ls.shb + (pre ? ls.sha - ls.shb + item : item - sched.G0 * a.Hkv);
      if (cc.lc == 0) sh->x = gw;
      if (last) sh->y = gw;
    }
    if (!more || last) {  // the pair's part of this wavefront ends
      int ln = lane;
      asm volatile("" : "+v"(ln));  // (as above)
      const int q4 = ln >> 4, c16 = ln & 15;
      float l = lsum + __shfl_xor(lsum, 16, 64);
      l += __shfl_xor(l, 32, 64);
      if (c16 < pair_rows(cc)) {
        const int64_t at = ((int64_t)gw + item) * ls.rows_b + c16;
        float* o = ls.ob + at * D + 4 * q4;
#pragma unroll
        for (int blk = 0; blk < DB; ++blk) *(f32x4*)(o + 16 * blk) = acc[blk];
        if (q4 == 0)  // (a NaN must not be left out for its weight)
          *(float2*)(ls.mlb + at * 2) = make_float2(l != l ? INFINITY : m, l);
      }
    }
    cc = ic;
  }
}

// ---- a workgroup a share: row tiles of 32 RW rows
// Entities: the groups (PREFIX: the tokens of their sequences over the prefix), the sequences
// (OWN: their tokens over their own rows), or the sequences over both (BOTH: where a
// sequence's tokens fill tiles of their own, so that nothing has to be joined).  Row r of an
// entity is query head r % n_rep of the KV head's of its token r / n_rep.  A tile meets the
// chunks of the prefix, then those of the own rows up to its last token's.
//
// Beginning a row tile and leaving its partial cost about as much as OVER chunks, so with
// several chunks per workgroup each tile has OVER units in front of its chunks in the list
// that is shared out.  (Without them the own rows' tiles of one chunk count for so little
// that a few workgroups get them all: 4 sequences of 64 new tokens behind 16384 keys, 64 / 8
// heads: 681 us.)
enum Role : int { PREFIX, OWN, BOTH };
constexpr int OVER = 2;
// tokens, own keys (the new tokens' among them), keys of the prefix
struct Entity {
  int n, y, p;
};
template <int ROLE>
struct TileSched {
  const BranchArgs& a;
  int n_rep, rows, kc, E, C, items, over = 0;  // C: units; items: tiles
  bool compact;
  Entity own{0, 0, 0};  // entity `lane`'s, all there are up to 64 of them
  __device__ __forceinline__ TileSched(const BranchArgs& a_, int rows_, int kc_, bool compact_,
                                       int lane)
      : a(a_), n_rep(a_.Hq / a_.Hkv), rows(rows_), kc(kc_), E(ROLE == PREFIX ? a_.G : a_.B),
        compact(compact_) {
    int tot = 0, n = 0;
    for (int e = lane; e < E; e += 64) {
      own = entity(e);
      tot += units(own);
      n += own.y + own.p > 0 ? a.Hkv * tiles(own) : 0;
    }
    C = __builtin_amdgcn_readlane(wave_prefix(tot), 63);
    items = __builtin_amdgcn_readlane(wave_prefix(n), 63);
  }
  __device__ __forceinline__ void count_beginnings() {
    over = OVER;
    C += OVER * items;
  }
  __device__ __forceinline__ Entity entity(int e) const {
    if (ROLE == PREFIX) return Entity{group_tokens(a, e, compact), 0, prefix_keys(a, e)};
    const Seq s = branch_seq(a, e);
    return s.n > 0 ? Entity{s.n, s.L + s.n, ROLE == BOTH ? s.P : 0} : Entity{0, 0, 0};
  }
  __device__ __forceinline__ Entity entity_of(int e) const {  // (uniform e)
    Entity x = E <= 64 ? own : entity(e);
    const int at = E <= 64 ? e : 0;
    return Entity{__builtin_amdgcn_readlane(x.n, at), __builtin_amdgcn_readlane(x.y, at),
                  __builtin_amdgcn_readlane(x.p, at)};
  }
  __device__ __forceinline__ int tiles(Entity s) const { return (s.n * n_rep + rows - 1) / rows; }
  __device__ __forceinline__ int prefix_chunks(Entity s) const { return (s.p + kc - 1) / kc; }
  // the last key of its own that a tile of the sequence sees, and one
  __device__ __forceinline__ int reach(Entity s, int t) const {
    return s.y - s.n + min(((t + 1) * rows - 1) / n_rep + 1, s.n);
  }
  __device__ __forceinline__ int nck(Entity s, int t) const {
    return prefix_chunks(s) + (ROLE == PREFIX ? 0 : (reach(s, t) + kc - 1) / kc);
  }
  // of one KV head
  __device__ __forceinline__ int head_units(Entity s) const {
    if (s.y + s.p == 0) return 0;
    const int n = tiles(s);
    if (ROLE == PREFIX) return n * (prefix_chunks(s) + over);
    int u = 0;
    for (int t = 0; t < n; ++t) u += nck(s, t) + over;
    return u;
  }
  __device__ __forceinline__ int units(Entity s) const { return a.Hkv * head_units(s); }
  // the first unit of worker w's share of n, floor(w C / n) (w and n are far below 2^16)
  __device__ __forceinline__ int start(int w, int n) const {
    const unsigned q = (unsigned)C / n, r = (unsigned)C % n;
    return (int)(w * q + (unsigned)w * r / n);
  }
  // for locate_chunk
  int B = E;
  __device__ __forceinline__ int chunks(int e) const { return units(entity(e)); }
};

// Place in the list: entity e, KV head g, row tile t, chunk c of nck, unit u.
template <int ROLE>
struct TileCursor {
  using S = TileSched<ROLE>;
  int e, g, t, c, u, nck, tiles, pck;  // pck: chunks of the prefix
  Entity s;
  __device__ __forceinline__ void at(const S& sched, int e_) {
    e = e_;
    s = sched.entity_of(e);
    tiles = sched.tiles(s);
    pck = sched.prefix_chunks(s);
  }
  __device__ __forceinline__ void seek(const S& sched, int unit, int lane) {
    int se, base;
    if (sched.E <= 64) {  // a lane an entity, without another load
      const int n = sched.units(sched.own), end = wave_prefix(n);
      se = __builtin_ctzll(__builtin_amdgcn_ballot_w64(end - n <= unit && unit < end) | 1ull << 63);
      base = __builtin_amdgcn_readlane(end - n, se);
    } else {
      locate_chunk(sched, unit, lane, se, base);
    }
    at(sched, se);
    const int per = sched.head_units(s);
    int off = unit - base;
    g = off / per;
    off -= g * per;
    u = unit - off;
    if (ROLE == PREFIX) {
      t = off / (pck + sched.over);
      u += t * (pck + sched.over);
      off -= t * (pck + sched.over);
      nck = pck;
    } else {
      for (t = 0;; ++t) {
        nck = sched.nck(s, t);
        if (off < nck + sched.over || t == tiles - 1) break;
        off -= nck + sched.over;
        u += nck + sched.over;
      }
    }
    c = max(off - sched.over, 0);
    u += sched.over + c;
  }
  __device__ __forceinline__ void next(const S& sched) {
    ++u;
    if (++c < nck) return;
    c = 0;
    u += sched.over;
    if (++t >= tiles) {
      t = 0;
      if (++g >= sched.a.Hkv) {
        g = 0;
        do {
          if (++e >= sched.E) return;  // behind the last chunk (u is past every share)
          at(sched, e);
        } while (s.y + s.p == 0 || tiles == 0);
      }
    }
    nck = sched.nck(s, t);
  }
};

// (a value that is the same for all lanes, in scalar registers)
__device__ __forceinline__ int64_t uniform(int64_t x) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)x),
                 hi = __builtin_amdgcn_readfirstlane((uint32_t)(x >> 32));
  return (int64_t)((uint64_t)hi << 32 | lo);
}

constexpr int MAX_COMPACT = 1024;  // sequences of a group whose rows are counted

template <typename T, int D, int RW, int BKW, int ROLE>
__device__ __forceinline__ void tile_role(const BranchArgs& a, const Lists& ls, char* lds, int* pre,
                                          uint32_t* sbad, const TileSched<ROLE>& sched, int blk,
                                          int nblk) {
  using namespace mfma;
  using X = Tile<T, D>;
  using P = Piece<T>;
  using Sh = Shape<T, D, RW, BKW>;
  constexpr int KW = Sh::KW, ROWS = Sh::ROWS, KC = Sh::KC, NB = BKW / 32, DT = D / 32;
  constexpr int E = P::E, HALF = D / 2;
  const int w = wave_id(), lane = threadIdx.x & 63, h = lane >> 5, l31 = lane & 31;
  const int rw = w % RW, kw = w / RW;
  const int N = a.N, W = a.B / a.G, n_rep = a.Hq / a.Hkv;
  const int NW = min(nblk, sched.C);
  // block ids go round the 8 XCDs: neighbours in the list, which read the same keys for
  // other rows, share one XCD's L2
  if (blk >= NW) return;
  const int xcd = blk % 8, gw = xcd * (NW / 8) + min(xcd, NW % 8) + blk / 8;
  const int u_hi = sched.start(gw + 1, NW);
  TileCursor<ROLE> cc;
  cc.seek(sched, sched.start(gw, NW), lane);
  if (cc.u >= u_hi) return;  // (a share of nothing but a tile's beginning)

  // A chunk is KC keys of the prefix or of the own rows, from key `key0` of keys `keys`.
  auto of_prefix = [&](const TileCursor<ROLE>& p) {
    return ROLE == PREFIX || (ROLE == BOTH && p.c < p.pck);
  };
  auto stage_k = [&](int i) { return (T*)(lds + (i & 1) * Sh::STAGE); };
  auto issue = [&](const TileCursor<ROLE>& p, int i) {
    const bool pre = of_prefix(p);
    const int key0 = (pre ? p.c : p.c - p.pck) * KC;
    const int64_t b = ROLE == BOTH && pre ? p.e / W : p.e;
    // (the tensors by their distance from one of them, as in the wavefronts' list)
    int64_t at = ((b * a.Hkv + p.g) * (pre ? a.Pmax : a.Smax) + key0) * (D * (int)sizeof(T));
    int64_t vt = at;
    if (ROLE == BOTH && pre) {
      at += (const char*)a.k_prefix - (const char*)a.k_cache;
      vt += (const char*)a.v_prefix - (const char*)a.v_cache;
    }
    const char* kb = (const char*)(ROLE == PREFIX ? a.k_prefix : a.k_cache) + uniform(at);
    const char* vb = (const char*)(ROLE == PREFIX ? a.v_prefix : a.v_cache) + uniform(vt);
    const int rows = (pre ? p.s.p : p.s.y) - key0;  // >= 1; rows past the last repeat it
    uint16_t* dst = (uint16_t*)stage_k(i);
    constexpr int U = sizeof(T) / 2;
    constexpr bool FRESH = RW == 2;  // (registers)
    tile_to_lds<KC, X::R, 4, FRESH>((const uint16_t*)kb, D * U, dst, w, lane, rows);
    tile_to_lds<KC, X::R, 4, FRESH>((const uint16_t*)vb, D * U, dst + Sh::TILE * U, w, lane, rows);
  };
  // E pairs of one row rotated (and normalised by rs with weights nw first)
  struct Angles {
    f32x4 c[E / 4], s[E / 4];
  };
  auto angles = [&](int64_t trow, int d) {
    Angles g;
#pragma unroll
    for (int x = 0; x < E / 4; ++x) {
      g.c[x] = *(const f32x4*)(a.cos + trow + d + 4 * x);
      g.s[x] = *(const f32x4*)(a.sin + trow + d + 4 * x);
    }
    return g;
  };
  auto rotate = [&](float* f1, float* f2, const Angles& g, int d, const float* nw, float rs) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (nw != nullptr) {
        f1[e] = f1[e] * rs * nw[d + e];
        f2[e] = f2[e] * rs * nw[d + HALF + e];
      }
      const float c = g.c[e / 4][e % 4], sn = g.s[e / 4][e % 4];
      const float y1 = f1[e] * c - f2[e] * sn;
      f2[e] = f2[e] * c + f1[e] * sn;
      f1[e] = y1;
    }
  };

  const typename X::VOff voff = X::v_off(lane);
  u32x4 q[X::QP][X::KS];
  f32x16 acc[DT];
  float m = -INFINITY, lsum = 0.f;
  // P = 2^(s - m + LIFT) stays below 2^(SLACK + LIFT); float16 fills its range up to 2^15, as
  // it has no numbers below 2^-24.
  constexpr bool HALF_P = std::is_same<T, _Float16>::value;
  constexpr float SLACK = HALF_P ? 2.f : 8.f, LIFT = HALF_P ? 13.f : 0.f;
  int limit = 0;  // own keys that the lane's row sees
  bool whole = false;  // (BOTH) this workgroup holds all of the row tile's chunks

  // the first compact token of each of a group's sequences (exclusive sums)
  auto count_group = [&](int grp) {
    __syncthreads();  // the previous group's readers are done
    if (w == 0) {
      int run = 0;
      for (int w0 = 0; w0 < W; w0 += 64) {
        const int i = w0 + lane;
        const int n = i < W ? min(max(a.counts[grp * W + i], 0), N) : 0;
        const int end = wave_prefix(n);
        if (i < W) pre[i] = run + end - n;
        run += __builtin_amdgcn_readlane(end, 63);
      }
    }
    __syncthreads();
  };
  // The beginning of a row tile: lane l's row of the queries, dims of half h, 16-byte pieces
  // 2 ks + h; a piece's RoPE partner is the lane's own piece KS / 2 further on.
  auto load_q = [&](u32x4* raw, int64_t& trow) {
    const int row = min(cc.t * ROWS + 32 * rw + l31, cc.s.n * n_rep - 1);
    const int tok = row / n_rep;
    int b = cc.e, i = tok;
    if (ROLE == PREFIX) {
      int at;
      if (sched.compact) {
        int lo = 0, hi = W;  // the last sequence that begins at or before the token
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (pre[mid] <= tok)
            lo = mid;
          else
            hi = mid;
        }
        at = lo;
        i = tok - pre[lo];
      } else {
        at = tok / N;
        i = tok % N;
      }
      b = cc.e * W + at;
    }
    const T* qr = (const T*)a.q_new +
                  (((int64_t)b * N + i) * a.Hq + (int64_t)cc.g * n_rep + row % n_rep) * D;
#pragma unroll
    for (int ks = 0; ks < X::KS; ++ks) raw[ks] = *(const u32x4*)(qr + (2 * ks + h) * E);
    const int L = a.lens[b];
    trow = table_row(a, (int64_t)a.prefix_lens[b / W] + L + i);
    limit = L + i + 1;
  };
  auto load_angles = [&](Angles* ang, int64_t trow) {  // (one round trip for all)
#pragma unroll
    for (int ks = 0; ks < X::KS / 2; ++ks) ang[ks] = angles(trow, (2 * ks + h) * E);
  };
  auto rotate_q = [&](const u32x4* raw, const Angles* ang) {
    float rs = 1.f;
    if (a.q_norm_w != nullptr) {
      float ss = 0.f;
#pragma unroll
      for (int ks = 0; ks < X::KS; ++ks) {
        float f[E];
        P::unpack(raw[ks], f);
#pragma unroll
        for (int e = 0; e < E; ++e) ss += f[e] * f[e];
      }
      rs = rsqrtf(pair_sum32(ss) / (float)D + a.norm_eps);
    }
    const float sc = a.scale * kLog2e;
#pragma unroll
    for (int ks = 0; ks < X::KS / 2; ++ks) {
      float f[2][E];
      P::unpack(raw[ks], f[0]);
      P::unpack(raw[ks + X::KS / 2], f[1]);
      rotate(f[0], f[1], ang[ks], (2 * ks + h) * E, a.q_norm_w, rs);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int at = ks + x * (X::KS / 2);
#pragma unroll
        for (int e = 0; e < E; ++e) f[x][e] *= sc;
        q[0][at] = P::pack(f[x]);
        if constexpr (X::QP == 2) {
          float hi[E];
          P::unpack(q[0][at], hi);
#pragma unroll
          for (int e = 0; e < E; ++e) f[x][e] -= hi[e];
          q[1][at] = P::pack(f[x]);
        }
      }
    }
    m = -INFINITY;
    lsum = 0.f;
    whole = ROLE == BOTH && cc.c == 0;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[dt][e] = 0.f;
  };
  {
    // Loads return in order, so what the first tile needs is waited for before its
    // first chunk is asked for.
    u32x4 raw[X::KS];
    Angles ang[X::KS / 2];
    int64_t trow;
    if (sched.compact) count_group(cc.e);
    load_q(raw, trow);
    load_angles(ang, trow);
#pragma unroll
    for (int ks = 0; ks < X::KS; ++ks) settle(raw[ks]);
#pragma unroll
    for (int ks = 0; ks < X::KS / 2; ++ks)
#pragma unroll
      for (int x = 0; x < E / 4; ++x) {
        settle(ang[ks].c[x]);
        settle(ang[ks].s[x]);
      }
    issue(cc, 0);
    rotate_q(raw, ang);
  }

  for (int i = 0;; ++i) {
    TileCursor<ROLE> ic = cc;
    ic.next(sched);
    const bool more = ic.u < u_hi;
    lds_copy_wait();
    __syncthreads();  // chunk i has landed for all; the other stage is free
    if (more) issue(ic, i + 1);
    T* kt = stage_k(i);
    T* vt = kt + Sh::TILE;
    const bool pre = of_prefix(cc);
    const int r0 = (pre ? cc.c : cc.c - cc.pck) * KC;  // the chunk's first key
    const int keys = pre ? cc.s.p : cc.s.y;
    const int old = pre ? keys : cc.s.y - cc.s.n;  // keys that every row sees, but for the new
    if (r0 + KC > old) {
      // The new tokens' rows, from k_new and v_new over what the cache held there; the
      // workgroup whose row tile a token begins in writes them to the cache as well.  V
      // rows behind the last become zero: 0 x NaN must not reach a sum.
      int tid = threadIdx.x;
      asm volatile("" : "+v"(tid));  // (nothing of this block is kept across the loop)
      if (!pre) {
        constexpr int G = HALF / E;  // lanes of a row, a piece of each half a lane
        const int j0 = max(r0 - old, 0), j1 = min(r0 + KC - old, cc.s.n);
        const int64_t head = (int64_t)cc.e * a.Hkv + cc.g;
        if (tid < KC / 32) sbad[tid] = 0;
        __syncthreads();
        for (int x = tid; x < (j1 - j0) * G; x += 256) {
          const int j = j0 + x / G, d = x % G * E, lr = old + j - r0, sw = swz<X::R>(lr);
          const int64_t src = (((int64_t)cc.e * N + j) * a.Hkv + cc.g) * D;
          const int ca = ((d / E) ^ sw) * E, cb = (((d + HALF) / E) ^ sw) * E;
          const int64_t dst = (head * a.Smax + old + j) * D + d;
          P kx, vx;  // all loads first: one round trip
          float f1[E], f2[E];
          kx.load((const T*)a.k_new + src, d, HALF);
          const Angles g =
              angles(table_row(a, (int64_t)a.prefix_lens[cc.e / W] + old + j), d);
          vx.load((const T*)a.v_new + src, d, HALF);
          __builtin_amdgcn_sched_barrier(0);
          P::unpack(kx.a, f1);
          P::unpack(kx.b, f2);
          float rs = 1.f;
          if (a.k_norm_w != nullptr) {
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) ss += f1[e] * f1[e] + f2[e] * f2[e];
#pragma unroll
            for (int o = 1; o < G; o <<= 1) ss += __shfl_xor(ss, o, 64);
            rs = rsqrtf(ss / (float)D + a.norm_eps);
          }
          rotate(f1, f2, g, d, a.k_norm_w, rs);
          kx.a = P::pack(f1);
          kx.b = P::pack(f2);
          __builtin_amdgcn_sched_barrier(0);
          *(u32x4*)(kt + lr * D + ca) = kx.a;
          *(u32x4*)(kt + lr * D + cb) = kx.b;
          *(u32x4*)(vt + lr * D + ca) = vx.a;
          *(u32x4*)(vt + lr * D + cb) = vx.b;
          if (j * n_rep / ROWS == cc.t) {
            *(u32x4*)((T*)a.k_cache + dst) = kx.a;
            *(u32x4*)((T*)a.k_cache + dst + HALF) = kx.b;
            *(u32x4*)((T*)a.v_cache + dst) = vx.a;
            *(u32x4*)((T*)a.v_cache + dst + HALF) = vx.b;
          }
          __builtin_amdgcn_sched_barrier(0);
          P::unpack(vx.a, f1);
          P::unpack(vx.b, f2);
          bool fin = true;
#pragma unroll
          for (int e = 0; e < E; ++e) fin = fin && finite(f1[e]) && finite(f2[e]);
          if (!fin) atomicOr(&sbad[lr >> 5], 1u << (lr & 31));
        }
      }
      for (int x = max(keys - r0, 0) * X::R + tid; x < KC * X::R; x += 256)
        *(u32x4*)(vt + x * E) = u32x4{0u, 0u, 0u, 0u};
      __syncthreads();
    }
    const int k0 = r0 + kw * BKW;  // the wavefront's first key
    auto sees = [&](int key) -> uint32_t {  // which of 32 keys the lane's row sees
      const int lo = (pre ? keys : limit) - key;
      return lo <= 0 ? 0u : lo >= 32 ? ~0u : (1u << lo) - 1u;
    };
    auto unclean = [&](int nb) -> uint32_t {
      return __builtin_amdgcn_readfirstlane(sbad[(kw * BKW + 32 * nb) / 32]);
    };
    // The blocks of 32 keys that the wavefront's last row sees; a wavefront of which the
    // tile has no rows leaves the SIMD to the others.
    const int blocks =
        cc.t * ROWS + 32 * rw < cc.s.n * n_rep
            ? ((pre ? keys : __builtin_amdgcn_readlane(limit, 31)) - k0 + 31) >> 5
            : 0;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {  // 32 keys at a time
      if (nb >= blocks) break;
      const int row0 = kw * BKW + 32 * nb, key0 = k0 + 32 * nb;
      f32x16 s;
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = 0.f;
      X::scores(kt, row0, q, s, lane);
      bool bad = false;
      if (key0 + 32 > old) {  // (uniform)
        const uint32_t bits = sees(key0) >> (4 * h);
#pragma unroll
        for (int e = 0; e < 16; ++e)
          s[e] = (bits >> (8 * (e / 4) + e % 4)) & 1 ? s[e] : -INFINITY;
        if (ROLE != PREFIX && !pre) bad = unclean(nb) != 0;
      }
      if (ROLE != PREFIX && bad) {  // 0 x Inf must not reach the rows that do not see the key
        for (uint32_t x = unclean(nb); x; x &= x - 1) {
          const int r = row0 + __builtin_ctz(x);
          if (lane < X::R) *(u32x4*)(vt + (r * X::R + lane) * (16 / (int)sizeof(T))) = u32x4{0, 0, 0, 0};
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
      typename X::VFrag vf;
      X::load_v(vt, row0, voff, vf, lane);  // (they land under the exponentials)
      float tmax = s[0];
#pragma unroll
      for (int e = 1; e < 16; ++e) tmax = fmaxf(tmax, s[e]);
      // The exponentials are taken against a reference m that need not be the row's
      // maximum: it moves only when a score is 2^SLACK above it (or none is set
      // yet), so the sums are hardly ever rescaled.
      if (__builtin_amdgcn_ballot_w64(tmax > m + SLACK || m == -INFINITY)) {
        const float mnew = fmaxf(m, pair_max32(tmax));
        const float alpha = m == -INFINITY ? 0.f : fast_exp2(m - mnew);
        m = mnew;
        lsum *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[dt] *= alpha;
      }
      const float ref = (m == -INFINITY ? 0.f : m) - LIFT;  // (-inf: has met no key yet)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[e] = fast_exp2(s[e] - ref);
        lsum += s[e];
      }
      X::values(vt, row0, voff, s, vf, acc, lane);
      if (ROLE != PREFIX && bad) {  // those keys one by one, for the rows that see them
        const uint32_t bits = sees(key0);
        int hh = 4 * h;
        asm volatile("" : "+v"(hh));  // (as above)
        for (uint32_t x = unclean(nb); x; x &= x - 1) {
          const int kk = __builtin_ctz(x);
          float p = 0.f;
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (8 * (e / 4) + hh + e % 4 == kk) p = s[e];
          p = pair_sum32(p);
          if ((bits >> kk) & 1) {
            const T* vr = (const T*)a.v_new +
                          (((int64_t)cc.e * N + key0 + kk - old) * a.Hkv + cc.g) * D + hh;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                acc[dt][e] += p * to_f32(vr[32 * dt + 8 * (e / 4) + e % 4]);
                if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // (registers)
              }
          }
        }
      }
    }
    const bool last = cc.c == cc.nck - 1;
    const int item = (cc.e * a.Hkv + cc.g) * (ROLE == PREFIX ? ls.tiles_a : ls.tiles_b) + cc.t;
    int2* sh = (ROLE == PREFIX ? ls.sha : ls.shb) + item;
    if (threadIdx.x == 0) {
      if (cc.c == 0) sh->x = gw;
      if (last) sh->y = gw;
    }
    if (last || !more) {
      // the row tile's part of this workgroup ends: the key waves' sums joined in
      // the stage just computed, then a partial in slot gw + item
      float l = pair_sum32(lsum);
      if (l != l) m = INFINITY;  // (a NaN must not be left out for its weight)
      // The key waves share the join out by blocks of 32 dims: block dt is wave
      // owner(dt)'s, the others leave theirs in LDS.
      auto owner = [](int dt) { return dt * KW / DT; };
      if constexpr (KW > 1) {
        __syncthreads();  // all wavefronts are done with the stage
        float* xo = (float*)kt;                    // [KW - 1][ROWS][D]
        float* xm = (float*)(lds + 2 * Sh::STAGE);  // [KW][ROWS][2]
        const int r = 32 * rw + l31;
        // place of a piece of wave j's block dt (a lane's pieces rotated by its row: the
        // rows lie D floats apart)
        auto piece = [&](int j, int dt, int e) {
          const int slot = j < owner(dt) ? j : j - 1;
          return (f32x4*)(xo + (slot * ROWS + r) * D + 4 * h +
                          (((8 * dt + 2 * (e / 4)) ^ (2 * (r & 3))) * 4));
        };
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
          if (owner(dt) != kw)
#pragma unroll
            for (int e = 0; e < 16; e += 4)
              *piece(kw, dt, e) = f32x4{acc[dt][e], acc[dt][e + 1], acc[dt][e + 2], acc[dt][e + 3]};
        if (h == 0) *(float2*)(xm + (kw * ROWS + r) * 2) = make_float2(m, l);
        __syncthreads();
        float2 ml[KW];
        float mj = -INFINITY;
#pragma unroll
        for (int j = 0; j < KW; ++j) {
          ml[j] = *(const float2*)(xm + (j * ROWS + r) * 2);
          mj = fmaxf(mj, ml[j].x);
        }
        const float rj = mj == -INFINITY ? 0.f : mj;
        const float own = fast_exp2(m - rj);
        m = mj;
        l = 0.f;
#pragma unroll
        for (int j = 0; j < KW; ++j) {
          ml[j].x = fast_exp2(ml[j].x - rj);
          l += ml[j].y * ml[j].x;
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
          if (owner(dt) == kw) {
            acc[dt] *= own;
#pragma unroll
            for (int j = 0; j < KW; ++j)
              if (j != owner(dt))
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                  const f32x4 y = *piece(j, dt, e);
#pragma unroll
                  for (int x = 0; x < 4; ++x) acc[dt][e + x] += y[x] * ml[j].x;
                }
          }
      }
      const int r = cc.t * ROWS + 32 * rw + l31;
      if (r < cc.s.n * n_rep) {
        if (whole && last) {
          const float inv = 1.f / l;
          T* o = (T*)a.out +
                 (((int64_t)cc.e * N + r / n_rep) * a.Hq + cc.g * n_rep + r % n_rep) * D + 4 * h;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int e = 0; e < 16 && owner(dt) == kw; e += 4) {
              T y[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) y[j] = from_f32<T>(acc[dt][e + j] * inv);
              __builtin_memcpy(__builtin_assume_aligned(o + 32 * dt + 2 * e, 4 * sizeof(T)), y,
                               sizeof(y));
            }
        } else {
          const int64_t at = ((int64_t)gw + item) * ROWS + 32 * rw + l31;
          float* o = (ROLE == PREFIX ? ls.oa : ls.ob) + at * D + 4 * h;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int e = 0; e < 16 && owner(dt) == kw; e += 4)
              *(f32x4*)(o + 32 * dt + 2 * e) =
                  f32x4{acc[dt][e], acc[dt][e + 1], acc[dt][e + 2], acc[dt][e + 3]};
          if (h == 0 && kw == 0)
            *(float2*)((ROLE == PREFIX ? ls.mla : ls.mlb) + at * 2) = make_float2(m, l);
        }
      }
    }
    if (!more) break;
    const bool new_group = ic.e != cc.e;
    cc = ic;
    if (cc.c == 0) {
      u32x4 raw[X::KS];
      Angles ang[X::KS / 2];
      int64_t trow;
      if (sched.compact && new_group) count_group(cc.e);
      load_q(raw, trow);
      load_angles(ang, trow);
      rotate_q(raw, ang);
    }
  }
}

// Row waves of the prefixes' and the own rows' tiles (0: one wavefront a share; prefixes -1:
// one list of the sequences over both).
template <typename T>
constexpr int bkw_of(int rw) {
  return rw == 4 && sizeof(T) == 2 ? 64 : 32;
}
template <typename T, int D, int RWA, int RWB>
struct Variant {
  static constexpr int RW = RWA > 0 ? RWA : RWB > 0 ? RWB : 4;
  using Sh = Shape<T, D, RW, bkw_of<T>(RW)>;
  static constexpr size_t LDS =
      RWA == 0  ? 4 * sizeof(WaveLds<T, D>)
      : RWA < 0 ? Sh::LDS
                : (Sh::LDS > 4 * sizeof(WaveLds<T, D>) ? Sh::LDS : 4 * sizeof(WaveLds<T, D>));
  static constexpr int PER_CU = sizeof(T) == 2 || D == 64 || RWA == 0 ? 2 : 1;
};

template <typename T, int D, int RWA, int RWB>
__global__ __launch_bounds__(256, (Variant<T, D, RWA, RWB>::PER_CU)) void branch_stream_kernel(
    BranchArgs a, Lists ls) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63, grid = gridDim.x, blk = blockIdx.x;
  if constexpr (RWA == 0) {  // one list for both
    const WaveSched<true, WK<T>> sched(a, lane);
    wave_role<T, D, true>(a, ls, lds, sched, blk * 4 + mfma::wave_id(), min(4 * grid, sched.C));
  } else if constexpr (RWA < 0) {
    constexpr int BKW = bkw_of<T>(RWB);
    using Sh = Shape<T, D, RWB, BKW>;
    __shared__ uint32_t sbad[Sh::KC / 32];
    TileSched<BOTH> s(a, Sh::ROWS, Sh::KC, false, lane);
    if (s.C >= 4 * grid) s.count_beginnings();
    tile_role<T, D, RWB, BKW, BOTH>(a, ls, lds, nullptr, sbad, s, blk, grid);
  } else {
    constexpr int BKW = bkw_of<T>(RWA);
    using Sh = Shape<T, D, RWA, BKW>;
    __shared__ int pre[MAX_COMPACT];
    __shared__ uint32_t sbad[Sh::KC / 32];
    TileSched<PREFIX> sa(a, Sh::ROWS, Sh::KC, ls.compact, lane);
    // The workgroups are shared out by the bytes of the two lists.
    auto split = [&](int most_b, float cost_b) {
      if (sa.C == 0 || most_b == 0) return sa.C == 0 ? 0 : grid;
      if (sa.C + most_b <= grid) return sa.C;
      const int n = (int)((float)grid * (float)sa.C / ((float)sa.C + cost_b) + 1.f);
      return min(max(n, 1), grid - 1);
    };
    if constexpr (RWB == 0) {
      const WaveSched<false, WK<T>> sb(a, lane);
      if (sa.C + sb.C >= 4 * grid) sa.count_beginnings();
      const int na = split((sb.C + 3) / 4, (float)sb.C * WK<T> / Sh::KC);
      if (blk < na)
        tile_role<T, D, RWA, BKW, PREFIX>(a, ls, lds, pre, sbad, sa, blk, na);
      else
        wave_role<T, D, false>(a, ls, lds, sb, (blk - na) * 4 + mfma::wave_id(),
                               min(4 * (grid - na), sb.C));
    } else {
      TileSched<OWN> sb(a, Sh::ROWS, Sh::KC, false, lane);
      if (sa.C + sb.C >= 4 * grid) {
        sa.count_beginnings();
        sb.count_beginnings();
      }
      const int na = split(sb.C, (float)sb.C);
      if (blk < na)
        tile_role<T, D, RWA, BKW, PREFIX>(a, ls, lds, pre, sbad, sa, blk, na);
      else
        tile_role<T, D, RWA, BKW, OWN>(a, ls, lds, pre, sbad, sb, blk - na, grid - na);
    }
  }
}

// The rows of a pair (sequence, KV head), 16 bytes of a row per thread and RPW rows a
// workgroup (pairs first: one dimension, as both may be many): the partials of the prefix's
// and the own rows' workers, rescaled to a common maximum and summed.  JG groups of threads
// take a row's partials in turn, U at a time, and are joined through LDS.  Bound by the round
// trips to what other compute units wrote: 4 us of some 5 for a few rows.
template <typename T, int D, int JG>
__global__ __launch_bounds__(256) void branch_merge_kernel(BranchArgs a, Lists ls) {
  constexpr int LPR = D / 4, RPW = 256 / (LPR * JG);  // lanes of a row, rows of a workgroup
  __shared__ f32x4 xo[JG > 1 ? 256 : 1];
  __shared__ float2 xm[JG > 1 ? 256 : 1];
  __shared__ int before;
  const int n_rep = a.Hq / a.Hkv, W = a.B / a.G;
  const int pairs = a.B * a.Hkv, pair = blockIdx.x % pairs;
  const int b = pair / a.Hkv, g = pair % a.Hkv, grp = b / W;
  const int r = blockIdx.x / pairs * RPW + threadIdx.x / (LPR * JG), jg = threadIdx.x / LPR % JG;
  const int col = threadIdx.x % LPR * 4, i = r / n_rep;
  const bool inside = i < a.N;
  int first = (b % W) * a.N;  // the sequence's first token in its group's rows
  if (ls.compact) {
    if (threadIdx.x == 0) before = 0;
    __syncthreads();
    int n = 0;
    for (int x = threadIdx.x; x < b % W; x += 256) n += min(max(a.counts[grp * W + x], 0), a.N);
    if (n) atomicAdd(&before, n);
    __syncthreads();
    first = before;
  }
  // (what the row is made of is asked for beside what says whether it is one)
  const int rr = inside ? r : 0, ra = (first + rr / n_rep) * n_rep + rr % n_rep;
  const int ia = (grp * a.Hkv + g) * ls.tiles_a + ra / max(ls.rows_a, 1);
  const int ib = (b * a.Hkv + g) * ls.tiles_b + rr / ls.rows_b;
  const int2 sha = ls.tiles_a > 0 ? ls.sha[ia] : int2{0, -1}, shb = ls.shb[ib];
  const Seq s = branch_seq(a, b);
  T* dst = (T*)a.out + (((int64_t)b * a.N + i) * a.Hq + g * n_rep + r % n_rep) * D + col;
  T y[4];
  if (inside && jg == 0 && i >= s.n) {  // a refused sequence, or an unused token
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = from_f32<T>(s.n < 0 ? NAN : 0.f);
    __builtin_memcpy(__builtin_assume_aligned(dst, 4 * sizeof(T)), y, sizeof(y));
  }
  bool live = inside && i < s.n;
  int na = 0, nb = 0;
  int64_t at = 0, bt = 0;
  if (live) {
    if (s.P > 0 && ls.tiles_a > 0) {
      na = sha.y - sha.x + 1;
      at = ((int64_t)sha.x + ia) * ls.rows_a + ra % ls.rows_a;
    }
    nb = shb.y - shb.x + 1;
    bt = ((int64_t)shb.x + ib + ls.item_b) * ls.rows_b + rr % ls.rows_b;
  }
  const int ns = na + nb;
  // (one list for both and one worker: it wrote the outputs)
  if (ls.tiles_a == 0 && ns == 1) live = false;
  float M = -INFINITY, l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  // joins a partial (of weight 0: left out, whatever it holds)
  auto add = [&](float f, const float2& ml, const f32x4& po) {
    const float w = fast_exp2(ml.x - M);
    l = l * f + (w != 0.f ? w * ml.y : 0.f);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = o[e] * f + (w != 0.f ? w * po[e] : 0.f);
  };
  constexpr int U = JG == 1 ? 4 : 8;  // (few partials a row: no loads of the same again)
  for (int j0 = jg; live && j0 < ns; j0 += U * JG) {
    f32x4 po[U];
    float2 ml[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = min(j0 + u * JG, ns - 1);
      const bool pre = j < na;
      const int64_t x = pre ? at + (int64_t)j * ls.rows_a : bt + (int64_t)(j - na) * ls.rows_b;
      ml[u] = *(const float2*)((pre ? ls.mla : ls.mlb) + x * 2);
      po[u] = *(const f32x4*)((pre ? ls.oa : ls.ob) + x * D + col);
    }
    float mx = M;
#pragma unroll
    for (int u = 0; u < U; ++u) mx = fmaxf(mx, ml[u].x);
    // (a chunk's scores can all be -inf: such a partial has no weight)
    float f = M == -INFINITY ? 0.f : fast_exp2(M - mx);
    M = mx;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (j0 + u * JG < ns && ml[u].x != -INFINITY) add(f, ml[u], po[u]), f = 1.f;
    }
    if (f != 1.f) l *= f, o *= f;
  }
  if constexpr (JG > 1) {
    xo[threadIdx.x] = o;
    xm[threadIdx.x] = make_float2(M, l);
    __syncthreads();
    if (live && jg == 0) {
      float mx = M;
#pragma unroll
      for (int j = 1; j < JG; ++j) mx = fmaxf(mx, xm[threadIdx.x + j * LPR].x);
      float f = M == -INFINITY ? 0.f : fast_exp2(M - mx);
      M = mx;
      l *= f;
      o *= f;
#pragma unroll
      for (int j = 1; j < JG; ++j) {
        const float2 ml = xm[threadIdx.x + j * LPR];
        if (ml.x != -INFINITY) add(1.f, ml, xo[threadIdx.x + j * LPR]);
      }
    }
  }
  if (!live || jg != 0) return;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = from_f32<T>(o[e] / l);
  __builtin_memcpy(__builtin_assume_aligned(dst, 4 * sizeof(T)), y, sizeof(y));
}

// ---- host ----------------------------------------------------------------------
size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

// The stream kernel's shape for a call: row waves of the prefixes' tiles and of the own
// rows' (0: one wavefront a share), or (none) one wavefront a row.  All times in us, 32 / 8
// heads of 128 in bfloat16 if nothing else is said:
//  - Up to 16 rows of a pair: a wavefront a share.  Its list has four times as many shares,
//    so a wavefront has little to read before the merge: 4 beams behind 1000 keys 13.8, in
//    tiles 15.2; 8 x 4 behind 4096 in float32 72, 114 (a tile of 64 rows is mostly padding,
//    and float32's products are slow).  4 x 4 behind 8192 in bfloat16 44, 40.  Beyond 16 rows
//    a second block of rows a wavefront needs its registers: 16 beams 21, tiles 17.5.
//  - Tiles of 64 rows up to 64 rows, of 128 beyond: 4 x 12 behind 8192 in float32 138, 203;
//    in bfloat16, bound by the keys' bytes, they are level (12 behind 4096: 22).  Beyond 64
//    rows 128 read the keys half as often: 4 x 16 of 64 / 8 heads behind 8192 75, 78.
//  - Sequences with over 16 rows of their own: one list of their tiles over prefix and cache
//    (fewer partials to join, none where a tile is one workgroup's), or a list of the group's
//    tiles over the prefix (whole tiles) beside one of theirs over their own keys.  8 x 16
//    tokens behind 512 keys and 512 of their own: 28, 34; behind 4096: 48, 40.  4 x 4 x 24
//    behind 1024 in float32: 108, 88.  So the first where it is no more than a fifth more
//    chunks of 128 rows.
struct Plan {
  bool none;
  int rwa, rwb, rows_a, rows_b, tiles_a, tiles_b, grid, workers_a, workers_b;
};
Plan plan_of(const BranchArgs& a) {
  Plan p = {};
  p.none = true;
  const int n_rep = a.Hq / a.Hkv, W = a.B / a.G;
  if (a.D != 64 && a.D != 128) return p;
  const int64_t ma = (int64_t)W * a.N * n_rep, mb = (int64_t)a.N * n_rep;
  const int rw = ma <= 64 ? 2 : 4;
  const int kc = rw == 4 && a.dtype == F32 ? 32 : 64;
  auto tiles = [&](int64_t m, int rows) { return (m + rows - 1) / rows; };
  auto chunks = [&](int n, int keys) { return ((int64_t)n + keys - 1) / keys; };
  const int64_t pt = chunks(a.max_prefix, kc), ot = chunks(a.max_len, kc);
  const int64_t na = a.G * tiles(ma, 128), nb = a.B * tiles(mb, 128);
  const bool both = rw == 4 && mb > 16 &&
                    nb * (pt + ot + OVER) * 5 <= (na * (pt + OVER) + nb * (ot + OVER)) * 6;
  p.rwa = both ? -1 : ma <= 16 ? 0 : rw;
  p.rwb = mb <= 16 ? 0 : rw;
  p.rows_a = both ? 0 : p.rwa ? 32 * rw : (int)ma;
  p.rows_b = p.rwb ? 32 * rw : p.rwa ? (int)mb : (int)ma;  // (one list: one kind of slot)
  const int64_t ta = both ? 0 : tiles(ma, p.rows_a), tb = tiles(mb, p.rows_b);
  const int wk = a.dtype == F32 ? WK<float> : WK<bf16>;
  const int ka = p.rwa ? kc : wk, kb = p.rwb ? kc : wk;
  const int64_t pk = chunks(a.max_prefix, ka), ca = a.G * ta * a.Hkv * (pk + OVER),
                cb = a.B * tb * a.Hkv *
                     (chunks(a.max_len, kb) + (both ? pk : 0) + (p.rwb ? OVER : 1));
  // (the merge launches 256 threads a pair and more: fewer than 2^32)
  if (ca + cb >= INT_MAX || (a.G * ta + a.B * tb) * a.Hkv >= 1 << 24) return p;
  p.tiles_a = (int)ta;
  p.tiles_b = (int)tb;
  const int per_cu = a.dtype != F32 || a.D == 64 || p.rwa == 0 ? 2 : 1;  // Variant::PER_CU
  // (no more workgroups than chunks, each list having one at least)
  const int64_t wgs = (p.rwa ? ca : (ca + 3) / 4) + (p.rwb ? cb : (cb + 3) / 4);
  p.grid = (int)std::min<int64_t>(per_cu * std::min(device_cu_count(), 512), wgs);
  p.none = false;
  return p;
}

// workspace: the partials and the first and last worker of each item; or, one wavefront a
// row, the rotated queries
struct Ws {
  Lists ls;
  float* qrot;
  size_t bytes;
};
Ws carve(const BranchArgs& a, const Plan& p, void* at) {
  char* c = (char*)at;
  Ws w = {};
  if (p.none) {
    w.qrot = (float*)c;
    w.bytes = up256((size_t)a.B * a.N * a.Hq * a.D * 4);
    return w;
  }
  auto take = [&](size_t n) {
    void* x = c;
    c += up256(n);
    return x;
  };
  const size_t ia = (size_t)a.G * a.Hkv * p.tiles_a, ib = (size_t)a.B * a.Hkv * p.tiles_b;
  Lists& ls = w.ls;
  ls.rows_a = p.rows_a;
  ls.rows_b = p.rows_b;
  ls.tiles_a = p.tiles_a;
  ls.tiles_b = p.tiles_b;
  ls.item_b = p.rwa ? 0 : (int)ia;
  ls.compact = p.rwa > 0 && a.counts != nullptr && a.B / a.G <= MAX_COMPACT;
  ls.sha = (int2*)take(ia * sizeof(int2));
  ls.shb = (int2*)take(ib * sizeof(int2));
  const size_t slots = ((size_t)(p.rwb ? p.grid : 4 * p.grid) + ls.item_b + ib) * p.rows_b;
  ls.ob = (float*)take(slots * a.D * 4);
  ls.mlb = (float*)take(slots * 8);
  ls.oa = ls.ob;
  ls.mla = ls.mlb;
  if (p.rwa > 0) {
    const size_t more = ((size_t)p.grid + ia) * p.rows_a;
    ls.oa = (float*)take(more * a.D * 4);
    ls.mla = (float*)take(more * 8);
  }
  w.bytes = (size_t)(c - (char*)at);
  return w;
}

template <typename T, int D, int RWA, int RWB>
int launch_stream(const BranchArgs& a, const Ws& w, const Plan& p) {
  constexpr size_t LDS = Variant<T, D, RWA, RWB>::LDS;
  auto kernel = branch_stream_kernel<T, D, RWA, RWB>;
  if (LDS + MAX_COMPACT * 4 + 1024 > 64 * 1024) {  // asked for once per device
    static std::atomic<uint64_t> done{0};
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    const uint64_t bit = dev >= 0 && dev < 64 ? 1ull << dev : 0;
    if (e == hipSuccess && !(done.load(std::memory_order_relaxed) & bit)) {
      e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize,
                              (int)LDS);
      if (e == hipSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    }
    if (e != hipSuccess) {
      set_error("branch attention: %s", hipGetErrorString(e));
      return KF_ERR_HIP;
    }
  }
  KF_LAUNCH("branch_stream", kernel, dim3(p.grid), dim3(256), LDS, a.stream, a, w.ls);
  KF_CHECK_LAUNCH();
  return KF_OK;
}

template <typename T, int D>
int stream_and_merge(const BranchArgs& a, const Ws& w, const Plan& p) {
  int rc;
  if (p.rwa < 0)
    rc = launch_stream<T, D, -1, 4>(a, w, p);
  else if (p.rwa == 0)
    rc = launch_stream<T, D, 0, 0>(a, w, p);
  else if (p.rwb == 0)
    rc = p.rwa == 2 ? launch_stream<T, D, 2, 0>(a, w, p) : launch_stream<T, D, 4, 0>(a, w, p);
  else
    rc = p.rwa == 2 ? launch_stream<T, D, 2, 2>(a, w, p) : launch_stream<T, D, 4, 4>(a, w, p);
  if (rc) return rc;
  // The more partials a row has, the more threads take them.  Calls by 1, 2 and 8, in us: 64
  // shares an item 18.6, 15.7, 13.8 (4 beams behind 1000 keys); 32 28.4, 26.5, 26.6 (8 x 4
  // behind 1000); 16 64.0, 65.6, 75.0 (4 x 16 behind 8192); 1 145, 161, 227 (questions).
  const int64_t items = (p.rwa < 0 ? (int64_t)a.B * p.tiles_b : (int64_t)a.G * p.tiles_a) * a.Hkv;
  const int64_t workers = p.rwa ? p.grid : 4 * p.grid;
  const int jg = workers > 32 * items ? 8 : workers > 16 * items ? 2 : 1;
  const int rpw = 256 / (D / 4) / jg;  // rows of a workgroup
  KF_LAUNCH("branch_merge",
            (jg == 8   ? branch_merge_kernel<T, D, 8>
             : jg == 2 ? branch_merge_kernel<T, D, 2>
                       : branch_merge_kernel<T, D, 1>),
            dim3(a.B * a.Hkv * ((a.N * (a.Hq / a.Hkv) + rpw - 1) / rpw)), dim3(256), 0, a.stream,
            a, w.ls);
  KF_CHECK_LAUNCH();
  return KF_OK;
}

template <typename T>
int branch_typed(const BranchArgs& a, void* workspace) {
  Plan p = plan_of(a);
  // (direct loads to LDS and 16-byte rows need aligned buffers)
  if (((uintptr_t)a.q_new | (uintptr_t)a.k_new | (uintptr_t)a.v_new | (uintptr_t)a.k_cache |
       (uintptr_t)a.v_cache | (uintptr_t)a.k_prefix | (uintptr_t)a.v_prefix | (uintptr_t)a.out |
       (uintptr_t)a.cos | (uintptr_t)a.sin) % 16 != 0)
    p.none = true;
  const Ws w = carve(a, p, workspace);
  if (!p.none)
    return a.D == 128 ? stream_and_merge<T, 128>(a, w, p) : stream_and_merge<T, 64>(a, w, p);
  const int per = 16;
  const int64_t rows = (int64_t)a.N * (a.Hq + 2 * a.Hkv);
  KF_LAUNCH("branch_prep", branch_prep_kernel<T>, dim3((unsigned)((rows + per - 1) / per), a.B),
            dim3(256), 0, a.stream, a, w.qrot, per);
  KF_CHECK_LAUNCH();
  KF_LAUNCH("branch_rows", branch_rows_kernel<T>,
            dim3((unsigned)(((int64_t)a.B * a.N * a.Hq + 3) / 4)), dim3(256), 0, a.stream, a,
            w.qrot);
  KF_CHECK_LAUNCH();
  return KF_OK;
}

}  // namespace

size_t branch_workspace(const BranchArgs& a) {
  // (which of the two a call takes goes by its buffers' alignment too)
  Plan none = {};
  none.none = true;
  return std::max(carve(a, plan_of(a), nullptr).bytes, carve(a, none, nullptr).bytes);
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
