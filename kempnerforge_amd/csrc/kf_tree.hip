// Attention of a tree of drafted tokens over a KV cache.
//
// Node i of sequence b sees the cached prefix (keys 0 .. lens[b] - 1), itself and
// its ancestors in the tree:
//   s_ij = q_i . k_j / sqrt(D),  j in prefix or anc(i);  o_i = softmax(s_i) V
// Its key is rotated at position lens[b] + depth(i) and stored in cache row
// lens[b] + i, so that the rows of all nodes lie behind the prefix in node order
// and are read like it, under a mask.
//
//  1. stream  split-K attention on the matrix cores: a workgroup takes up to 128
//             (node, query head) rows of a KV head and an equal share of all key
//             chunks; it rotates its queries into registers, and the nodes' keys
//             and values where its chunks hold them (the first row tile's
//             workgroups write them to the caches); a row tile that more than one
//             workgroup met leaves float32 partials
//  2. merge   joins the partials; rows of unused nodes and refused sequences
// Other head sizes and misaligned buffers: prep (rotated queries, ancestor masks,
// the nodes' cache rows), then one wavefront per row (rows).
//
// Rounding: the norm and the rotation of q and k are formed in 32 bits.  k is
// rounded once, where it is stored.  What goes through the 16-bit matrix
// instructions is not rounded to 16 bits: q and P enter as sums of two numbers of the
// input type (hi = x rounded, lo = x - hi rounded: 16 bits in bfloat16, 22 in float16),
// for twice the products; the sums, the row maxima and the row sums stay in 32 bits.
// Against 64 bits that leaves the error of rounding the outputs and no more.  With P
// alone rounded to the type it would be 1.2 to 1.4 times (and 220 us instead of 266
// below), with q too 1.7 times (and 163 us).
//
// What bounds it, in bfloat16 with heads of 128: the matrix instructions for wide
// trees (4 sequences, 64 nodes, 16384 keys, 64 / 8 heads: 266 us, 1030 TFLOP/s with
// the lo products), HBM for narrow ones (32 sequences of up to 8192 keys, 16 nodes,
// 32 / 8 heads: 133 to 141 us, 5.0 to 5.3 TB/s), dependent loads for single ones (5
// nodes, 1000 keys: 13.7 us in two launches; a launch for the rotation in front costs
// 2.8 more).
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

constexpr int MAXN = KF_TREE_MAX_NODES;
constexpr int MAXW = MAXN / 32;  // 32-bit words of an ancestor mask

// A sequence's nodes in use and prefix length; -1 nodes where they are out of range.
__device__ __forceinline__ int2 tree_seq(const TreeArgs& a, int b) {
  const int n = a.counts ? a.counts[b] : a.N, L = a.lens[b];
  const bool ok = n >= 0 && n <= a.N && L >= 0 && (int64_t)L + n <= a.max_len;
  return ok ? make_int2(n, L) : make_int2(-1, 0);
}

// One sequence's tree in LDS: each node's ancestors (itself among them) as bits,
// and its depth.
struct TreeLds {
  uint32_t mask[MAXN][MAXW + 1];
  int ptr[MAXN], depth[MAXN];
};

// Forms the tree of a sequence (s: its nodes and prefix; par: the parent of the node that
// tree_parent gives the thread), by a workgroup of 256; returns whether the sequence is
// refused.  A chain needs no LDS: node i sees
// nodes 0 .. i and lies at depth i.
//
// The masks come from pointer doubling: after round r, mask[i] holds the 2^r
// nearest of i and its ancestors and ptr[i] the next one beyond, so 8 rounds
// cover 256 nodes whatever their depth (a walk up a chain of 200 would take 200
// dependent reads).  Up to 64 nodes every wavefront forms them all by itself, a lane a
// node, by shuffles and as many rounds as the depth needs (27 nodes: 1.3 us where the rounds
// with barriers take 2.7).
__device__ __forceinline__ int tree_parent(const TreeArgs& a, int b, int2 s) {
  const int t = a.N <= 64 ? threadIdx.x & 63 : threadIdx.x;
  return a.parents != nullptr && t < s.x ? a.parents[(int64_t)b * a.parents_stride + t] : -1;
}
__device__ __forceinline__ bool tree_build(const TreeArgs& a, int2 s, int W, TreeLds& lds,
                                           int par) {
  const int64_t low = (int64_t)s.y - a.rope_row_offset;  // table row of depth 0
  if (a.parents == nullptr)
    return s.x < 0 || (s.x > 0 && (low < 0 || low + s.x > a.rope_rows));
  const int t = threadIdx.x, used = max(s.x, 0);
  bool bad = s.x < 0;
  if (a.N <= 64) {
    const int lane = t & 63;
    if (par < -1 || par >= lane) {
      bad = true;
      par = -1;
    }
    uint32_t lo = lane < 32 ? 1u << lane : 0u, hi = lane < 32 ? 0u : 1u << (lane - 32);
    while (__builtin_amdgcn_ballot_w64(par >= 0)) {  // (parents come first: it ends)
      const int from = max(par, 0), next = __shfl(par, from, 64);
      const uint32_t l = __shfl(lo, from, 64), h = __shfl(hi, from, 64);
      if (par >= 0) {
        lo |= l;
        hi |= h;
        par = next;
      }
    }
    const int depth = __popc(lo) + __popc(hi) - 1;
    bad |= lane < used && (low + depth < 0 || low + depth >= a.rope_rows);
    __syncthreads();  // the previous tree's readers are done
    if (t < 64) {
      lds.mask[t][0] = lo;
      lds.mask[t][1] = hi;
      lds.depth[t] = depth;
    }
    __syncthreads();
    return __builtin_amdgcn_ballot_w64(bad) != 0;
  }
  if (par < -1 || par >= t) {
    bad = true;
    par = -1;
  }
  __syncthreads();  // the previous tree's readers are done
  for (int k = 0; k < W; ++k) lds.mask[t][k] = k == t >> 5 ? 1u << (t & 31) : 0u;
  lds.ptr[t] = par;
  __syncthreads();
  for (int span = 1; span < used; span <<= 1) {
    const int p = lds.ptr[t];
    uint32_t m[MAXW];
    int next = -1;
    if (p >= 0) {
#pragma unroll
      for (int k = 0; k < MAXW; ++k) m[k] = k < W ? lds.mask[p][k] : 0u;
      next = lds.ptr[p];
    }
    __syncthreads();
    if (p >= 0) {
#pragma unroll
      for (int k = 0; k < MAXW; ++k)
        if (k < W) lds.mask[t][k] |= m[k];
      lds.ptr[t] = next;
    }
    __syncthreads();
  }
  int depth = -1;
  for (int k = 0; k < W; ++k) depth += __popc(lds.mask[t][k]);
  lds.depth[t] = depth;
  if (t < used && (low + depth < 0 || low + depth >= a.rope_rows)) bad = true;
  return __syncthreads_or(bad);
}

// One workgroup: sequence blockIdx.y, `per` of its N * (Hq + 2 Hkv) rows, a
// wavefront a row.  The queries go to `qrot`, float32 [B][Hkv][node, head of the
// group][D], scaled by D^-1/2 log2(e).  Every workgroup of a sequence forms its tree
// (under a microsecond); the first one stores the masks.
template <typename T>
__global__ __launch_bounds__(256) void tree_prep_kernel(TreeArgs a, float* __restrict__ qrot,
                                                        uint32_t* __restrict__ anc,
                                                        int2* __restrict__ seq, int W, int per) {
  __shared__ TreeLds tree;
  const int b = blockIdx.y, t = threadIdx.x, lane = t & 63, w = t >> 6;
  const int N = a.N, D = a.D, half = D / 2;
  const int heads = a.Hq + 2 * a.Hkv, n_rep = a.Hq / a.Hkv;
  const int2 s = tree_seq(a, b);
  const bool bad = tree_build(a, s, W, tree, tree_parent(a, b, s));
  const int n = s.x, L = s.y;
  if (blockIdx.x == 0) {
    if (t == 0) seq[b] = bad ? make_int2(-1, 0) : s;
    if (t < N)
      for (int k = 0; k < W; ++k) {
        const int lo = t + 1 - 32 * k;  // (chain: nodes 0 .. t)
        anc[((int64_t)b * N + t) * W + k] = a.parents != nullptr ? tree.mask[t][k]
                                            : lo <= 0              ? 0u
                                            : lo >= 32             ? ~0u
                                                                   : (1u << lo) - 1u;
      }
  }
  if (bad) return;
  const int64_t r1 = min((int64_t)n * heads, (int64_t)(blockIdx.x + 1) * per);
  for (int64_t r = (int64_t)blockIdx.x * per + w; r < r1; r += 4) {
    const int i = (int)(r / heads), h = (int)(r % heads);
    const int64_t node = (int64_t)b * N + i;
    if (h >= a.Hq + a.Hkv) {
      const int g = h - a.Hq - a.Hkv;
      const T* src = (const T*)a.v_new + (node * a.Hkv + g) * D;
      T* dst = (T*)a.v_cache + (((int64_t)b * a.Hkv + g) * a.Smax + L + i) * D;
      for (int d = lane; d < D; d += 64) dst[d] = src[d];
      continue;
    }
    const bool is_q = h < a.Hq;
    const int g = is_q ? h / n_rep : h - a.Hq;
    const T* src = is_q ? (const T*)a.q_new + (node * a.Hq + h) * D
                        : (const T*)a.k_new + (node * a.Hkv + g) * D;
    const int64_t qrow =
        (((int64_t)b * a.Hkv + g) * N * n_rep + (int64_t)i * n_rep + h % n_rep) * D;
    T* kdst = (T*)a.k_cache + (((int64_t)b * a.Hkv + g) * a.Smax + L + i) * D;
    const float* nw = is_q ? a.q_norm_w : a.k_norm_w;
    float rs = 1.f;
    if (nw != nullptr) {
      float ss = 0.f;
      for (int d = lane; d < D; d += 64) ss += to_f32(src[d]) * to_f32(src[d]);
      rs = rsqrtf(wave_sum(ss) / (float)D + a.norm_eps);
    }
    const int depth = a.parents != nullptr ? tree.depth[i] : i;
    const int64_t row = ((int64_t)L + depth - a.rope_row_offset) * half;
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
          qrot[qrow + at] = y[e] * (a.scale * kLog2e);
        else
          kdst[at] = from_f32<T>(y[e]);
      }
    }
  }
}

// One wavefront per (b, node, query head), any D <= 256: the prefix and the
// node's own row and ancestors, one key at a time.  Masked keys are not read.  Bound by
// a key's chain of load, sum over the wavefront and exponential, 0.7 us each (heads of 96:
// 5 nodes over 1000 keys 722 us, 8 sequences of 16 nodes over 4096 keys 4.9 ms).
template <typename T>
__global__ __launch_bounds__(256) void tree_rows_kernel(TreeArgs a, const float* __restrict__ qrot,
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
  const float* q = qrot + (((int64_t)b * a.Hkv + g) * a.N * n_rep + (int64_t)i * n_rep + hq % n_rep) * D;
  const T* kb = (const T*)a.k_cache + ((int64_t)b * a.Hkv + g) * a.Smax * D;
  const T* vb = (const T*)a.v_cache + ((int64_t)b * a.Hkv + g) * a.Smax * D;
  float qv[4], acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int e = 0; e < 4; ++e) qv[e] = lane + 64 * e < D ? q[lane + 64 * e] : 0.f;
  float m = -INFINITY, l = 0.f;
  auto key = [&](int j) {
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
  };
  for (int j = 0; j < L; ++j) key(j);
  const uint32_t* words = anc + ((int64_t)b * a.N + i) * W;
  for (int k = 0; k < W; ++k)
    for (uint32_t bits = words[k]; bits; bits &= bits - 1) key(L + 32 * k + __builtin_ctz(bits));
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (lane + 64 * e < D) out[lane + 64 * e] = from_f32<T>(acc[e] / l);
}

// ---- split-K attention on the matrix cores -------------------------------------
// Row tile t of pair (b, g) holds rows t ROWS .. of the pair's n_b n_rep rows
// (node-major: the heads of a node side by side); every tile meets the nck(b) =
// ceil((lens[b] + n_b) / KC) key chunks of its pair.
//
// Beginning a row tile costs about as much as OVER chunks (its queries are loaded
// and rotated, the tree formed), so with several chunks per workgroup each tile
// has `over` units in front of its chunks in the list that is shared out: OVER, or
// one where that spares the largest share a unit (8 x 8 heads, 4000 keys, 80 rows: 8
// units for 9, 43.3 -> 40.6 us; 4 x 8 heads, 1224 keys, 800 rows, 11 units with two or
// one: 61 and 64).
struct TreeSched {
  const TreeArgs& a;
  int n_rep, rows, kc;
  int over, C, NW;  // units of the list, workgroups that share it
  static constexpr int OVER = 2;
  int B;
  int2 own{-1, 0};  // sequence `lane`'s tree_seq, all there are up to 64 of them
  __device__ __forceinline__ TreeSched(const TreeArgs& a_, int n_rep_, int rows_, int kc_,
                                       int grid, int lane)
      : a(a_), n_rep(n_rep_), rows(rows_), kc(kc_), B(a_.B) {
    int tot = 0, items = 0;
    for (int b = lane; b < B; b += 64) {
      const int2 s = tree_seq(a, b);
      const int i = s.x > 0 ? a.Hkv * tiles(s) : 0;
      items += i;
      tot += i > 0 ? i * nck(s) : 0;
      own = s;
    }
    tot = __builtin_amdgcn_readlane(wave_prefix(tot), 63);
    items = __builtin_amdgcn_readlane(wave_prefix(items), 63);
    over = tot >= 4 * grid ? OVER : 0;
    const unsigned n = grid, chunks = tot, one = (chunks + items + n - 1) / n,
                   two = (chunks + OVER * items + n - 1) / n;
    if (over && one < two) over = 1;
    C = tot + over * items;
    NW = min(grid, C);
  }
  // the first unit of workgroup w's share, floor(w C / NW) (w and NW are far below 2^16)
  __device__ __forceinline__ int start(int w) const {
    const unsigned n = max(NW, 1), q = (unsigned)C / n, r = (unsigned)C % n;
    return (int)(w * q + (unsigned)w * r / n);
  }
  __device__ __forceinline__ int nck(int2 s) const { return (s.x + s.y + kc - 1) / kc; }
  __device__ __forceinline__ int tiles(int2 s) const { return (s.x * n_rep + rows - 1) / rows; }
  __device__ __forceinline__ int per(int2 s) const { return nck(s) + over; }
  __device__ __forceinline__ int units(int2 s) const {
    return s.x > 0 ? a.Hkv * tiles(s) * per(s) : 0;
  }
  __device__ __forceinline__ int chunks(int b) const { return units(tree_seq(a, b)); }
};

// Place in the list: sequence b (s: its nodes in use and prefix length), KV head
// g, row tile t, chunk c of nck, unit u.
struct TreeCursor {
  int b, g, t, c, u, nck, tiles;
  int2 s;
  __device__ __forceinline__ void at(const TreeSched& sched, int b_, int2 s_) {
    b = b_;
    s = s_;
    s.x = __builtin_amdgcn_readfirstlane(s.x);
    s.y = __builtin_amdgcn_readfirstlane(s.y);
    nck = sched.nck(s);
    tiles = sched.tiles(s);
  }
  // the first chunk at or behind a unit
  __device__ __forceinline__ void seek(const TreeSched& sched, int unit, int lane) {
    int sb, base;
    if (sched.B <= 64) {  // a lane a sequence, without another load
      const int n = sched.units(sched.own), end = wave_prefix(n);
      sb = __builtin_ctzll(__builtin_amdgcn_ballot_w64(end - n <= unit && unit < end) | 1ull << 63);
      base = __builtin_amdgcn_readlane(end - n, sb);
      at(sched, sb, make_int2(__builtin_amdgcn_readlane(sched.own.x, sb),
                              __builtin_amdgcn_readlane(sched.own.y, sb)));
    } else {
      locate_chunk(sched, unit, lane, sb, base);
      at(sched, sb, tree_seq(sched.a, sb));
    }
    const int per = nck + sched.over, item = (unit - base) / per;
    c = max(unit - base - item * per - sched.over, 0);
    u = base + item * per + sched.over + c;
    t = item % tiles;
    g = item / tiles;
  }
  __device__ __forceinline__ void next(const TreeSched& sched) {
    ++u;
    if (++c < nck) return;
    c = 0;
    u += sched.over;
    if (++t < tiles) return;
    t = 0;
    if (++g < sched.a.Hkv) return;
    g = 0;
    for (int nb = b + 1; nb < sched.B; ++nb) {
      const int2 sn = tree_seq(sched.a, nb);
      if (sn.x > 0) {
        at(sched, nb, sn);
        return;
      }
    }
    b = sched.B;  // behind the last chunk (u is past every share)
  }
};

template <typename T, int D, int RW, int BKW>
__global__ __launch_bounds__(256, (Shape<T, D, RW, BKW>::PER_CU)) void tree_stream_kernel(
    TreeArgs a, int W, float* __restrict__ opart, float* __restrict__ mlpart,
    int* __restrict__ refusals, int2* __restrict__ shares, int tiles_max) {
  using namespace mfma;
  using X = Tile<T, D>;
  using P = Piece<T>;
  using Sh = Shape<T, D, RW, BKW>;
  constexpr int KW = Sh::KW, ROWS = Sh::ROWS, KC = Sh::KC, NB = BKW / 32, DT = D / 32;
  constexpr int E = P::E, HALF = D / 2;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  __shared__ TreeLds tree;
  __shared__ uint32_t sbad[KC / 32];  // the chunk's V rows with Inf or NaN
  const int w = wave_id(), lane = threadIdx.x & 63, h = lane >> 5, l31 = lane & 31;
  const int rw = w % RW, kw = w / RW;
  const int N = a.N, n_rep = a.Hq / a.Hkv;
  const TreeSched sched(a, n_rep, ROWS, KC, gridDim.x, lane);
  const int NW = sched.NW;
  // block ids go round the 8 XCDs: neighbours in the chunk list, which read the
  // same keys for other rows, share one XCD's L2
  if ((int)blockIdx.x >= NW) return;
  const int xcd = blockIdx.x % 8, gw = xcd * (NW / 8) + min(xcd, NW % 8) + (int)blockIdx.x / 8;
  const int u_hi = sched.start(gw + 1);
  TreeCursor cc;
  cc.seek(sched, sched.start(gw), lane);
  if (cc.u >= u_hi) return;  // (a share of nothing but a tile's beginning)

  auto stage_k = [&](int i) { return (T*)(lds + (i & 1) * Sh::STAGE); };
  auto issue = [&](const TreeCursor& p, int i) {
    const int64_t row = ((int64_t)p.b * a.Hkv + p.g) * a.Smax + (int64_t)p.c * KC;
    const int rows = p.s.x + p.s.y - p.c * KC;  // >= 1; rows past the last repeat it
    uint16_t* dst = (uint16_t*)stage_k(i);
    constexpr int U = sizeof(T) / 2;
    // (two row waves: the loads' offsets formed anew each time, for registers; 7%
    // of the time where the products bound it, nothing where HBM does)
    constexpr bool FRESH = RW == 2;
    tile_to_lds<KC, X::R, 4, FRESH>((const uint16_t*)((const T*)a.k_cache + row * D), D * U, dst,
                                    w, lane, rows);
    tile_to_lds<KC, X::R, 4, FRESH>((const uint16_t*)((const T*)a.v_cache + row * D), D * U,
                                    dst + Sh::TILE * U, w, lane, rows);
  };
  // the table row of node j (kept inside the table: a refused sequence's may not be)
  auto table_row = [&](int2 s, int j) {
    const int64_t r = (int64_t)s.y + (a.parents != nullptr ? tree.depth[j] : j) - a.rope_row_offset;
    return min(max(r, (int64_t)0), a.rope_rows - 1) * HALF;
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
  // P = 2^(s - m + LIFT) stays below 2^(SLACK + LIFT).  float16 has no numbers below 2^-24:
  // thousands of keys at 2^-25 of one key's probability (a first token that takes most of
  // the mass and has no value) would all round to 0, so its P fills the range up to 2^15
  // and the reference moves more often; the other types have float32's range.  (tree of 64
  // nodes, 16384 keys, as above: 282 us in float16, of which 10 for the conversions of P's
  // split and this.)
  constexpr bool HALF_P = std::is_same<T, _Float16>::value;
  constexpr float SLACK = HALF_P ? 2.f : 8.f, LIFT = HALF_P ? 13.f : 0.f;
  bool whole = false;    // this workgroup holds all of the row tile's chunks
  bool refused = false;  // the sequence's tree or tables are out of range
  int node = 0;

  // The beginning of a row tile: lane l's row of the queries, dims of half h,
  // 16-byte pieces 2 ks + h; a piece's RoPE partner is the lane's own piece KS / 2
  // further on.
  auto load_q = [&](u32x4* raw) {
    const int row = min(cc.t * ROWS + 32 * rw + l31, cc.s.x * n_rep - 1);
    node = row / n_rep;
    const T* qr = (const T*)a.q_new +
                  (((int64_t)cc.b * N + node) * a.Hq + cc.g * n_rep + row % n_rep) * D;
#pragma unroll
    for (int ks = 0; ks < X::KS; ++ks) raw[ks] = *(const u32x4*)(qr + (2 * ks + h) * E);
  };
  auto load_angles = [&](Angles* ang) {  // (one round trip for all)
    const int64_t trow = table_row(cc.s, node);
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
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[dt][e] = 0.f;
    whole = cc.c == 0;
    if (whole && threadIdx.x == 0) {
      shares[(cc.b * a.Hkv + cc.g) * tiles_max + cc.t].x = gw;
      if (cc.g == 0 && cc.t == 0) refusals[cc.b] = refused;
    }
  };
  {
    // Loads return in order, so what the first tile needs is waited for before its
    // first chunk is asked for, and the rest of its beginning runs under that.
    u32x4 raw[X::KS];
    Angles ang[X::KS / 2];
    int par = tree_parent(a, cc.b, cc.s);
    load_q(raw);
    settle(par);
#pragma unroll
    for (int ks = 0; ks < X::KS; ++ks) settle(raw[ks]);
    if (a.parents == nullptr) {
      load_angles(ang);
#pragma unroll
      for (int ks = 0; ks < X::KS / 2; ++ks)
#pragma unroll
        for (int x = 0; x < E / 4; ++x) {
          settle(ang[ks].c[x]);
          settle(ang[ks].s[x]);
        }
    }
    issue(cc, 0);
    refused = tree_build(a, cc.s, W, tree, par);
    if (a.parents != nullptr) load_angles(ang);
    rotate_q(raw, ang);
  }

  for (int i = 0;; ++i) {
    TreeCursor ic = cc;
    ic.next(sched);
    const bool more = ic.u < u_hi;
    lds_copy_wait();
    __syncthreads();  // chunk i has landed for all; the other stage is free
    if (more) issue(ic, i + 1);
    T* kt = stage_k(i);
    T* vt = kt + Sh::TILE;
    const bool tail = cc.c * KC + KC > cc.s.y;  // the chunk holds nodes, or ends behind them
    if (tail) {
      // The nodes' rows, from k_new and v_new over what the cache held there;
      // the first row tile's workgroup writes them to the cache as well.  V rows
      // behind the last become zero: 0 x NaN must not reach a sum.
      constexpr int G = HALF / E;  // lanes of a row, a piece of each half a lane
      const int r0 = cc.c * KC, L = cc.s.y, n = cc.s.x;
      const int j0 = max(r0 - L, 0), j1 = min(r0 + KC - L, n);
      const int64_t head = (int64_t)cc.b * a.Hkv + cc.g;
      int tid = threadIdx.x;
      asm volatile("" : "+v"(tid));  // (nothing of this block is kept across the loop)
      if (tid < KC / 32) sbad[tid] = 0;
      __syncthreads();
      for (int x = tid; x < (j1 - j0) * G; x += 256) {
        const int j = j0 + x / G, d = x % G * E, lr = L + j - r0, sw = swz<X::R>(lr);
        const int64_t src = (((int64_t)cc.b * N + j) * a.Hkv + cc.g) * D;
        const int ca = ((d / E) ^ sw) * E, cb = (((d + HALF) / E) ^ sw) * E;
        const int64_t dst = (head * a.Smax + L + j) * D + d;
        const bool store = cc.t == 0 && !refused;
        P kx, vx;  // all loads first: one round trip
        float f1[E], f2[E];
        kx.load((const T*)a.k_new + src, d, HALF);
        const Angles g = angles(table_row(cc.s, j), d);
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
        if (store) {
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
      for (int x = (L + j1 - r0) * X::R + tid; x < KC * X::R; x += 256)
        *(u32x4*)(vt + x * E) = u32x4{0u, 0u, 0u, 0u};
      __syncthreads();
    }
    const int L = cc.s.y;
    const int k0 = cc.c * KC + kw * BKW;  // the wavefront's first key
    // Which of a block's 32 keys the lane's row sees, the first of them node t0 (>
    // -32; keys before node 0 are the prefix); and which have Inf or NaN in V.
    auto sees = [&](int t0) -> uint32_t {
      if (a.parents == nullptr) {  // nodes 0 .. node
        const int lo = node + 1 - t0;
        return lo <= 0 ? 0u : lo >= 32 ? ~0u : (1u << lo) - 1u;
      }
      const int idx = t0 >> 5, sh = t0 & 31;
      const uint32_t w0 = idx < 0 ? ~0u : idx < W ? tree.mask[node][idx] : 0u;
      const uint32_t w1 = idx + 1 < W ? tree.mask[node][idx + 1] : 0u;
      return sh ? (w0 >> sh) | (w1 << (32 - sh)) : w0;
    };
    auto unclean = [&](int nb) -> uint32_t {
      return __builtin_amdgcn_readfirstlane(sbad[(kw * BKW + 32 * nb) / 32]);
    };
    // The blocks of 32 keys that the wavefront's last row sees (no node sees one behind
    // it; a chain of 200 for 4 sequences: 58.3 us with all of them, 57.1 without); a
    // wavefront of which the tile has no rows leaves the SIMD to the others.
    const int blocks = cc.t * ROWS + 32 * rw < cc.s.x * n_rep
                           ? (__builtin_amdgcn_readlane(node, 31) + L - k0 + 32) >> 5
                           : 0;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {  // 32 keys at a time
      if (nb >= blocks) break;
      const int row0 = kw * BKW + 32 * nb;
      const int t0 = k0 + 32 * nb - L;
      f32x16 s;
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = 0.f;
      X::scores(kt, row0, q, s, lane);
      bool bad = false;
      if (t0 > -32) {  // (uniform)
        const uint32_t bits = sees(t0) >> (4 * h);
#pragma unroll
        for (int e = 0; e < 16; ++e)
          s[e] = (bits >> (8 * (e / 4) + e % 4)) & 1 ? s[e] : -INFINITY;
        bad = unclean(nb) != 0;
      }
      if (bad) {  // 0 x Inf must not reach the rows that do not see the key
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
      if (bad) {  // those keys one by one, for the rows that see them
        const uint32_t bits = sees(t0);
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
                          (((int64_t)cc.b * N + t0 + kk) * a.Hkv + cc.g) * D + hh;
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
    if (last || !more) {
      // the row tile's part of this workgroup ends: the key waves' sums joined in
      // the stage just computed, then the output, or a partial in slot gw + tile
      whole = whole && last;
      if (last && threadIdx.x == 0) shares[(cc.b * a.Hkv + cc.g) * tiles_max + cc.t].y = gw;
      float l = pair_sum32(lsum);
      if (refused) l = NAN;
      if (l != l) m = INFINITY;  // (a NaN must not be left out for its weight)
      // The key waves share the join out by blocks of 32 dims: block dt is wave
      // owner(dt)'s, the others leave theirs in LDS (one wave joining all of them: 5
      // nodes over 1000 keys 15.8 us, shared out 14.6).
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
      if (r < cc.s.x * n_rep) {
        if (whole) {
          const float inv = 1.f / l;
          T* o = (T*)a.out + (((int64_t)cc.b * N + r / n_rep) * a.Hq + cc.g * n_rep + r % n_rep) * D +
                 4 * h;
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
          const int64_t slot = (int64_t)gw + ((int64_t)cc.b * a.Hkv + cc.g) * tiles_max + cc.t;
          float* o = opart + (slot * ROWS + 32 * rw + l31) * D + 4 * h;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int e = 0; e < 16 && owner(dt) == kw; e += 4)
              *(f32x4*)(o + 32 * dt + 2 * e) =
                  f32x4{acc[dt][e], acc[dt][e + 1], acc[dt][e + 2], acc[dt][e + 3]};
          if (h == 0 && kw == 0)
            *(float2*)(mlpart + (slot * ROWS + 32 * rw + l31) * 2) = make_float2(m, l);
        }
      }
    }
    if (!more) break;
    const bool new_tree = ic.b != cc.b;
    cc = ic;
    if (cc.c == 0) {
      u32x4 raw[X::KS];
      Angles ang[X::KS / 2];
      load_q(raw);
      if (new_tree) refused = tree_build(a, cc.s, W, tree, tree_parent(a, cc.b, cc.s));
      load_angles(ang);
      rotate_q(raw, ang);
    }
  }
}

// The rows of tile blockIdx.x, 16 bytes of a row per thread and blockIdx.y's share
// of them: the partials of the workgroups that met the tile, rescaled to a common
// maximum and summed; a tile that one workgroup finished is left alone.  JG groups of
// threads take a row's partials in turn, U at a time, and are joined through LDS:
// what it costs is the round trips of a thread's loads, one a batch.
template <typename T, int D, int JG>
__global__ __launch_bounds__(256) void tree_merge_kernel(
    TreeArgs a, const float* __restrict__ opart, const float* __restrict__ mlpart,
    const int* __restrict__ refusals, const int2* __restrict__ shares, int rows, int tiles_max) {
  constexpr int LPR = D / 4, RPW = 256 / (LPR * JG);  // lanes of a row, rows of a workgroup
  __shared__ f32x4 xo[JG > 1 ? 256 : 1];
  __shared__ float2 xm[JG > 1 ? 256 : 1];
  const int n_rep = a.Hq / a.Hkv;
  const int item = blockIdx.x, t = item % tiles_max, bg = item / tiles_max, b = bg / a.Hkv,
            g = bg % a.Hkv;
  const int r = blockIdx.y * RPW + threadIdx.x / (LPR * JG), jg = threadIdx.x / LPR % JG;
  const int col = threadIdx.x % LPR * 4;
  const int row = t * rows + r, i = row / n_rep, hq = g * n_rep + row % n_rep;
  const int2 s = tree_seq(a, b);
  const bool inside = i < a.N && r < rows;
  T* dst = (T*)a.out + (((int64_t)b * a.N + i) * a.Hq + hq) * D + col;
  T y[4];
  if (inside && jg == 0 && (s.x < 0 || i >= s.x)) {  // a refused sequence, or an unused node
    const bool refused = s.x < 0 || (s.x > 0 && refusals[b]);
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = from_f32<T>(refused ? NAN : 0.f);
    __builtin_memcpy(__builtin_assume_aligned(dst, 4 * sizeof(T)), y, sizeof(y));
  }
  const int2 share = shares[item];  // (of a tile without rows: whatever was there)
  const int w0 = share.x, ns = inside && i < s.x ? share.y - w0 + 1 : 0;
  const bool live = ns > 1;
  float M = -INFINITY, l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  // joins a partial (of weight 0: left out, whatever it holds)
  auto add = [&](float f, const float2& ml, const f32x4& po) {
    const float w = fast_exp2(ml.x - M);
    l = l * f + (w != 0.f ? w * ml.y : 0.f);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = o[e] * f + (w != 0.f ? w * po[e] : 0.f);
  };
  if (live) {
    const int64_t first = ((int64_t)w0 + item) * rows + r;
    const float* ob = opart + first * D + col;
    const float2* mb = (const float2*)mlpart + first;
    constexpr int U = 8;
    for (int j0 = jg; j0 < ns; j0 += U * JG) {
      f32x4 po[U];
      float2 ml[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t j = min(j0 + u * JG, ns - 1);
        ml[u] = mb[j * rows];
        po[u] = *(const f32x4*)(ob + j * rows * D);
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

// The stream kernel's shape for a call: row waves (0: one wavefront per row) and
// what follows from it.
struct Plan {
  int rw, bkw, rows, kc, tiles, grid, per_cu;
};
Plan plan_of(const TreeArgs& a) {
  Plan p = {};
  const int n_rep = a.Hq / a.Hkv, m = a.N * n_rep;
  if (a.D != 64 && a.D != 128) return p;
  // Enough row waves for the pair's rows, up to four: finer tiles have fewer rows to
  // spare, but load the keys more often (800 rows of 4 x 8 heads over 1224 keys: 73 us
  // with 128 rows a tile, 84 with 64, 125 with 32; 135 rows 36, 39, 38; 36 rows the
  // other way, 40.9 and 39.5).  float32, which has no LDS for four key waves, is bound
  // by its products: two row waves where they need five sixths of four's row waves or
  // fewer (30 x 2 heads, 2121 keys, 145 rows, 6 to 8: 157 us with two, 170 with four; 4 x
  // 8 heads, 1224 keys, 400 rows, 14 to 16: 133 and 126).
  const int two = 2 * ((m + 63) / 64), four = 4 * ((m + 127) / 128);
  p.rw = a.dtype == F32 ? (6 * two <= 5 * four ? 2 : 4) : m <= 32 ? 1 : m <= 64 ? 2 : 4;
  p.bkw = p.rw == 4 && a.dtype != F32 ? 64 : 32;
  p.rows = 32 * p.rw;
  p.kc = p.bkw * 4 / p.rw;
  p.tiles = (m + p.rows - 1) / p.rows;
  const size_t lds = (size_t)4 * p.kc * a.D * (a.dtype == F32 ? 4 : 2) +
                     (p.rw < 4 ? (size_t)(4 / p.rw) * p.rows * 8 : 0);  // Shape::LDS
  p.per_cu = 2 * lds <= 160 * 1024 && !(a.dtype == F32 && a.D == 128) ? 2 : 1;  // Shape::PER_CU
  const int64_t chunks = (int64_t)a.B * a.Hkv * p.tiles * ((a.max_len + p.kc - 1) / p.kc);
  if (chunks + (int64_t)a.B * a.Hkv * p.tiles * TreeSched::OVER >= INT_MAX) return Plan{};
  p.grid = (int)std::min<int64_t>(p.per_cu * std::min(device_cu_count(), 512), chunks);
  return p;
}

// workspace: the partials, per row tile the first and last of the workgroups that met it
// (each writes itself; formed again from the lengths by every workgroup of the merge
// it cost that 3 us), whether each sequence's tree or tables are refused; or, one wavefront per row, rotated queries, ancestor
// masks and per sequence (nodes in use or -1, prefix length)
struct Ws {
  float *opart, *mlpart;
  int* refusals;
  int2* shares;
  float* qrot;
  uint32_t* anc;
  int2* seq;
  size_t bytes;
};
Ws carve(const TreeArgs& a, const Plan& pl, void* p) {
  char* c = (char*)p;
  Ws w = {};
  if (pl.rw) {
    const size_t rows = ((size_t)pl.grid + (size_t)a.B * a.Hkv * pl.tiles) * pl.rows;
    w.opart = (float*)c;
    c += up256(rows * a.D * 4);
    w.mlpart = (float*)c;
    c += up256(rows * 2 * 4);
    w.refusals = (int*)c;
    c += up256((size_t)a.B * 4);
    w.shares = (int2*)c;
    c += up256((size_t)a.B * a.Hkv * pl.tiles * sizeof(int2));
  } else {
    w.qrot = (float*)c;
    c += up256((size_t)a.B * a.N * a.Hq * a.D * 4);
    w.anc = (uint32_t*)c;
    c += up256((size_t)a.B * a.N * ((a.N + 31) / 32) * 4);
    w.seq = (int2*)c;
    c += up256((size_t)a.B * sizeof(int2));
  }
  w.bytes = (size_t)(c - (char*)p);
  return w;
}

template <typename T, int D, int RW, int BKW>
int launch_stream(const TreeArgs& a, const Ws& w, const Plan& p) {
  using Sh = Shape<T, D, RW, BKW>;
  auto kernel = tree_stream_kernel<T, D, RW, BKW>;
  if (Sh::LDS + sizeof(TreeLds) + 1024 > 64 * 1024) {  // asked for once per device
    static std::atomic<uint64_t> done{0};
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    const uint64_t bit = dev >= 0 && dev < 64 ? 1ull << dev : 0;
    if (e == hipSuccess && !(done.load(std::memory_order_relaxed) & bit)) {
      e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize,
                              (int)Sh::LDS);
      if (e == hipSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    }
    if (e != hipSuccess) {
      set_error("tree attention: %s", hipGetErrorString(e));
      return KF_ERR_HIP;
    }
  }
  KF_LAUNCH("tree_stream", kernel, dim3(p.grid), dim3(256), Sh::LDS, a.stream, a,
            (a.N + 31) / 32, w.opart, w.mlpart, w.refusals, w.shares, p.tiles);
  KF_CHECK_LAUNCH();
  return KF_OK;
}

template <typename T, int D>
int stream_and_merge(const TreeArgs& a, const Ws& w, const Plan& p) {
  int rc;
  if constexpr (std::is_same<T, float>::value)
    rc = p.rw == 2 ? launch_stream<T, D, 2, 32>(a, w, p) : launch_stream<T, D, 4, 32>(a, w, p);
  else
    rc = p.rw == 1   ? launch_stream<T, D, 1, 32>(a, w, p)
         : p.rw == 2 ? launch_stream<T, D, 2, 32>(a, w, p)
                     : launch_stream<T, D, 4, 64>(a, w, p);
  if (rc) return rc;
  // About `grid / items` partials a tile; a batch of 8 is one round trip.  63 of them (27
  // nodes of 5 heads over 4000 keys): the whole call 29.8 us with one group, 26.4 with
  // two, 23.8 with eight; 16 of them: 29.5 with one, 28.2 with two, 29 with four (each
  // further group is as many workgroups more).
  const int items = a.B * a.Hkv * p.tiles;
  const int jg = p.grid > 32 * items ? 8 : p.grid > 8 * items ? 2 : 1;
  const int rpw = 256 / (D / 4) / jg;  // rows of a workgroup
  KF_LAUNCH("tree_merge",
            (jg == 8   ? tree_merge_kernel<T, D, 8>
             : jg == 2 ? tree_merge_kernel<T, D, 2>
                       : tree_merge_kernel<T, D, 1>),
            dim3(items, (p.rows + rpw - 1) / rpw), dim3(256), 0, a.stream, a, w.opart, w.mlpart,
            w.refusals, w.shares, p.rows, p.tiles);
  KF_CHECK_LAUNCH();
  return KF_OK;
}

template <typename T>
int tree_typed(const TreeArgs& a, void* workspace) {
  Plan p = plan_of(a);
  // (direct loads to LDS and 16-byte rows need aligned buffers)
  if (((uintptr_t)a.q_new | (uintptr_t)a.k_new | (uintptr_t)a.v_new | (uintptr_t)a.k_cache |
       (uintptr_t)a.v_cache | (uintptr_t)a.out | (uintptr_t)a.cos | (uintptr_t)a.sin) % 16 != 0)
    p = Plan{};
  const Ws w = carve(a, p, workspace);
  if (p.rw)
    return a.D == 128 ? stream_and_merge<T, 128>(a, w, p) : stream_and_merge<T, 64>(a, w, p);
  const int W = (a.N + 31) / 32, per = 16;
  const int64_t rows = (int64_t)a.N * (a.Hq + 2 * a.Hkv);
  KF_LAUNCH("tree_prep", tree_prep_kernel<T>, dim3((unsigned)((rows + per - 1) / per), a.B),
            dim3(256), 0, a.stream, a, w.qrot, w.anc, w.seq, W, per);
  KF_CHECK_LAUNCH();
  KF_LAUNCH("tree_rows", tree_rows_kernel<T>,
            dim3((unsigned)(((int64_t)a.B * a.N * a.Hq + 3) / 4)), dim3(256), 0, a.stream, a,
            w.qrot, w.anc, w.seq, W);
  KF_CHECK_LAUNCH();
  return KF_OK;
}

}  // namespace

size_t tree_workspace(const TreeArgs& a) {
  // (which of the two a call takes goes by its buffers' alignment too)
  return std::max(carve(a, plan_of(a), nullptr).bytes, carve(a, Plan{}, nullptr).bytes);
}

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
