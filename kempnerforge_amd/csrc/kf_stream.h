// What the split-K kernels over KV caches with several rows per KV head share: the
// attention of drafted trees (kf_tree.hip) and of branches behind a shared prefix
// (kf_branch.hip).
#pragma once

#include "kf_common.h"
#include "kf_mfma.h"

namespace kf {

template <typename T>
__device__ __forceinline__ bool finite(T x) {
  return fabsf(to_f32(x)) < INFINITY;  // false for NaN too
}

// One piece of a row: E = 16 / sizeof(T) elements of each RoPE half, 16-byte
// loads and stores.
template <typename T>
struct Piece {
  static constexpr int E = 16 / sizeof(T);
  u32x4 a, b;
  __device__ __forceinline__ void load(const T* row, int d, int half) {
    a = *(const u32x4*)(row + d);
    b = *(const u32x4*)(row + d + half);
  }
  static __device__ __forceinline__ void unpack(const u32x4& u, float* f) {
    if constexpr (sizeof(T) == 4)
      __builtin_memcpy(f, &u, 16);
    else
      unpack8<T>(u, f);
  }
  static __device__ __forceinline__ u32x4 pack(const float* f) {
    if constexpr (sizeof(T) == 4)
      return u32x4{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                   __float_as_uint(f[3])};
    else
      return pack8<T>(f);
  }
};

// Inclusive prefix sums over the wavefront, by data parallel primitives (a shuffle
// goes through the LDS, six of them cost 0.3 us): within rows of 16 lanes, then lane
// 15 of rows 0 and 2 into the next row, then lane 31 into rows 2 and 3.
__device__ __forceinline__ int wave_prefix(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);   // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);   // row_shr:2
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);   // row_shr:4
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);   // row_shr:8
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31
  return x;
}

// What depends on the element type: the products on 32 x 32 tiles.
//   S^T (keys x rows) += K q^T: lane l supplies row l % 32 of both operands, dims
//       of its half h = l / 32 in 16-byte pieces
//   O^T (dims x rows) += V^T P^T: P^T straight from the S registers (lane l holds
//       row l % 32, register i key 8 (i / 4) + 4 h + i % 4), hi and lo one after the
//       other on each V fragment: 16 keys at a time, so that those of the other 16 hold
//       no registers
// Every fragment is read PF steps ahead of its products: left to itself the
// compiler, short of registers, reads each one right before them and waits out
// the LDS (512 rows over 16384 keys, 4 x 8 KV heads of 128: 232 us, read ahead 218).
template <typename T, int D>
struct Tile {
  static constexpr int R = D / 8;     // 16-byte chunks per cache row
  static constexpr int KS = D / 16;   // pieces of a lane's half row
  static constexpr int QP = 2;        // q as hi and lo
  static constexpr int PF = D == 128 ? 2 : 4;  // (what the registers hold)
  static constexpr int DT = D / 32, NV = 2 * DT;  // V fragments: 16 keys of 32 dims
  // lds_frag_t's offsets: block dt's are the first block's with bits 6.. flipped by
  // dt (a swizzled chunk index is 4 dt ^ ...), which saves the registers of the others
  struct VOff {
    uint32_t o[2];
  };
  typedef bf16x8 VFrag[PF];
  static __device__ __forceinline__ VOff v_off(int lane) {
    const mfma::TrOffsets<D> t = mfma::tr_offsets<D>(lane);
    return VOff{{t.o[0][0], t.o[0][1]}};
  }
  static __device__ __forceinline__ bf16x8 v_frag(const T* v, int row0, const VOff& off, int c,
                                                  int dt) {
    using namespace mfma;
    const char* base = (const char*)v + (row0 + c * 16) * D * 2;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_s16x4_ptr)(base + (off.o[0] ^ (dt * 64))));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_s16x4_ptr)(base + (off.o[1] ^ (dt * 64))));
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    const s16x8 x = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(bf16x8, x);
  }
  static __device__ __forceinline__ void scores(const T* k, int row0, const u32x4 (*q)[KS],
                                                f32x16& s, int lane) {
    using namespace mfma;
    bf16x8 f[PF];
#pragma unroll
    for (int i = 0; i < PF; ++i) f[i] = lds_frag<R>(k, row0 + (lane & 31), 2 * i + (lane >> 5));
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      s = mfma32<T>(f[ks % PF], as_bf16x8(q[0][ks]), s);
      s = mfma32<T>(f[ks % PF], as_bf16x8(q[1][ks]), s);
      if (ks + PF < KS)
        f[ks % PF] = lds_frag<R>(k, row0 + (lane & 31), 2 * (ks + PF) + (lane >> 5));
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  static __device__ __forceinline__ void load_v(const T* v, int row0, const VOff& off, VFrag& f,
                                                int) {
#pragma unroll
    for (int i = 0; i < PF; ++i) f[i] = v_frag(v, row0, off, i / DT, i % DT);
    __builtin_amdgcn_sched_barrier(0);
  }
  // x and y as sums hi + lo of two numbers of the type
  static __device__ __forceinline__ uint2 split2(float x, float y) {
    const uint32_t hi = pack2<T>(x, y);
    float a, b;
    unpack2<T>(hi, a, b);
    return make_uint2(hi, pack2<T>(x - a, y - b));
  }
  static __device__ __forceinline__ void values(const T* v, int row0, const VOff& off,
                                                const f32x16& p, VFrag& f, f32x16* acc, int) {
    using namespace mfma;
    u32x4 hi, lo;
#pragma unroll
    for (int i = 0; i < NV; ++i) {  // keys 16 (i / DT) .., dims 32 (i % DT) ..
      if (i % DT == 0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int e = 8 * (i / DT) + 2 * j;
          const uint2 u = split2(p[e], p[e + 1]);
          hi[j] = u.x;
          lo[j] = u.y;
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      acc[i % DT] = mfma32<T>(f[i % PF], as_bf16x8(hi), acc[i % DT]);
      acc[i % DT] = mfma32<T>(f[i % PF], as_bf16x8(lo), acc[i % DT]);
      if (i + PF < NV) f[i % PF] = v_frag(v, row0, off, (i + PF) / DT, (i + PF) % DT);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
};
template <int D>
struct Tile<float, D> {
  static constexpr int R = D / 4;
  static constexpr int KS = D / 8;
  static constexpr int QP = 1;
  static constexpr int PF = 2;
  struct VOff {};
  struct VFrag {};
  static __device__ __forceinline__ VOff v_off(int) { return {}; }
  static __device__ __forceinline__ f32x16 mma(float a, float b, const f32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ void scores(const float* k, int row0, const u32x4 (*q)[KS],
                                                f32x16& s, int lane) {
    const int row = row0 + (lane & 31), sw = mfma::swz<R>(row);
    auto frag = [&](int ks) {
      return *(const f32x4*)(k + (row * R + ((2 * ks + (lane >> 5)) ^ sw)) * 4);
    };
    f32x4 f[PF];
#pragma unroll
    for (int i = 0; i < PF; ++i) f[i] = frag(i);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const f32x4 b = __builtin_bit_cast(f32x4, q[0][ks]);
#pragma unroll
      for (int e = 0; e < 4; ++e) s = mma(f[ks % PF][e], b[e], s);
      if (ks + PF < KS) f[ks % PF] = frag(ks + PF);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  static __device__ __forceinline__ void load_v(const float*, int, const VOff&, VFrag&, int) {}
  static __device__ __forceinline__ void values(const float* v, int row0, const VOff&,
                                                const f32x16& p, VFrag&, f32x16* acc, int lane) {
    constexpr int DT = D / 32;
    auto frag = [&](int i, float* f) {  // keys 8 (i / 4) + 4 h + i % 4
      const int row = row0 + 8 * (i / 4) + 4 * (lane >> 5) + i % 4, sw = mfma::swz<R>(row);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
        f[dt] = v[(row * R + ((8 * dt + ((lane & 31) >> 2)) ^ sw)) * 4 + (lane & 3)];
    };
    float f[PF][DT];
#pragma unroll
    for (int i = 0; i < PF; ++i) frag(i, f[i]);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) acc[dt] = mma(f[i % PF][dt], p[i], acc[dt]);
      if (i + PF < 16) frag(i + PF, f[i % PF]);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
};

// A workgroup of four wavefronts: RW of them side by side over the rows (32
// each), KW = 4 / RW over the keys of a chunk (BKW each).  A chunk's K and V rows
// go straight from the cache to one of two LDS stages while the other one is
// computed; one barrier per chunk.
template <typename T, int D, int RW, int BKW>
struct Shape {
  static constexpr int KW = 4 / RW, ROWS = 32 * RW, KC = BKW * KW;
  static constexpr int TILE = KC * D;                  // elements of a K (or V) tile
  static constexpr size_t STAGE = 2 * TILE * sizeof(T);
  static constexpr size_t LDS = 2 * STAGE + (KW > 1 ? KW : 0) * ROWS * 2 * sizeof(float);
  // (float32 rows of 128: q, the sums and a block's scores leave no room for two
  // wavefronts per SIMD)
  static constexpr int PER_CU = LDS * 2 <= 160 * 1024 && D * sizeof(T) <= 256 ? 2 : 1;
  static_assert((KW - 1) * ROWS * D * sizeof(float) <= STAGE, "the key waves' exchange");
};

}  // namespace kf
