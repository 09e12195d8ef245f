// Weight tiles in the matrix cores' operand order, and their products with
// row-major activation rows. Shared by the 4-bit projections (mx4.hip) and the
// mixture-of-experts layer (moe.hip).
//
// A tile is 16 weight rows x 128 k. Lane l of a wave holds row l % 16 and the 32
// consecutive k of block l / 16 -- in the 4-bit format one microscaling block with
// its one scale, so a tile of codes is a single 16-byte load a lane and its scales
// one byte a lane. The other formats keep the same k order (4 pieces of 8 bf16, 8
// pieces of 4 float), so one activation operand serves every format: a lane's
// 32 consecutive activations of a row. The sum over k is taken in any order as
// long as both operands agree, and every load of weights is whole lines
// (1 KB a wave) however k is split over waves.
//
//   tiles  [matrix][row tile][k tile] of  MX4: 1024 B codes (dword s of a lane:
//            its elements 8 s .. 8 s + 7, the first in the low nibble) and, in an
//            array of their own, 64 B scales (one per lane);
//          bf16: [4][64 lanes][16 B];  float: [8][64 lanes][16 B]
// Rows past n and blocks past k hold zeros (scale byte 0).
//
// Products: bf16 16x16x32 MFMAs accumulate in float. 4-bit weights times a power
// of two are exact in bf16 (two significant bits, bf16's exponent range and
// subnormals reach every scale), so they lose nothing on the way in; float
// activations meet them as three bf16 parts of 8 bits each, whose sum is the
// float exactly. Float weights take 16x16x4 float MFMAs.
#pragma once

#include "common.h"

constexpr int WT_ROWS = 16;
constexpr int WT_K = 128;
constexpr int MX_BLOCK = 32;

struct WMx4 {};
struct WBf16 {};
struct WF32 {};

// a tiled weight: matrices of rt x kt tiles; scales is null but for MX4
struct WMat {
  const void* data;
  const uint8_t* scales;
};

__host__ __device__ __forceinline__ int wt_row_tiles(int n) { return (n + WT_ROWS - 1) / WT_ROWS; }
__host__ __device__ __forceinline__ int wt_k_tiles(int k) { return (k + WT_K - 1) / WT_K; }

// 8 codes (a dword) times 2^(scale - 127) as 8 bf16, by the hardware conversion
// (scale byte 255 gives NaN)
__device__ __forceinline__ bf16x8_t mx4_frag(unsigned q, float scale) {
  const u32x4_t r = {
      __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 0)),
      __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 1)),
      __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 2)),
      __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 3))};
  return __builtin_bit_cast(bf16x8_t, r);
}

__device__ __forceinline__ f32x4_t mma_bf16(bf16x8_t a, bf16x8_t b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// A float as three bf16 parts of 8 significant bits, cut and not rounded: the
// sum is the float. Infinities and NaN sit in the first part alone.
__device__ __forceinline__ void split3(float v, unsigned& hi, unsigned& mid, unsigned& lo) {
  const unsigned b = __float_as_uint(v);
  const bool finite = (b & 0x7f800000u) != 0x7f800000u;
  hi = (b & 0xffff0000u) | (v != v ? 0x00400000u : 0u);
  const float r = finite ? v - __uint_as_float(hi) : 0.f;
  mid = __float_as_uint(r) & 0xffff0000u;
  lo = __float_as_uint(r - __uint_as_float(mid));
}

// One format of weights against one type of activations.
//   W / X   a lane's part of a weight tile / of 16 activation rows over the same k
//   step    acc += W X over the tile's 128 k; lane: weight rows 4 (l / 16) + i,
//           activation row l % 16
template <typename WF, typename T> struct Fmt;

template <> struct Fmt<WBf16, bf16_t> {
  static constexpr int TILE = 4096;
  struct W { u32x4_t f[4]; };
  struct X { u32x4_t f[4]; };
  __device__ __forceinline__ static W load_w(const WMat& m, long tile, int lane) {
    W w;
    const char* p = static_cast<const char*>(m.data) + tile * TILE + lane * 16;
#pragma unroll
    for (int s = 0; s < 4; ++s) w.f[s] = *reinterpret_cast<const u32x4_t*>(p + s * 1024);
    return w;
  }
  // p: the lane's 32 activations, or null for zeros
  __device__ __forceinline__ static X load_x(const bf16_t* p) {
    X x;
#pragma unroll
    for (int s = 0; s < 4; ++s) x.f[s] = u32x4_t{0u, 0u, 0u, 0u};
    if (p) {
#pragma unroll
      for (int s = 0; s < 4; ++s) x.f[s] = *reinterpret_cast<const u32x4_t*>(p + 8 * s);
    }
    return x;
  }
  template <int TN, int MT>
  __device__ __forceinline__ static void step(f32x4_t (&acc)[TN][MT], const W (&w)[TN], const X (&x)[MT]) {
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int t = 0; t < TN; ++t)
#pragma unroll
        for (int u = 0; u < MT; ++u)
          acc[t][u] = mma_bf16(__builtin_bit_cast(bf16x8_t, w[t].f[s]), __builtin_bit_cast(bf16x8_t, x[u].f[s]), acc[t][u]);
  }
};

template <> struct Fmt<WF32, float> {
  static constexpr int TILE = 8192;
  struct W { u32x4_t f[8]; };
  struct X { u32x4_t f[8]; };
  __device__ __forceinline__ static W load_w(const WMat& m, long tile, int lane) {
    W w;
    const char* p = static_cast<const char*>(m.data) + tile * TILE + lane * 16;
#pragma unroll
    for (int s = 0; s < 8; ++s) w.f[s] = *reinterpret_cast<const u32x4_t*>(p + s * 1024);
    return w;
  }
  __device__ __forceinline__ static X load_x(const float* p) {
    X x;
#pragma unroll
    for (int s = 0; s < 8; ++s) x.f[s] = u32x4_t{0u, 0u, 0u, 0u};
    if (p) {
#pragma unroll
      for (int s = 0; s < 8; ++s) x.f[s] = *reinterpret_cast<const u32x4_t*>(p + 4 * s);
    }
    return x;
  }
  template <int TN, int MT>
  __device__ __forceinline__ static void step(f32x4_t (&acc)[TN][MT], const W (&w)[TN], const X (&x)[MT]) {
#pragma unroll
    for (int s = 0; s < 8; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int t = 0; t < TN; ++t)
#pragma unroll
          for (int u = 0; u < MT; ++u)
            acc[t][u] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(w[t].f[s][i]), __uint_as_float(x[u].f[s][i]),
                                                             acc[t][u], 0, 0, 0);
  }
};

struct WMx4Lane {
  u32x4_t q;
  unsigned char s;
};
__device__ __forceinline__ WMx4Lane load_mx4(const WMat& m, long tile, int lane) {
  WMx4Lane w;
  w.q = *reinterpret_cast<const u32x4_t*>(static_cast<const char*>(m.data) + tile * 1024 + lane * 16);
  w.s = m.scales[tile * 64 + lane];
  return w;
}

template <> struct Fmt<WMx4, bf16_t> {
  using W = WMx4Lane;
  using X = Fmt<WBf16, bf16_t>::X;
  __device__ __forceinline__ static W load_w(const WMat& m, long tile, int lane) { return load_mx4(m, tile, lane); }
  __device__ __forceinline__ static X load_x(const bf16_t* p) { return Fmt<WBf16, bf16_t>::load_x(p); }
  template <int TN, int MT>
  __device__ __forceinline__ static void step(f32x4_t (&acc)[TN][MT], const W (&w)[TN], const X (&x)[MT]) {
#pragma unroll
    for (int t = 0; t < TN; ++t) {
      const float scale = __uint_as_float((unsigned)w[t].s << 23);
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const bf16x8_t a = mx4_frag(w[t].q[s], scale);
#pragma unroll
        for (int u = 0; u < MT; ++u) acc[t][u] = mma_bf16(a, __builtin_bit_cast(bf16x8_t, x[u].f[s]), acc[t][u]);
      }
    }
  }
};

template <> struct Fmt<WMx4, float> {
  using W = WMx4Lane;
  using X = Fmt<WF32, float>::X;
  __device__ __forceinline__ static W load_w(const WMat& m, long tile, int lane) { return load_mx4(m, tile, lane); }
  __device__ __forceinline__ static X load_x(const float* p) { return Fmt<WF32, float>::load_x(p); }
  template <int TN, int MT>
  __device__ __forceinline__ static void step(f32x4_t (&acc)[TN][MT], const W (&w)[TN], const X (&x)[MT]) {
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      bf16x8_t a[TN];
#pragma unroll
      for (int t = 0; t < TN; ++t) a[t] = mx4_frag(w[t].q[s], __uint_as_float((unsigned)w[t].s << 23));
#pragma unroll
      for (int u = 0; u < MT; ++u) {
        u32x4_t hi, mid, lo;
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          unsigned h[2], m[2], l[2];
#pragma unroll
          for (int e = 0; e < 2; ++e)
            split3(__uint_as_float(x[u].f[2 * s + (d >> 1)][2 * (d & 1) + e]), h[e], m[e], l[e]);
          hi[d] = (h[0] >> 16) | h[1];
          mid[d] = (m[0] >> 16) | m[1];
          lo[d] = (l[0] >> 16) | (l[1] & 0xffff0000u);
        }
        // the small parts first
#pragma unroll
        for (int t = 0; t < TN; ++t) acc[t][u] = mma_bf16(a[t], __builtin_bit_cast(bf16x8_t, lo), acc[t][u]);
#pragma unroll
        for (int t = 0; t < TN; ++t) acc[t][u] = mma_bf16(a[t], __builtin_bit_cast(bf16x8_t, mid), acc[t][u]);
#pragma unroll
        for (int t = 0; t < TN; ++t) acc[t][u] = mma_bf16(a[t], __builtin_bit_cast(bf16x8_t, hi), acc[t][u]);
      }
    }
  }
};
