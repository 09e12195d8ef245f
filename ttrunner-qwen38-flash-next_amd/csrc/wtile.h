// Weight tiles in the matrix cores' operand order, and their products with
// row-major activation rows. Shared by the 4-bit projections (mx4.hip) and the
// mixture-of-experts layer (moe.hip).
//
// A tile is 16 weight rows x 128 k; lane l of a wave holds row l % 16, four pieces
// of 8 consecutive k, so that every load of weights is whole lines (1 KB a wave)
// however k is split over waves.
//   MX4    piece s of lane l: k 32 (l / 16) + 8 s .. + 7. The lane's 32 k are one
//          microscaling block with its one scale: a tile of codes is one 16-byte
//          load a lane (dword s: piece s, the first element in the low nibble),
//          its scales one byte a lane in an array of their own
//   bf16   piece s: k 32 s + 8 (l / 16) .. + 7; tiles [4 pieces][64 lanes][16 B]
//   float  the same k; tiles [4 pieces][2 halves][64 lanes][16 B]
// in [matrix][row tile][k tile]. Rows past n and k past the matrix hold zeros
// (scale byte 0).
//
// Products: bf16 16x16x32 MFMAs accumulate in float. 4-bit weights times a power
// of two are exact in bf16 (two significant bits, and bf16's exponents and
// subnormals reach every scale), so they lose nothing on the way in; float
// activations meet them as three bf16 parts of 8 bits each, whose sum is the
// float exactly, but for bits below 2^-133, bf16's smallest. Float weights take 16x16x4 float MFMAs.
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

// The activations of one piece: 8 consecutive k of a row
template <typename T> struct Piece;
template <> struct Piece<bf16_t> {
  u32x4_t f;
  __device__ __forceinline__ static Piece load(const bf16_t* p) { return {*reinterpret_cast<const u32x4_t*>(p)}; }
  __device__ __forceinline__ static Piece zero() { return {u32x4_t{0u, 0u, 0u, 0u}}; }
};
template <> struct Piece<float> {
  u32x4_t f[2];
  __device__ __forceinline__ static Piece load(const float* p) {
    return {{*reinterpret_cast<const u32x4_t*>(p), *reinterpret_cast<const u32x4_t*>(p + 4)}};
  }
  __device__ __forceinline__ static Piece zero() { return {{u32x4_t{0u, 0u, 0u, 0u}, u32x4_t{0u, 0u, 0u, 0u}}}; }
};

// Floats as three bf16 parts of 8 significant bits each, cut and not rounded: the
// parts add up to the float (bits below 2^-133 are cut off). Infinities and NaN sit in the first part alone.
__device__ __forceinline__ void split3(const Piece<float>& x, u32x4_t& hi, u32x4_t& mid, u32x4_t& lo) {
  constexpr unsigned UPPER = 0x07060302u;                    // the upper halves of two words
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    unsigned b[2], r[2], q[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float v = __builtin_canonicalizef(__uint_as_float(x.f[d >> 1][2 * (d & 1) + e]));   // NaN: its bits in the upper half
      b[e] = __float_as_uint(v);
      const float m = __builtin_amdgcn_classf(v, 0x207) ? 0.f : v - __uint_as_float(b[e] & 0xffff0000u);
      r[e] = __float_as_uint(m);
      q[e] = __float_as_uint(m - __uint_as_float(r[e] & 0xffff0000u));
    }
    hi[d] = __builtin_amdgcn_perm(b[1], b[0], UPPER);
    mid[d] = __builtin_amdgcn_perm(r[1], r[0], UPPER);
    lo[d] = __builtin_amdgcn_perm(q[1], q[0], UPPER);
  }
}

// One format of weights against one type of activations.
//   TILE     bytes of a tile (its codes), SPAN the k of one stage of wgemm.h and
//            SPAN_B the stage's bytes of a row tile
//   unit     which piece of a row's k tile lane group g4 multiplies as its piece s
//   W        a lane's part of a row tile over a span: loaded from memory or LDS
//   step     acc += W X over piece s; lane: weight rows 4 (l / 16) + i, activation
//            row l % 16
template <typename WF, typename T> struct Fmt;

template <> struct Fmt<WBf16, bf16_t> {
  static constexpr int TILE = 4096, SPAN = 64, SPAN_B = 2048;
  static constexpr bool SCALED = false;
  struct W { u32x4_t f[4]; };
  __device__ __forceinline__ static int unit(int g4, int s) { return 4 * s + g4; }
  __device__ __forceinline__ static W load_w(const WMat& m, long tile, int lane) {
    W w;
    const char* p = static_cast<const char*>(m.data) + tile * TILE + lane * 16;
#pragma unroll
    for (int s = 0; s < 4; ++s) w.f[s] = *reinterpret_cast<const u32x4_t*>(p + s * 1024);
    return w;
  }
  __device__ __forceinline__ static void span_w(W& w, const char* lds, const char*, int lane) {
#pragma unroll
    for (int s = 0; s < 2; ++s) w.f[s] = *reinterpret_cast<const u32x4_t*>(lds + s * 1024 + lane * 16);
  }
  template <int TN, int MT>
  __device__ __forceinline__ static void step(f32x4_t (&acc)[TN][MT], const W (&w)[TN], int s, const Piece<bf16_t> (&x)[MT]) {
#pragma unroll
    for (int t = 0; t < TN; ++t)
#pragma unroll
      for (int u = 0; u < MT; ++u)
        acc[t][u] = mma_bf16(__builtin_bit_cast(bf16x8_t, w[t].f[s]), __builtin_bit_cast(bf16x8_t, x[u].f), acc[t][u]);
  }
};

template <> struct Fmt<WF32, float> {
  static constexpr int TILE = 8192, SPAN = 64, SPAN_B = 4096;
  static constexpr bool SCALED = false;
  struct W { u32x4_t f[8]; };
  __device__ __forceinline__ static int unit(int g4, int s) { return 4 * s + g4; }
  __device__ __forceinline__ static W load_w(const WMat& m, long tile, int lane) {
    W w;
    const char* p = static_cast<const char*>(m.data) + tile * TILE + lane * 16;
#pragma unroll
    for (int s = 0; s < 8; ++s) w.f[s] = *reinterpret_cast<const u32x4_t*>(p + s * 1024);
    return w;
  }
  __device__ __forceinline__ static void span_w(W& w, const char* lds, const char*, int lane) {
#pragma unroll
    for (int s = 0; s < 4; ++s) w.f[s] = *reinterpret_cast<const u32x4_t*>(lds + s * 1024 + lane * 16);
  }
  template <int TN, int MT>
  __device__ __forceinline__ static void step(f32x4_t (&acc)[TN][MT], const W (&w)[TN], int s, const Piece<float> (&x)[MT]) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int t = 0; t < TN; ++t)
#pragma unroll
          for (int u = 0; u < MT; ++u)
            acc[t][u] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(w[t].f[2 * s + h][i]),
                                                             __uint_as_float(x[u].f[h][i]), acc[t][u], 0, 0, 0);
  }
};

// 4-bit weights, whatever the activations
struct FmtMx4 {
  static constexpr int TILE = 1024, SPAN = 128, SPAN_B = 1024;
  static constexpr bool SCALED = true;
  struct W {
    u32x4_t q;
    unsigned char s;
  };
  __device__ __forceinline__ static int unit(int g4, int s) { return 4 * g4 + s; }
  __device__ __forceinline__ static W load_w(const WMat& m, long tile, int lane) {
    W w;
    w.q = *reinterpret_cast<const u32x4_t*>(static_cast<const char*>(m.data) + tile * 1024 + lane * 16);
    w.s = m.scales[tile * 64 + lane];
    return w;
  }
  __device__ __forceinline__ static void span_w(W& w, const char* lds, const char* scales, int lane) {
    w.q = *reinterpret_cast<const u32x4_t*>(lds + lane * 16);
    w.s = (unsigned char)scales[lane];
  }
  __device__ __forceinline__ static bf16x8_t frag(const W& w, int s) {
    return mx4_frag(w.q[s], __uint_as_float((unsigned)w.s << 23));
  }
};

template <> struct Fmt<WMx4, bf16_t> : FmtMx4 {
  template <int TN, int MT>
  __device__ __forceinline__ static void step(f32x4_t (&acc)[TN][MT], const W (&w)[TN], int s, const Piece<bf16_t> (&x)[MT]) {
#pragma unroll
    for (int t = 0; t < TN; ++t) {
      const bf16x8_t a = frag(w[t], s);
#pragma unroll
      for (int u = 0; u < MT; ++u) acc[t][u] = mma_bf16(a, __builtin_bit_cast(bf16x8_t, x[u].f), acc[t][u]);
    }
  }
};

template <> struct Fmt<WMx4, float> : FmtMx4 {
  template <int TN, int MT>
  __device__ __forceinline__ static void step(f32x4_t (&acc)[TN][MT], const W (&w)[TN], int s, const Piece<float> (&x)[MT]) {
    bf16x8_t a[TN];
#pragma unroll
    for (int t = 0; t < TN; ++t) a[t] = frag(w[t], s);
#pragma unroll
    for (int u = 0; u < MT; ++u) {
      u32x4_t hi, mid, lo;
      split3(x[u], hi, mid, lo);
      // the small parts first
#pragma unroll
      for (int t = 0; t < TN; ++t) acc[t][u] = mma_bf16(a[t], __builtin_bit_cast(bf16x8_t, lo), acc[t][u]);
#pragma unroll
      for (int t = 0; t < TN; ++t) acc[t][u] = mma_bf16(a[t], __builtin_bit_cast(bf16x8_t, mid), acc[t][u]);
#pragma unroll
      for (int t = 0; t < TN; ++t) acc[t][u] = mma_bf16(a[t], __builtin_bit_cast(bf16x8_t, hi), acc[t][u]);
    }
  }
};

// A lane's part of 16 activation rows over k tile ks, from memory: zeros past k
template <typename F, typename T> struct Acts {
  Piece<T> p[4];
  __device__ __forceinline__ void load(const T* row, int ks, int k, int g4) {
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int at = ks * WT_K + 8 * F::unit(g4, s);
      p[s] = Piece<T>::zero();
      if (at < k) p[s] = Piece<T>::load(row + at);
    }
  }
};
template <typename F, typename T, int TN, int MT>
__device__ __forceinline__ void step_tile(f32x4_t (&acc)[TN][MT], const typename F::W (&w)[TN], const Acts<F, T> (&x)[MT]) {
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    Piece<T> xs[MT];
#pragma unroll
    for (int u = 0; u < MT; ++u) xs[u] = x[u].p[s];
    F::step(acc, w, s, xs);
  }
}
template <int TN, int MT> __device__ __forceinline__ void clear(f32x4_t (&acc)[TN][MT]) {
#pragma unroll
  for (int t = 0; t < TN; ++t)
#pragma unroll
    for (int u = 0; u < MT; ++u) acc[t][u] = f32x4_t{0.f, 0.f, 0.f, 0.f};
}

// ---------------------------------------------------------------------------
// Rows in LDS, filled straight from memory
// ---------------------------------------------------------------------------

// 16 or 4 bytes a lane from memory to lds + lane * 16 or 4 (lds uniform)
__device__ __forceinline__ void lds_load16(const void* p, char* lds) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)p,
                                   (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
}
// (the non-temporal form: not kept in the L2 before what is read more often)
__device__ __forceinline__ void lds_load16_stream(const void* p, char* lds) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)p,
                                   (__attribute__((address_space(3))) void*)lds, 16, 0, 2);
}
__device__ __forceinline__ void lds_load4(const void* p, char* lds) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)p,
                                   (__attribute__((address_space(3))) void*)lds, 4, 0, 0);
}

static __device__ const u32x4_t g_zero_unit[1] = {{0u, 0u, 0u, 0u}};

// A barrier of the workgroup that leaves OUT of this wave's memory loads in flight
// (__syncthreads waits for all): loads return in order, so all but the youngest
// OUT are in LDS, and this wave's own LDS reads are done.
template <int OUT> __device__ __forceinline__ void wave_loads_barrier() {
  static_assert(OUT < 64, "vmcnt has 6 bits");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"i"(OUT) : "memory");
}

// Piece p (8 k) of a row in LDS whose 16-byte units sit at their number exclusive
// or `swz`
template <typename T> __device__ __forceinline__ Piece<T> lds_piece(const char* row, int p, int swz) {
  if constexpr (sizeof(T) == 2) {
    return {*reinterpret_cast<const u32x4_t*>(row + ((p ^ swz) * 16))};
  } else {
    return {{*reinterpret_cast<const u32x4_t*>(row + (((2 * p) ^ swz) * 16)),
             *reinterpret_cast<const u32x4_t*>(row + (((2 * p + 1) ^ swz) * 16))}};
  }
}

// one piece of 16 rows against one of 16 others
__device__ __forceinline__ f32x4_t mma_piece(const Piece<bf16_t>& a, const Piece<bf16_t>& b, f32x4_t c) {
  return mma_bf16(__builtin_bit_cast(bf16x8_t, a.f), __builtin_bit_cast(bf16x8_t, b.f), c);
}
__device__ __forceinline__ f32x4_t mma_piece(const Piece<float>& a, const Piece<float>& b, f32x4_t c) {
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.f[h][i]), __uint_as_float(b.f[h][i]), c, 0, 0, 0);
  return c;
}
