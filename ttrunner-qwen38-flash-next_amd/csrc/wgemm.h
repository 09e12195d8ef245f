// Products of tiled weights (wtile.h) with many activation rows.
//
// A workgroup of WN x WM waves forms 16 TN WN weight rows x 16 TM WM activation
// rows. Both operands of one span of k go straight from memory into LDS, in a
// ring of S buffers: S - 1 spans are in flight or in use while one is multiplied,
// one barrier a span. Weights arrive in operand order; an activation row's 16-byte
// units are exchanged by an exclusive or with its number, so that the 16 rows of
// an operand read distinct banks. 4-bit weights become bf16 in the registers of
// the waves that multiply them. STREAM: the weights are read once or twice (few row
// tiles) and are not kept in the L2 before the activations.
#pragma once

#include "wtile.h"

// logical work item of a workgroup: each XCD (workgroups are dealt to the 8 in
// turn) takes a run of consecutive items, so that neighbours share its L2
__device__ __forceinline__ int xcd_run(int bid, int n) {
  const int x = bid % 8, q = n / 8, r = n % 8;
  return x * q + min(x, r) + bid / 8;
}

template <typename WF, typename T, int TN, int TM, int WN, int WM, int S, bool STREAM = false, int KS = 1>
struct SpanGemm {
  using F = Fmt<WF, T>;
  static constexpr int NW = WN * WM;
  static constexpr int BN = 16 * TN * WN, BM = 16 * TM * WM;
  static constexpr int ROW_B = F::SPAN * sizeof(T), UNITS = ROW_B / 16, VE = 16 / sizeof(T);
  static constexpr int RPL = 1024 / ROW_B;                     // rows of one wave-wide load
  static constexpr int XL = BM / RPL / NW;                     // activation loads of a wave, per span
  static constexpr int WL = TN * WN * F::SPAN_B / 1024 / NW;   // weight loads
  static constexpr int W_LOADS = WL + (F::SCALED ? 1 : 0);
  static constexpr int X_B = BM * ROW_B, W_B = TN * WN * F::SPAN_B, S_B = F::SCALED ? NW * 256 : 0;
  static constexpr int BUF = X_B + W_B + S_B, LDS_BYTES = KS * S * BUF;
  static_assert(XL * RPL * NW == BM && WL * 1024 * NW == W_B && TN <= 4 && XL > 0 && WL > 0, "loads of a wave");
  static_assert((KS - 1) * NW * TN * TM * 1024 <= LDS_BYTES, "the groups' sums take the ring's place");

  // where this lane's loads come from: activation rows (clamped into the matrix),
  // pieces of weights, and the scales of the wave's own row tiles
  struct Src {
    const T* x[XL];
    const char* w[WL];
    const uint8_t* s;
  };
  // rows(i): activation row i of the tile; tile(q): row tile q of TN WN, as the
  // bytes of its first k tile; scale(q): its scales'
  template <typename Rows, typename Tile, typename Scale>
  __device__ __forceinline__ static Src source(int wid, int lane, Rows rows, Tile tile, Scale scale) {
    Src r;
#pragma unroll
    for (int i = 0; i < XL; ++i) r.x[i] = rows((wid * XL + i) * RPL + lane / UNITS);
#pragma unroll
    for (int i = 0; i < WL; ++i) {
      const int at = (wid * WL + i) * 1024;
      r.w[i] = tile(at / F::SPAN_B) + at % F::SPAN_B + lane * 16;
    }
    if constexpr (F::SCALED) r.s = scale(wid / WM * TN + min(lane / 16, TN - 1)) + lane % 16 * 4;
    return r;
  }
  __device__ __forceinline__ static int swizzle(int row) { return UNITS >= 16 ? row & 15 : row >> 1 & 7; }

  __device__ __forceinline__ static void fetch(char* buf, const Src& src, int k, int rows, int j, int wid, int lane) {
#pragma unroll
    for (int i = 0; i < XL; ++i) {
      const int at = (wid * XL + i) * 1024, row = (wid * XL + i) * RPL + lane / UNITS;
      const int unit = (lane % UNITS) ^ swizzle(row);
      // units past k (a last span that is partly past it) are zeros: whatever lies
      // behind a row would meet weights of zero, but infinities make NaN of those
      const int kk = j * F::SPAN + unit * VE;
      const void* p = kk < k ? static_cast<const void*>(src.x[i] + kk) : g_zero_unit;
      if (row < rows) lds_load16(p, buf + at);                // (rows past the last multiply what lies there, unread)
    }
#pragma unroll
    for (int i = 0; i < WL; ++i) {
      const char* p = src.w[i] + (long)j * F::SPAN_B;
      char* to = buf + X_B + (wid * WL + i) * 1024;
      if constexpr (STREAM) lds_load16_stream(p, to);
      else lds_load16(p, to);
    }
    if constexpr (F::SCALED) lds_load4(src.s + (long)j * 64, buf + X_B + W_B + wid * 256);
  }
  __device__ __forceinline__ static void run(f32x4_t (&acc)[TN][TM], char* lds, const Src& src, int k, int rows) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wid = KS > 1 ? wave % NW : wave, part = KS > 1 ? wave / NW : 0;
    if constexpr (KS > 1) lds += part * (S * BUF);
    const int g4 = lane >> 4, row0 = (wid % WM) * 16 * TM + (lane & 15), wn = wid / WM;
    // of this group, and of the first, which has as many as any
    const int all = (k + F::SPAN - 1) / F::SPAN, spans = (all - part + KS - 1) / KS, most = (all + KS - 1) / KS;
#pragma unroll
    for (int j = 0; j < S - 1; ++j)
      if (j < spans) fetch(lds + j * BUF, src, k, rows, j * KS + part, wid, lane);
    for (int j0 = 0; j0 < most; j0 += S) {
#pragma unroll
      for (int b = 0; b < S; ++b) {
        const int j = j0 + b;
        if (j >= most) break;
        // this wave's part of span j is in LDS when at most the S - 2 later
        // spans' loads are outstanding (loads return in order; those of
        // activations do not count, a wave whose rows lie past the last makes
        // none), its reads of the buffer that is filled next when none of LDS is
        if (j + S - 2 < spans)
          wave_loads_barrier<(S - 2) * W_LOADS>();
        else
          wave_loads_barrier<0>();
        if (j + S - 1 < spans) fetch(lds + (b + S - 1) % S * BUF, src, k, rows, (j + S - 1) * KS + part, wid, lane);
        if (KS > 1 && j >= spans) continue;
        const char* buf = lds + b * BUF;
        typename F::W w[TN];
#pragma unroll
        for (int t = 0; t < TN; ++t)
          F::span_w(w[t], buf + X_B + (wn * TN + t) * F::SPAN_B, buf + X_B + W_B + wid * 256 + t * 64, lane);
        f32x4_t sum[TN][TM];
        if constexpr (sizeof(T) == 4) clear(sum);
        // a piece's activations are read while the one before is multiplied
        Piece<T> x[2][TM];
#pragma unroll
        for (int u = 0; u < TM; ++u) x[0][u] = lds_piece<T>(buf + (row0 + 16 * u) * ROW_B, F::unit(g4, 0), swizzle(row0));
#pragma unroll
        for (int s = 0; s < F::SPAN / 32; ++s) {
          if (s + 1 < F::SPAN / 32) {
#pragma unroll
            for (int u = 0; u < TM; ++u) x[(s + 1) & 1][u] = lds_piece<T>(buf + (row0 + 16 * u) * ROW_B, F::unit(g4, s + 1), swizzle(row0));
          }
          // float sums in two levels: a span, then the spans
          if constexpr (sizeof(T) == 4) F::step(sum, w, s, x[s & 1]);
          else F::step(acc, w, s, x[s & 1]);
        }
        if constexpr (sizeof(T) == 4) {
#pragma unroll
          for (int t = 0; t < TN; ++t)
#pragma unroll
            for (int u = 0; u < TM; ++u) acc[t][u] += sum[t][u];
        }
      }
    }
  }
  // The groups' sums, in their order, in the first group's waves; false in the others,
  // which have nothing left to do.
  __device__ __forceinline__ static bool join(f32x4_t (&acc)[TN][TM], char* lds) {
    if constexpr (KS > 1) {
      const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
      f32x4_t* s = reinterpret_cast<f32x4_t*>(lds) + lane;
      __syncthreads();
      if (wave >= NW) {
#pragma unroll
        for (int t = 0; t < TN; ++t)
#pragma unroll
          for (int u = 0; u < TM; ++u) s[(((wave - NW) * TN + t) * TM + u) * 64] = acc[t][u];
      }
      __syncthreads();
      if (wave >= NW) return false;
#pragma unroll
      for (int p = 0; p < KS - 1; ++p)
#pragma unroll
        for (int t = 0; t < TN; ++t)
#pragma unroll
          for (int u = 0; u < TM; ++u) acc[t][u] += s[(((p * NW + wave) * TN + t) * TM + u) * 64];
    }
    return true;
  }
};
