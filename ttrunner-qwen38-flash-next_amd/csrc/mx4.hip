// Microscaled 4-bit weights (OCP MX: E2M1 elements, blocks of 32 along k with one
// E8M0 scale), gfx950: quantisation, reading back, the layout of a checkpoint's
// codes, and the product with activation rows.
//
// A block's scale is 2^s, s = max(floor(log2 max|w|) - 2, -127), so the largest
// magnitude lies in [4, 8) scales; an element is w / 2^s to the nearest of
// 0, .5, 1, 1.5, 2, 3, 4, 6 (ties to the even code), 6 beyond. The hardware
// conversion (v_cvt_scalef32_pk_fp4_f32) does just that for every finite input,
// subnormals included, so the division is exact. A block that holds a NaN or an
// infinity becomes NaN as a whole (scale byte 255). A block of zeros has scale
// byte 0.
//
// Weights are kept in the operand order of wtile.h, 17 bytes for 32 weights.
#include "qwen4mix_internal.h"
#include "wgemm.h"

namespace {

constexpr int MX_NT = 256;

struct MxGeom {
  int n, k;          // a matrix
  int rt, kt;        // its tiles
  long tiles;        // of all matrices
};

MxGeom mx_geom(int mats, int n, int k) {
  MxGeom g = {n, k, wt_row_tiles(n), wt_k_tiles(k), 0};
  g.tiles = (long)mats * g.rt * g.kt;
  return g;
}

// where a lane's block lies: its matrix row (of all matrices) and first column
__device__ __forceinline__ bool block_of(const MxGeom& g, long tile, int lane, long& row, int& k0) {
  const int ks = (int)(tile % g.kt);
  const long rest = tile / g.kt;
  const int r = (int)(rest % g.rt) * WT_ROWS + (lane & 15);
  k0 = ks * WT_K + (lane >> 4) * MX_BLOCK;
  row = rest / g.rt * g.n + r;
  return r < g.n && k0 < g.k;
}

__device__ __forceinline__ void load32(const float* p, float (&v)[32]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float4 u = *reinterpret_cast<const float4*>(p + 4 * i);
    v[4 * i] = u.x; v[4 * i + 1] = u.y; v[4 * i + 2] = u.z; v[4 * i + 3] = u.w;
  }
}
__device__ __forceinline__ void load32(const bf16_t* p, float (&v)[32]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint4 u = *reinterpret_cast<const uint4*>(p + 8 * i);
    const unsigned d[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[8 * i + 2 * j] = __uint_as_float(d[j] << 16);
      v[8 * i + 2 * j + 1] = __uint_as_float(d[j] & 0xffff0000u);
    }
  }
}

// One wave per tile, one lane per block: its 32 weights in whole 16-byte loads, the
// largest magnitude without another lane, codes in operand order in one store of the
// wave. A stream: 105 M floats (478 MB) in 107 us, 8.4 M bf16 in 5.4 us.
template <typename T>
__global__ __launch_bounds__(MX_NT) void mx4_quantize_kernel(MxGeom g, const T* w, uint8_t* codes, uint8_t* scales) {
  const int lane = threadIdx.x & 63;
  const long tile = (long)blockIdx.x * (MX_NT / 64) + (threadIdx.x >> 6);
  if (tile >= g.tiles) return;
  long row;
  int k0;
  u32x4_t q = {0u, 0u, 0u, 0u};
  unsigned s = 0;
  if (block_of(g, tile, lane, row, k0)) {
    float v[32];
    load32(w + row * g.k + k0, v);
    unsigned amax = 0;                                     // magnitudes order as their bits do, NaN above all
#pragma unroll
    for (int i = 0; i < 32; ++i) amax = max(amax, __float_as_uint(v[i]) & 0x7fffffffu);
    if (amax >= 0x7f800000u) {
      s = 255u;
    } else {
      s = (unsigned)max((int)(amax >> 23) - 2, 0);
      const float scale = __uint_as_float(s << 23);
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        unsigned c = 0;
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[8 * d], v[8 * d + 1], scale, 0);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[8 * d + 2], v[8 * d + 3], scale, 1);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[8 * d + 4], v[8 * d + 5], scale, 2);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[8 * d + 6], v[8 * d + 7], scale, 3);
        q[d] = c;
      }
    }
  }
  *reinterpret_cast<u32x4_t*>(codes + tile * 1024 + lane * 16) = q;
  scales[tile * 64 + lane] = (uint8_t)s;
}

// A lane writes 16 bytes of the output, 256 or 512 contiguous bytes a row (a lane
// per block, 64 or 128 bytes apart, wrote 52 M bf16 weights at 3.4 TB/s). 105 M
// floats (478 MB) take 86 us.
template <typename T>
__global__ __launch_bounds__(MX_NT) void mx4_dequantize_kernel(MxGeom g, const uint8_t* codes, const uint8_t* scales,
                                                              T* out) {
  constexpr int VE = 16 / sizeof(T), UNITS = WT_K / VE, RPS = 64 / UNITS;   // rows of one wave-wide store
  const int lane = threadIdx.x & 63;
  const long tile = (long)blockIdx.x * (MX_NT / 64) + (threadIdx.x >> 6);
  if (tile >= g.tiles) return;
  const int ks = (int)(tile % g.kt);
  const long rest = tile / g.kt;
  const int u = lane % UNITS, k0 = ks * WT_K + u * VE, g4 = u * VE / MX_BLOCK;
  const int r0 = (int)(rest % g.rt) * WT_ROWS;
  unsigned q[WT_ROWS / RPS];
  unsigned char s[WT_ROWS / RPS];
#pragma unroll
  for (int i = 0; i < WT_ROWS / RPS; ++i) {
    const int slot = g4 * 16 + i * RPS + lane / UNITS;
    // the dword with this unit's codes: 8 of them (all of it, or a half)
    q[i] = *reinterpret_cast<const unsigned*>(codes + tile * 1024 + slot * 16 + u * VE % MX_BLOCK / 8 * 4);
    s[i] = scales[tile * 64 + slot];
  }
#pragma unroll
  for (int i = 0; i < WT_ROWS / RPS; ++i) {
    const int r = r0 + i * RPS + lane / UNITS;
    if (r >= g.n || k0 >= g.k) continue;
    const float scale = __uint_as_float((unsigned)s[i] << 23);
    T* p = out + (rest / g.rt * g.n + r) * g.k + k0;
    if constexpr (sizeof(T) == 2) {
      *reinterpret_cast<uint4*>(p) = __builtin_bit_cast(uint4, mx4_frag(q[i], scale));
    } else {
      const unsigned h = u & 1 ? q[i] >> 16 : q[i];
      const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(h, scale, 0);
      const auto b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(h, scale, 1);
      *reinterpret_cast<float4*>(p) = make_float4(a[0], a[1], b[0], b[1]);
    }
  }
}

// between the plain order (codes [rows, k / 2], scales [rows, k / 32]) and tiles
template <bool TO_TILES>
__global__ __launch_bounds__(MX_NT) void mx4_layout_kernel(MxGeom g, uint8_t* codes, uint8_t* scales, uint8_t* plain_codes,
                                                          uint8_t* plain_scales) {
  const int lane = threadIdx.x & 63;
  const long tile = (long)blockIdx.x * (MX_NT / 64) + (threadIdx.x >> 6);
  if (tile >= g.tiles) return;
  long row;
  int k0;
  const bool in = block_of(g, tile, lane, row, k0);
  uint4* tc = reinterpret_cast<uint4*>(codes + tile * 1024 + lane * 16);
  uint8_t* ts = scales + tile * 64 + lane;
  const long b = in ? row * (g.k / MX_BLOCK) + k0 / MX_BLOCK : 0;
  if constexpr (TO_TILES) {
    *tc = in ? *reinterpret_cast<const uint4*>(plain_codes + b * 16) : make_uint4(0u, 0u, 0u, 0u);
    *ts = in ? plain_scales[b] : (uint8_t)0;
  } else if (in) {
    *reinterpret_cast<uint4*>(plain_codes + b * 16) = *tc;
    plain_scales[b] = *ts;
  }
}

// ---------------------------------------------------------------------------
// y[m][n] = sum_k W[n][k] x[m][k] for a few activation rows: a stream over the
// weights. A workgroup takes TN row tiles against a tile of 16 activation rows, its
// waves split the k tiles, the partial results meet in LDS. Every weight is loaded once per 16 rows. A wave's activations go through
// its own part of LDS: straight from memory their operand would take each lane of a
// load from another row than its neighbour, and such a load costs a cycle a lane
// (bf16, 12352 x 2048: 16 rows 7.4 us so, 5.7 through LDS; 1 row 5.0 and 5.2).
template <typename T>
struct Mx4LinearArgs {
  WMat w;
  const T* x;
  long ldx;
  int m, n, k, rt, kt;
  int n_seg;
  int seg_end[QM_GEMV_MAX_SEG];
  T* seg_out[QM_GEMV_MAX_SEG];
};

// outputs n .. n + 3 of row m
template <typename T>
__device__ __forceinline__ void store4(const Mx4LinearArgs<T>& A, int m, int n, f32x4_t v) {
  if (m >= A.m || n >= A.n) return;
  int s = 0, start = 0;
  while (s + 1 < A.n_seg && n >= A.seg_end[s]) { start = A.seg_end[s]; ++s; }
  const int n_s = A.seg_end[s] - start;
  T* o = A.seg_out[s] + (long)m * n_s + (n - start);
  if (n + 4 <= A.seg_end[s] && (reinterpret_cast<uintptr_t>(o) & (4 * sizeof(T) - 1)) == 0) {
    store_act4(o, v);
    return;
  }
  for (int i = 0; i < 4 && n + i < A.n; ++i) {
    while (s + 1 < A.n_seg && n + i >= A.seg_end[s]) { start = A.seg_end[s]; ++s; }
    Act<T>::store(A.seg_out[s], (long)m * (A.seg_end[s] - start) + (n + i - start), v[i]);
  }
}

template <typename T, int TN, int NW>
__global__ __launch_bounds__(64 * NW) void mx4_rows_kernel(Mx4LinearArgs<T> A) {
  using F = Fmt<WMx4, T>;
  constexpr int ROW_B = WT_K * sizeof(T), UNITS = ROW_B / 16, VE = 16 / sizeof(T), RPL = 1024 / ROW_B;
  constexpr int X_B = 16 * ROW_B;
  __shared__ __attribute__((aligned(16))) char s_buf[NW * (X_B > TN * 1024 ? X_B : TN * 1024)];
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g4 = lane >> 4, r16 = lane & 15;
  const int t0 = blockIdx.x * TN, m0 = blockIdx.y * 16, rows = min(16, A.m - m0);
  char* s_x = s_buf + wid * X_B;                             // 16 rows, units exchanged as in wgemm.h
  f32x4_t acc[TN][1];
  clear(acc);
  for (int ks = wid; ks < A.kt; ks += NW) {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");       // the rows before are read
#pragma unroll
    for (int q = 0; q < 16 / RPL; ++q) {
      if (q * RPL >= rows) continue;                         // (rows past the last multiply what lies there, unread)
      const int row = q * RPL + lane / UNITS, k = ks * WT_K + ((lane % UNITS) ^ row) * VE;
      const T* src = A.x + (long)min(m0 + row, A.m - 1) * A.ldx + k;
      lds_load16(k < A.k ? static_cast<const void*>(src) : g_zero_unit, s_x + q * 1024);
    }
    typename F::W w[TN];
    Acts<F, T> x[1];
#pragma unroll
    for (int t = 0; t < TN; ++t) w[t] = F::load_w(A.w, (long)min(t0 + t, A.rt - 1) * A.kt + ks, lane);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");         // this wave's rows are in LDS
#pragma unroll
    for (int s = 0; s < 4; ++s) x[0].p[s] = lds_piece<T>(s_x + r16 * ROW_B, F::unit(g4, s), r16);
    step_tile<F, T>(acc, w, x);
  }
  __syncthreads();                                           // the sums take the rows' place
  f32x4_t (*s_red)[TN][64] = reinterpret_cast<f32x4_t (*)[TN][64]>(s_buf);
#pragma unroll
  for (int t = 0; t < TN; ++t) s_red[wid][t][lane] = acc[t][0];
  __syncthreads();
  for (int r = wid; r < TN; r += NW) {
    f32x4_t v = s_red[0][r][lane];
#pragma unroll
    for (int w = 1; w < NW; ++w) v += s_red[w][r][lane];
    store4(A, m0 + r16, (t0 + r) * 16 + 4 * g4, v);
  }
}

template <typename T, int TN, int NW>
int launch_rows(const Mx4LinearArgs<T>& A, hipStream_t stream) {
  hipLaunchKernelGGL((mx4_rows_kernel<T, TN, NW>), dim3((A.rt + TN - 1) / TN, (A.m + 15) / 16), dim3(64 * NW), 0, stream, A);
  QM_CHECK_LAUNCH();
  return QM_OK;
}

// Many activation rows: a workgroup per 16 TN WN weight rows x 16 TM WM
// activation rows (wgemm.h), the activation rows' tiles of one range of weights
// side by side on an XCD.
template <typename T, int TN, int TM, int WN, int WM, int S, int KS>
__global__ __launch_bounds__(64 * WN * WM * KS, 2) void mx4_gemm_kernel(Mx4LinearArgs<T> A) {
  using G = SpanGemm<WMx4, T, TN, TM, WN, WM, S, false, KS>;
  extern __shared__ __attribute__((aligned(16))) char s_buf[];
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % (WN * WM);
  const int mt = (A.m + G::BM - 1) / G::BM;
  const int item = xcd_run(blockIdx.x, gridDim.x);
  const int m0 = item % mt * G::BM, t0 = item / mt * WN * TN;
  auto first = [&](int q) { return (long)min(t0 + q, A.rt - 1) * A.kt; };
  const typename G::Src src = G::source(
      wid, lane, [&](int i) { return A.x + (long)min(m0 + i, A.m - 1) * A.ldx; },
      [&](int q) { return static_cast<const char*>(A.w.data) + first(q) * G::F::TILE; },
      [&](int q) { return A.w.scales + first(q) * 64; });
  f32x4_t acc[TN][TM];
  clear(acc);
  G::run(acc, s_buf, src, A.k, A.m - m0);
  if (!G::join(acc, s_buf)) return;
#pragma unroll
  for (int t = 0; t < TN; ++t)
#pragma unroll
    for (int u = 0; u < TM; ++u)
      store4(A, m0 + (wid % WM) * 16 * TM + 16 * u + (lane & 15), (t0 + wid / WM * TN + t) * 16 + 4 * (lane >> 4), acc[t][u]);
}

template <typename T, int TN, int TM, int WN, int WM, int S, int KS = 1>
int launch_gemm(const Mx4LinearArgs<T>& A, hipStream_t stream) {
  using G = SpanGemm<WMx4, T, TN, TM, WN, WM, S, false, KS>;
  constexpr int NT = 64 * WN * WM * KS;
  const long nb = (long)((A.rt + TN * WN - 1) / (TN * WN)) * ((A.m + G::BM - 1) / G::BM);
  if (nb > 0x7fffffffL / NT) return qm_fail(QM_ERR_UNSUPPORTED, "qm_mx4_linear: too many tiles for one launch");
  static std::atomic<uint64_t> allowed{0};
  const int rc = qm_allow_lds(reinterpret_cast<const void*>(mx4_gemm_kernel<T, TN, TM, WN, WM, S, KS>), G::LDS_BYTES, allowed);
  if (rc) return rc;
  hipLaunchKernelGGL((mx4_gemm_kernel<T, TN, TM, WN, WM, S, KS>), dim3((unsigned)nb), dim3(NT), G::LDS_BYTES, stream, A);
  QM_CHECK_LAUNCH();
  return QM_OK;
}

// The kernel for m rows (weights from memory, graph replays, us a call). g(TN) is the
// number of workgroups of the few-row kernel with TN row tiles each.
//   few rows   up to one workgroup a CU, k is split over 16 waves (2048 x 4096, 64
//     rows: 16 waves 5.2, 8 waves 5.5); more of them keep 8 (12352 x 2048, one row:
//     5.1 against 6.2). Of bf16 a workgroup takes one row tile while there is one a
//     CU (2048 x 4096, 16 rows: 1, 2, 4 tiles 4.5 / 5.3 / 6.7; 64 rows 7.5 / 5.6 /
//     6.9), two while there are two (12352 x 2048, 16 rows: 7.0 / 5.6 / 5.7), else
//     four (256 rows of 2048 x 4096: - / 11.8 / 10.5). Floats are cut into parts by
//     every workgroup, so as many tiles as leave one a CU share them, up to eight
//     (12352 x 2048, 1 row: 1, 2, 4, 8 tiles 12.5 / 8.7 / 7.6 / 10; 32 rows 22 / 16 /
//     12.0 / 11.5).
//   bf16, more than 512 of them with four tiles each   wgemm.h, its tile by how many
//     workgroups it makes: 128 x 32 with k over four groups of waves up to one a CU,
//     over two up to 640; then 256 x 32 up to 768, then 256 x 64. Few-row kernel /
//     four groups / two / 256 x 32 / 256 x 64, and the number of 128 x 32 tiles: 12352
//     x 2048: 32 rows (97) 8.4 / 9.2 / 9.9 / 13.7 / 18.1, 48 rows (194) 10.5 / 9.4 /
//     9.9 / 13.4 / 19.6, 128 rows (388) 20.1 / 16.7 / 13.0 / 14.5 / 20.6, 256 rows
//     (776) - / 30.5 / 22.9 / 20.0 / 21.2, 512 rows (1552) - / 52 / 40 / 37 / 33.5; 9856
//     x 2048: 400 rows (1001) 39 / 31 / 23.7 / 21.1 / 29.7; 2048 x 4096: 256 rows (128)
//     10.4 / 13.4 / 15.4 / 23.0 / 35, 400 rows (208) 16.6 / 13.6 / 15.3 / 19.7 / 35
//     Wide weights, whose few rows make as many workgroups: up to 8 rows stay with the
//     few-row kernel, up to 32 with tiles of 32 (few-row / 256 x 32 / 256 x 64, x 2048:
//     65536, 1 row 16.8 / 19.3 / 20.7; 98304, 1 row 23.2 / 23.9 / 33.2, 8 rows 24.8 /
//     23.9 / 32.9, 16 rows 26.6 / 24.0 / 34.5; 151936: 1 row 33.1 / 35.6 / 47.4, 8 rows 34.9 /
//     35.9 / 49.7, 16 rows 38.6 / 36.6 / 52.1, 32 rows 60 / 40.8 / 56.8; 262144: 1 row
//     51.7 / 61.8 / 63.3, 8 rows 54.0 / 63.1 / 66.0, 32 rows 120 / 66.2 / 73.0)
//   float   256 x 32 tiles from 512 workgroups on (2000 rows of 9856 x 2048: 283
//     against 328; 256 of 12352 x 2048, 392 of them: 60 against 63), but for up to 16
//     rows of a wide weight, which keep four row tiles a workgroup (four / eight / 256 x
//     32, x 2048: 65536, 1 row 22.1 / 23.9 / 41; 151936: 1 row 49 / 53 / 91, 16 rows 53 /
//     56 / 96, 17 rows 89 / 100 / 97; 262144: 1 row 76 / 83 / 119, 17 rows 148 / 162 / 130)
template <typename T>
int run_linear(const Mx4LinearArgs<T>& A, hipStream_t stream) {
  auto groups = [&A](int bn, int bm) { return (long)((A.rt * 16 + bn - 1) / bn) * ((A.m + bm - 1) / bm); };
  if constexpr (sizeof(T) == 2) {
    if (groups(64, 16) > 512) {
      if (A.m <= 8) return launch_rows<T, 4, 8>(A, stream);
      if (groups(128, 32) <= 256) return launch_gemm<T, 2, 2, 4, 1, 2, 4>(A, stream);
      if (groups(128, 32) <= 640) return launch_gemm<T, 2, 2, 4, 1, 2, 2>(A, stream);
      if (groups(256, 32) <= 768 || A.m <= 32) return launch_gemm<T, 2, 2, 8, 1, 2>(A, stream);
      return launch_gemm<T, 2, 4, 8, 1, 2>(A, stream);
    }
    if (groups(16, 16) <= 256) return launch_rows<T, 1, 16>(A, stream);
    if (groups(32, 16) <= 256) return launch_rows<T, 2, 16>(A, stream);
    if (groups(32, 16) <= 512) return launch_rows<T, 2, 8>(A, stream);
    return launch_rows<T, 4, 8>(A, stream);
  } else {
    if (groups(256, 32) >= 512 && A.m > 16) return launch_gemm<T, 4, 2, 4, 1, 2>(A, stream);
    if (groups(16, 16) <= 256) return launch_rows<T, 1, 16>(A, stream);
    if (groups(32, 16) <= 256) return launch_rows<T, 2, 16>(A, stream);
    if (groups(64, 16) <= 256 || A.m <= 16) return launch_rows<T, 4, 8>(A, stream);
    return launch_rows<T, 8, 8>(A, stream);
  }
}

bool mx_sizes_ok(int mats, int n, int k) {
  return mats > 0 && n > 0 && k > 0 && k % MX_BLOCK == 0 && n <= (1 << 24) && k <= (1 << 20);
}
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// grid of one wave per tile; 0 when the launch would be too large
unsigned tile_grid(const MxGeom& g) {
  const long nb = (g.tiles + MX_NT / 64 - 1) / (MX_NT / 64);
  return nb > 0x7fffffffL / MX_NT ? 0u : (unsigned)nb;
}

}  // namespace

extern "C" size_t qm_mx4_code_bytes(int mats, int n, int k) {
  return mx_sizes_ok(mats, n, k) ? (size_t)mx_geom(mats, n, k).tiles * 1024 : 0;
}

#define QM_MX4_GEOM(name)                                                                                        \
  if (!mx_sizes_ok(mats, n, k))                                                                                  \
    return qm_fail(QM_ERR_ARG, name ": mats and n must be positive, k a positive multiple of 32 (n <= 2^24, k <= 2^20)"); \
  const MxGeom g = mx_geom(mats, n, k);                                                                          \
  const unsigned nb = tile_grid(g);                                                                              \
  if (!nb) return qm_fail(QM_ERR_UNSUPPORTED, name ": too many tiles for one launch")

extern "C" int qm_mx4_quantize(int act_dtype, int mats, int n, int k, const void* w, void* codes, void* scales,
                               hipStream_t stream) {
  if (act_dtype != QM_ACT_BF16 && act_dtype != QM_ACT_F32)
    return qm_fail(QM_ERR_DTYPE, "qm_mx4_quantize: act_dtype must be QM_ACT_F32 or QM_ACT_BF16");
  QM_MX4_GEOM("qm_mx4_quantize");
  if (!w || !codes || !scales) return qm_fail(QM_ERR_ARG, "qm_mx4_quantize: null pointer");
  if (!aligned16(w) || !aligned16(codes)) return qm_fail(QM_ERR_ARG, "qm_mx4_quantize: w and codes must be 16-byte aligned");
  uint8_t* c = static_cast<uint8_t*>(codes);
  uint8_t* s = static_cast<uint8_t*>(scales);
  if (act_dtype == QM_ACT_BF16)
    hipLaunchKernelGGL(mx4_quantize_kernel<bf16_t>, dim3(nb), dim3(MX_NT), 0, stream, g, static_cast<const bf16_t*>(w), c, s);
  else
    hipLaunchKernelGGL(mx4_quantize_kernel<float>, dim3(nb), dim3(MX_NT), 0, stream, g, static_cast<const float*>(w), c, s);
  QM_CHECK_LAUNCH();
  return QM_OK;
}

extern "C" int qm_mx4_dequantize(int act_dtype, int mats, int n, int k, const void* codes, const void* scales, void* w,
                                 hipStream_t stream) {
  if (act_dtype != QM_ACT_BF16 && act_dtype != QM_ACT_F32)
    return qm_fail(QM_ERR_DTYPE, "qm_mx4_dequantize: act_dtype must be QM_ACT_F32 or QM_ACT_BF16");
  QM_MX4_GEOM("qm_mx4_dequantize");
  if (!w || !codes || !scales) return qm_fail(QM_ERR_ARG, "qm_mx4_dequantize: null pointer");
  if (!aligned16(w) || !aligned16(codes))
    return qm_fail(QM_ERR_ARG, "qm_mx4_dequantize: w and codes must be 16-byte aligned");
  const uint8_t* c = static_cast<const uint8_t*>(codes);
  const uint8_t* s = static_cast<const uint8_t*>(scales);
  if (act_dtype == QM_ACT_BF16)
    hipLaunchKernelGGL(mx4_dequantize_kernel<bf16_t>, dim3(nb), dim3(MX_NT), 0, stream, g, c, s, static_cast<bf16_t*>(w));
  else
    hipLaunchKernelGGL(mx4_dequantize_kernel<float>, dim3(nb), dim3(MX_NT), 0, stream, g, c, s, static_cast<float*>(w));
  QM_CHECK_LAUNCH();
  return QM_OK;
}

extern "C" int qm_mx4_layout(int to_tiles, int mats, int n, int k, void* codes, void* scales, void* plain_codes,
                             void* plain_scales, hipStream_t stream) {
  QM_MX4_GEOM("qm_mx4_layout");
  if (!codes || !scales || !plain_codes || !plain_scales) return qm_fail(QM_ERR_ARG, "qm_mx4_layout: null pointer");
  if (!aligned16(codes) || !aligned16(plain_codes))
    return qm_fail(QM_ERR_ARG, "qm_mx4_layout: codes must be 16-byte aligned");
  uint8_t* c = static_cast<uint8_t*>(codes);
  uint8_t* s = static_cast<uint8_t*>(scales);
  uint8_t* pc = static_cast<uint8_t*>(plain_codes);
  uint8_t* ps = static_cast<uint8_t*>(plain_scales);
  if (to_tiles)
    hipLaunchKernelGGL(mx4_layout_kernel<true>, dim3(nb), dim3(MX_NT), 0, stream, g, c, s, pc, ps);
  else
    hipLaunchKernelGGL(mx4_layout_kernel<false>, dim3(nb), dim3(MX_NT), 0, stream, g, c, s, pc, ps);
  QM_CHECK_LAUNCH();
  return QM_OK;
}

namespace {

template <typename T>
int linear(int m, int n, int k, const void* codes, const void* scales, const void* x, long ldx, int n_seg,
           const int* seg_rows, void* const* seg_out, hipStream_t stream) {
  Mx4LinearArgs<T> A = {};
  A.w = {codes, static_cast<const uint8_t*>(scales)};
  A.x = static_cast<const T*>(x);
  A.ldx = ldx; A.m = m; A.n = n; A.k = k; A.rt = wt_row_tiles(n); A.kt = wt_k_tiles(k);
  A.n_seg = n_seg;
  long end = 0;
  for (int s = 0; s < n_seg; ++s) {
    end += seg_rows[s];
    A.seg_end[s] = (int)end;
    A.seg_out[s] = static_cast<T*>(seg_out[s]);
  }
  if (end != n) return qm_fail(QM_ERR_ARG, "qm_mx4_linear: segment rows must add up to n");
  return run_linear<T>(A, stream);
}

}  // namespace

extern "C" int qm_mx4_linear(int act_dtype, int m, int n, int k, const void* codes, const void* scales, const void* x,
                             long ldx, int n_seg, const int* seg_rows, void* const* seg_out, hipStream_t stream) {
  if (act_dtype != QM_ACT_BF16 && act_dtype != QM_ACT_F32)
    return qm_fail(QM_ERR_DTYPE, "qm_mx4_linear: act_dtype must be QM_ACT_F32 or QM_ACT_BF16");
  if (m <= 0 || m > 16 * 65535 || !mx_sizes_ok(1, n, k))
    return qm_fail(QM_ERR_ARG, "qm_mx4_linear: m and n must be positive (m <= 1048560), k a positive multiple of 32");
  if (!codes || !scales || !x || !seg_rows || !seg_out) return qm_fail(QM_ERR_ARG, "qm_mx4_linear: null pointer");
  const int unit = act_dtype == QM_ACT_BF16 ? 8 : 4;
  if (ldx < k || ldx % unit) return qm_fail(QM_ERR_ARG, "qm_mx4_linear: ldx must be at least k and whole 16-byte units");
  if (!aligned16(codes) || !aligned16(x)) return qm_fail(QM_ERR_ARG, "qm_mx4_linear: codes and x must be 16-byte aligned");
  // (the staged kernels load them four at a time)
  if (reinterpret_cast<uintptr_t>(scales) & 3) return qm_fail(QM_ERR_ARG, "qm_mx4_linear: scales must be 4-byte aligned");
  if (n_seg <= 0 || n_seg > QM_GEMV_MAX_SEG) return qm_fail(QM_ERR_ARG, "qm_mx4_linear: 1..8 output segments");
  for (int s = 0; s < n_seg; ++s)
    if (seg_rows[s] <= 0 || !seg_out[s]) return qm_fail(QM_ERR_ARG, "qm_mx4_linear: empty segment or null output");
  if (act_dtype == QM_ACT_BF16)
    return linear<bf16_t>(m, n, k, codes, scales, x, ldx, n_seg, seg_rows, seg_out, stream);
  return linear<float>(m, n, k, codes, scales, x, ldx, n_seg, seg_rows, seg_out, stream);
}
