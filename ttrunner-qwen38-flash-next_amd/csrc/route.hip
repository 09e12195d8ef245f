// Routing of token rows to experts, gfx950 (reference/model.py:387-417):
//
//   l[t][e] = sum_k x[t][k] R[e][k]            ids[t] = the top_k largest, ties to the lower index
//   w[t][j] = softmax(l[t])[ids[t][j]]         (over the chosen ones alone when normalize)
//
// The choice is that of the logits summed in double: which experts a token takes
// then depends on its values alone, not on the number of rows beside it or the
// order of a float sum: equal rows are routed alike in a verify step and a single one.
//
// Few rows form those sums outright, a wave per router row. Many rows take the
// matrix cores: products of 128 k are summed in float, the sums of 128 in double,
// so a logit is off by at most
//     B = (129 2^-23) |x| |R[e]| + hidden 2^-126      (|.| the 2-norms; the last
// for products below float's range), and only where two of a token's leading
// logits come closer than 2 B can the order be another. Those logits alone are
// summed again in double (about one token in ten of normal rows has such a pair). The
// weights come of the logits as they then are. Their exponentials and sums are floats
// (of differences in double; 8e-8 of a weight, where a double's would leave the 3e-8
// of its rounding): what a layer multiplies by them has a float's bits at most.
#include "moe_internal.h"
#include "moe_topk.h"
#include "wgemm.h"

namespace {

// Products of a call (rows x columns x hidden) up to which every logit is summed in
// double. Logits and choice over 2048, us, so / by matrix cores: bf16 128 experts 256
// rows (7e7) 16 / 20, 330 rows (9e7) 20 / 20, 400 rows (1.05e8) 22 / 21; float 128
// experts 1250 rows (3.3e8) 62 / 70, 1400 rows (3.7e8) 69 / 70, 1500 rows (3.9e8) 74 /
// 70; 256 experts 700 rows (3.7e8) 69 / 71, 800 rows 78 / 69; 64 experts 2800 rows
// (3.7e8) 70 / 70, 3000 rows 76 / 70.
template <typename T> constexpr double ROUTE_FEW = sizeof(T) == 2 ? 1e8 : 3.7e8;
// Choices of an expert, on average, up to which the choosing waves file them by
// atomics (they serialise: 8 each +2.4 us, 16 +4.2, 32 +7.2, 250 +31); beyond, a
// launch of its own does (6.0 us and its start, 7.7 at 16000 choices)
constexpr int LISTS_ATOMIC = 24;

constexpr int RT_TB = 4;                 // token rows of one wave of the few-row logits

// 16 bytes as floats
__device__ __forceinline__ void unit_get(const uint4& c, float (&v)[8], const bf16_t*) {
  const unsigned d[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(d[i] << 16);
    v[2 * i + 1] = __uint_as_float(d[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void unit_get(const uint4& c, float (&v)[4], const float*) {
  v[0] = __uint_as_float(c.x); v[1] = __uint_as_float(c.y); v[2] = __uint_as_float(c.z); v[3] = __uint_as_float(c.w);
}

// s + w x in double (a product of two bf16 fits a float's bits, but not its range)
__device__ __forceinline__ double exact_fma(float w, float x, double s) { return fma((double)w, (double)x, s); }

template <int LANES> __device__ __forceinline__ double lanes_sum_f64(double v) {
#pragma unroll
  for (int m = LANES / 2; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
  return v;
}

template <typename T>
__device__ __forceinline__ const T* router_row(const QmLogits<T>& A, int r) {
  return r < A.experts ? A.router + (long)r * A.hidden : A.shared_router;
}

// the experts' counts of pairs, for the choice that follows
template <typename T> __device__ __forceinline__ void clear_counts(const QmLogits<T>& A) {
  if (A.counts && blockIdx.x == 0 && blockIdx.y == 0)
    for (int i = threadIdx.x; i <= A.experts; i += blockDim.x) A.counts[i] = 0;
}

// logits[t][r] of the router's rows and, when there is one, the shared experts' row:
// a wave per router row and TB tokens (four share a row's loads and conversions; a
// single token takes the form without them). A launch and two round trips to memory
// bound a few rows (128 experts over 2048, bf16: 1 row 3.0 us, 9 rows 4.1), the
// double sums many (256 rows 12.4).
template <typename T, int TB>
__global__ __launch_bounds__(256) void moe_logits_kernel(QmLogits<T> A) {
  constexpr int VE = 16 / sizeof(T), B = TB == 1 ? 4 : 2;    // units of a lane in flight
  const int lane = threadIdx.x & 63;
  const int r = blockIdx.x * 4 + (threadIdx.x >> 6);
  clear_counts(A);
  if (r >= A.cols) return;
  const int t0 = blockIdx.y * TB, units = A.hidden / VE;
  const T* w = router_row(A, r);
  const T* x[TB];
  double acc[TB];
#pragma unroll
  for (int i = 0; i < TB; ++i) {
    x[i] = A.x + (long)min(t0 + i, A.rows - 1) * A.ldx;
    acc[i] = 0.0;
  }
  for (int u0 = lane; u0 < units; u0 += 64 * B) {
    uint4 wu[B], xu[B][TB];
#pragma unroll
    for (int b = 0; b < B; ++b) {
      const long at = (long)min(u0 + 64 * b, units - 1) * VE;
      wu[b] = *reinterpret_cast<const uint4*>(w + at);
#pragma unroll
      for (int i = 0; i < TB; ++i) xu[b][i] = *reinterpret_cast<const uint4*>(x[i] + at);
    }
    __builtin_amdgcn_sched_barrier(0);                       // all of them in flight
#pragma unroll
    for (int b = 0; b < B; ++b) {
      if (u0 + 64 * b >= units) break;
      float wv[VE];
      unit_get(wu[b], wv, w);
#pragma unroll
      for (int i = 0; i < TB; ++i) {
        float xv[VE];
        unit_get(xu[b][i], xv, w);
#pragma unroll
        for (int e = 0; e < VE; ++e) acc[i] = exact_fma(wv[e], xv[e], acc[i]);
      }
    }
  }
  // the lanes' sums meet in the order of their numbers' bits, as in exact_logits; of
  // four tokens half a wave, then a quarter goes on with its own
  int t = t0;
  if constexpr (TB == 4) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const double give = lane & 32 ? acc[i] : acc[i + 2];
      acc[i] = (lane & 32 ? acc[i + 2] : acc[i]) + __shfl_xor(give, 32, 64);
    }
    const double give = lane & 16 ? acc[0] : acc[1];
    acc[0] = lanes_sum_f64<16>((lane & 16 ? acc[1] : acc[0]) + __shfl_xor(give, 16, 64));
    t += (lane >> 4 & 1) + (lane >> 4 & 2);
  } else {
    acc[0] = lanes_sum_f64<64>(acc[0]);
  }
  if ((TB == 4 ? lane & 15 : lane) == 0 && t < A.rows) A.logits[(long)t * A.cols + r] = acc[0];
}

// The same by matrix cores: a workgroup per 64 router rows x 64 tokens (those of the
// same tokens on one XCD, whose L2 then reads them once), both kinds of rows in LDS
// (two stages of LG_SPANS times 128 k, units exchanged as in wgemm.h), a wave per
// 16 x 32. norms: |R[r]|^2, then |x[t]|^2, the diagonals of products of 16 rows with
// themselves, by the first workgroups of a column or a row of tiles. A span takes a
// workgroup 0.6 us whatever else runs, its loads, its reads of LDS and the steps
// between them one after the other (bf16, 256 experts over 2048: 4001 rows 16.9 us;
// 64 experts, 2000 rows 13; with stages of one span, four or five of them, 17.6 and
// 15; 32 x 32 a wave and a quarter of k 17.5 and 14). Float products are bound by the
// matrix cores: 4000 rows over 256 experts 64 us, 76 with the norms in fewer waves.
constexpr int LG_ROWS = 128;
template <typename T> constexpr int LG_SPANS = sizeof(T) == 2 ? 2 : 1;

template <typename T>
__global__ __launch_bounds__(512) void moe_logits_mma_kernel(QmLogits<T> A, float* norms) {
  constexpr int ROW_B = WT_K * sizeof(T), UNITS = ROW_B / 16, VE = 16 / sizeof(T), RPL = 1024 / ROW_B;
  constexpr int LOADS = LG_ROWS / RPL / 8, BUF = LG_ROWS * ROW_B, SP = LG_SPANS<T>;
  extern __shared__ __attribute__((aligned(16))) char s_buf[];
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g4 = lane >> 4, r16 = lane & 15;
  const int et = (A.cols + 63) / 64, item = xcd_run(blockIdx.x, gridDim.x);
  const int e0 = item % et * 64, t0 = item / et * 64;
  // a group of 16 rows a wave: of the four of router rows waves 0, 2, 5 and 7, of the
  // tokens' 4, 6, 1 and 3 (each multiplies them anyway)
  const bool of_router = (((wid >> 2) ^ wid) & 1) == 0, norm = of_router ? item < et : e0 == 0;
  const T* src[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int row = (wid * LOADS + i) * RPL + lane / UNITS;
    src[i] = row < 64 ? router_row(A, min(e0 + row, A.cols - 1)) : A.x + (long)min(t0 + row - 64, A.rows - 1) * A.ldx;
  }
  auto fetch = [&](int j) {
#pragma unroll
    for (int h = 0; h < SP; ++h) {
      char* buf = s_buf + (j % 2 * SP + h) * BUF;
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int row = (wid * LOADS + i) * RPL + lane / UNITS;
        const int k = (j * SP + h) * WT_K + ((lane % UNITS) ^ (row & 15)) * VE;
        lds_load16(k < A.hidden ? static_cast<const void*>(src[i] + k) : g_zero_unit, buf + (wid * LOADS + i) * 1024);
      }
    }
  };
  const int stages = (wt_k_tiles(A.hidden) + SP - 1) / SP;
  clear_counts(A);
  fetch(0);
  double acc[2][4];
  f32x4_t gram = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[u][i] = 0.0;
  for (int j = 0; j < stages; ++j) {
    wave_loads_barrier<0>();
    if (j + 1 < stages) fetch(j + 1);
#pragma unroll
    for (int h = 0; h < SP; ++h) {
      const char* buf = s_buf + (j % 2 * SP + h) * BUF;
      Piece<T> a[4], b[4][2];
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        a[s] = lds_piece<T>(buf + ((wid >> 1) * 16 + r16) * ROW_B, 4 * s + g4, r16);
#pragma unroll
        for (int u = 0; u < 2; ++u)
          b[s][u] = lds_piece<T>(buf + (64 + (wid & 1) * 32 + 16 * u + r16) * ROW_B, 4 * s + g4, r16);
      }
      __builtin_amdgcn_sched_barrier(0);                     // all reads in flight before the first product
      f32x4_t part[1][2];
      clear(part);
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int u = 0; u < 2; ++u) part[0][u] = mma_piece(a[s], b[s][u], part[0][u]);
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[u][i] += (double)part[0][u][i];
      if (norm && of_router) {
#pragma unroll
        for (int s = 0; s < 4; ++s) gram = mma_piece(a[s], a[s], gram);
      } else if (norm && (wid & 2)) {
#pragma unroll
        for (int s = 0; s < 4; ++s) gram = mma_piece(b[s][1], b[s][1], gram);
      } else if (norm) {
#pragma unroll
        for (int s = 0; s < 4; ++s) gram = mma_piece(b[s][0], b[s][0], gram);
      }
    }
  }
  // a lane holds rows 4 g4 + i of column r16: the diagonal's element in one of four
  if (norm && (r16 >> 2) == g4) {
    const float n = (r16 & 2) ? (r16 & 1) ? gram[3] : gram[2] : (r16 & 1) ? gram[1] : gram[0];
    const int r = of_router ? e0 + (wid >> 1) * 16 + r16 : t0 + (wid & 1) * 32 + (wid & 2) * 8 + r16;
    if (r < (of_router ? A.cols : A.rows)) norms[of_router ? r : A.cols + r] = n;
  }
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int t = t0 + (wid & 1) * 32 + 16 * u + r16;
    if (t >= A.rows) continue;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = e0 + (wid >> 1) * 16 + 4 * g4 + i;
      if (r < A.cols) A.logits[(long)t * A.cols + r] = acc[u][i];
    }
  }
}

struct TopArgs {
  int top_k, normalize, ld_w, shared;
  int* ids;            // [rows][top_k]
  float* weights;      // [rows][ld_w]: the choices, then the shared experts
  QmRouteLists lists;  // counts null: none wanted
  const float* norms;  // null: the logits are sums in double already
};

// The logits of two columns in double (a close pair, mostly), by the wave: lane c < 2
// gets that of e[c]. One round trip for both; the lanes' partial sums meet in the order
// of their numbers' bits, whichever two are asked for.
constexpr int EXACT = RT_EXACT;
template <typename T>
__device__ __forceinline__ double exact_logits(const QmLogits<T>& A, int t, const int (&e)[EXACT], int lane) {
  constexpr int VE = 16 / sizeof(T), B = 4;                  // units of a lane in flight
  const int units = A.hidden / VE;
  const T* x = A.x + (long)t * A.ldx;
  double s[EXACT];
#pragma unroll
  for (int c = 0; c < EXACT; ++c) s[c] = 0.0;
  for (int u0 = lane; u0 < units; u0 += 64 * B) {
    uint4 xu[B], wu[EXACT][B];
#pragma unroll
    for (int b = 0; b < B; ++b) {
      const long at = (long)min(u0 + 64 * b, units - 1) * VE;
      xu[b] = *reinterpret_cast<const uint4*>(x + at);
#pragma unroll
      for (int c = 0; c < EXACT; ++c) wu[c][b] = *reinterpret_cast<const uint4*>(router_row(A, e[c]) + at);
    }
#pragma unroll
    for (int b = 0; b < B; ++b) {
      if (u0 + 64 * b >= units) break;
      float xv[VE];
      unit_get(xu[b], xv, x);
#pragma unroll
      for (int c = 0; c < EXACT; ++c) {
        float wv[VE];
        unit_get(wu[c][b], wv, x);
#pragma unroll
        for (int i = 0; i < VE; ++i) s[c] = exact_fma(wv[i], xv[i], s[c]);
      }
    }
  }
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1)
#pragma unroll
    for (int c = 0; c < EXACT; ++c) s[c] += __shfl_xor(s[c], m, 64);
  double mine = s[0];
#pragma unroll
  for (int c = 1; c < EXACT; ++c) mine = lane == c ? s[c] : mine;
  return mine;
}

// The workgroup that finishes last makes the table of row tiles from the counts,
// the shared experts first.
template <int NT>
__device__ __forceinline__ void finish_lists(int rows, int experts, const QmRouteLists& L) {
  __shared__ int s_wave[NT / 64];
  __shared__ bool s_last;
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  wait_all_memory();                                         // this wave's counts are in
  __syncthreads();
  if (threadIdx.x == 0)
    s_last = __hip_atomic_fetch_add(L.counts + experts, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (int)gridDim.x - 1;
  __syncthreads();
  if (!s_last) return;
  int start = 0;
  const int all = L.shared + experts;
  for (int y0 = 0; y0 < all; y0 += NT) {
    const int y = y0 + threadIdx.x;
    int count = 0;
    if (y < all) count = y < L.shared ? rows : (int)ld_flag(reinterpret_cast<const unsigned*>(L.counts + y - L.shared));
    const int mine = (count + L.bm - 1) / L.bm;
    int before = mine;                                       // inclusive scan over the wave
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(before, d, 64);
      if (lane >= d) before += o;
    }
    __syncthreads();
    if (lane == 63) s_wave[wid] = before;
    __syncthreads();
    int place = start + before - mine;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) {
      const int c = s_wave[w];
      if (w < wid) place += c;
      start += c;
    }
    for (int i = 0; i < mine; ++i) L.tiles[place + i] = make_int2(y, i * L.bm);
  }
  if (threadIdx.x == 0) *L.n_tiles = start;
}

// The lists of many choices, a workgroup per expert: a thread finds the hits among
// 16 consecutive choices, a scan over the workgroup places them (16000 choices of 64
// experts 7 us).
constexpr int LS_NT = 1024, LS_PER = 16;
__global__ __launch_bounds__(LS_NT) void moe_lists_kernel(const int* ids, int rows, int top_k, QmRouteLists L) {
  __shared__ int s_hits[LS_NT / 64];
  const int e = blockIdx.x, lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int n = rows * top_k;
  int* list = L.lists + (long)e * rows;
  int at = 0;
  for (int p0 = 0; p0 < n; p0 += LS_NT * LS_PER) {
    const int p = p0 + threadIdx.x * LS_PER;
    unsigned hits = 0;
    if (p + LS_PER <= n) {                                   // ids are 16-byte aligned
#pragma unroll
      for (int i = 0; i < LS_PER / 4; ++i) {
        const int4 v = *reinterpret_cast<const int4*>(ids + p + 4 * i);
        hits |= ((v.x == e) | (v.y == e) << 1 | (v.z == e) << 2 | (v.w == e) << 3) << (4 * i);
      }
    } else {
      for (int i = 0; i < LS_PER; ++i)
        if (p + i < n && ids[p + i] == e) hits |= 1u << i;
    }
    const int mine = __popc(hits);
    int before = mine;                                       // inclusive scan over the wave
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(before, d, 64);
      if (lane >= d) before += o;
    }
    if (lane == 63) s_hits[wid] = before;
    __syncthreads();
    int place = at + before - mine;
#pragma unroll
    for (int w = 0; w < LS_NT / 64; ++w) {
      const int c = s_hits[w];
      if (w < wid) place += c;
      at += c;
    }
    while (hits) {
      const int q = p + __ffs(hits) - 1;
      list[place++] = q / top_k * L.ppt + q % top_k;
      hits &= hits - 1;
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) st_flag(reinterpret_cast<unsigned*>(L.counts + e), (unsigned)at);
  finish_lists<LS_NT>(rows, gridDim.x, L);
}

// A token's choice, by one wave
template <typename T, int PER>
__device__ __forceinline__ void topk_row(const QmLogits<T>& A, const TopArgs& P, int t, int lane) {
  double* l = A.logits + (long)t * A.cols;
  double off = 0.0;                        // the logits' own error
  bool all = false;                        // every logit has to be summed again
  if (P.norms) {
    const float xn = P.norms[A.cols + t];
    float wn = 0.f;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = lane + 64 * i;
      if (e >= A.experts) continue;
      const float v = P.norms[e];
      wn = fmaxf(wn, v);
      bad |= !(v < INFINITY) || !(fabs(l[e]) < (double)INFINITY);
    }
    wn = wave_max(wn);
    // squares below float's range hide a norm: a row of zeros is looked through
    bool zero = false;
    if (xn < 0x1p-80f) {
      constexpr int VE = 16 / sizeof(T);
      unsigned any = 0u;
      for (int u = lane; u < A.hidden / VE; u += 64) {
        const uint4 v = *reinterpret_cast<const uint4*>(A.x + (long)t * A.ldx + (long)u * VE);
        any |= (v.x | v.y | v.z | v.w) & (sizeof(T) == 2 ? 0x7fff7fffu : 0x7fffffffu);
      }
      zero = __builtin_amdgcn_ballot_w64(any != 0u) == 0ull;
    }
    all = __builtin_amdgcn_ballot_w64(bad) != 0ull || !(xn < INFINITY) || (!zero && (xn < 0x1p-80f || wn < 0x1p-80f));
    // (its logits are zero; a norm's own sum is off by at most a step each time)
    if (!zero)
      off = 129.0 * 0x1p-23 * (1.0 + A.hidden * 0x1p-22) * sqrt((double)xn * (double)wn) + A.hidden * 0x1p-126;
  }
  long long key;                           // lane j: the j-th largest
  int id;
  if (!all)
    all = !wave_topk<PER>(l, A.experts, P.top_k, off, lane, key, id,
                          [&](const int (&e)[EXACT]) { return exact_logits(A, t, e, lane); });
  if (all) {
    if (P.norms) {
      for (int e0 = 0; e0 < A.experts; e0 += EXACT) {
        const int last = A.experts - 1, e[EXACT] = {e0, min(e0 + 1, last)};
        const double s = exact_logits(A, t, e, lane);
        if (lane < EXACT && e0 + lane < A.experts) l[e0 + lane] = s;
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      wait_all_memory();
    }
    wave_topk_exact(l, A.experts, P.top_k, lane, key, id);
  }
  const double v0 = key_logit(lane_key(key, 0));
  const float mine = lane < P.top_k ? expf((float)(key_logit(key) - v0)) : 0.f;
  float sum = 0.f;
  if (P.normalize) {
    sum = wave_sum(mine);
  } else {
    for (int e = lane; e < A.experts; e += 64) sum += expf((float)(l[e] - v0));
    sum = wave_sum(sum);
  }
  if (lane < P.top_k) {
    P.ids[(long)t * P.top_k + lane] = id;
    P.weights[(long)t * P.ld_w + lane] = mine / sum;
    if (P.lists.counts) {
      // the order of an expert's pairs is that of arrival; their products do not
      // depend on it
      const int at = __hip_atomic_fetch_add(P.lists.counts + id, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      P.lists.lists[(long)id * A.rows + at] = t * P.lists.ppt + lane;
    }
  }
  if (P.shared > 0) {
    float w = 1.f;
    if (A.cols > A.experts) {
      double s = l[A.experts];
      // No part of a float sum leaves float's range where both squared norms are in it
      // (it is at most their root); elsewhere the sum in double, as few rows have it.
      if (P.norms && !(P.norms[A.cols + t] < INFINITY && P.norms[A.experts] < INFINITY)) {
        const int e[EXACT] = {A.experts, A.experts};
        s = exact_logits(A, t, e, lane);
      }
      w = sigmoid_f((float)s);
    }
    if (lane < P.shared) P.weights[(long)t * P.ld_w + P.top_k + lane] = w;
  }
}

// One wave per token: a chain of a load, a search and a ranking (moe_topk.h) and, for
// one token in ten of the many-row logits, another load and two sums in double (4001
// tokens over 256 experts 14.3 us, one over 128 3.0)
template <typename T, int PER>
__global__ __launch_bounds__(256) void moe_topk_kernel(QmLogits<T> A, TopArgs P) {
  const int lane = threadIdx.x & 63;
  const int t = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t < A.rows) topk_row<T, PER>(A, P, t, lane);
  if (P.lists.counts) finish_lists<256>(A.rows, A.experts, P.lists);
}

template <typename T, int PER>
int launch_topk(const QmLogits<T>& A, const TopArgs& P, hipStream_t stream) {
  hipLaunchKernelGGL((moe_topk_kernel<T, PER>), dim3((A.rows + 3) / 4), dim3(256), 0, stream, A, P);
  QM_CHECK_LAUNCH();
  return QM_OK;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

size_t qm_route_norms(int rows, int experts) { return ((size_t)rows + experts + 1) * sizeof(float); }

template <typename T>
int qm_route_logits(const QmLogits<T>& A, hipStream_t stream) {
  if (A.rows == 1) hipLaunchKernelGGL((moe_logits_kernel<T, 1>), dim3((A.cols + 3) / 4), dim3(256), 0, stream, A);
  else hipLaunchKernelGGL((moe_logits_kernel<T, RT_TB>), dim3((A.cols + 3) / 4, (A.rows + RT_TB - 1) / RT_TB), dim3(256), 0, stream, A);
  QM_CHECK_LAUNCH();
  return QM_OK;
}

template <typename T>
int qm_route(const QmLogits<T>& A, int top_k, int normalize, int* ids, float* weights, int ld_w, int shared,
             const QmRouteLists* lists, float* norms, hipStream_t stream) {
  TopArgs P = {top_k, normalize, ld_w, shared, ids, weights, lists ? *lists : QmRouteLists{}, nullptr};
  int rc;
  if ((double)A.rows * A.cols * A.hidden <= ROUTE_FEW<T>) {
    rc = qm_route_logits(A, stream);
  } else {
    P.norms = norms;
    const size_t lds = (size_t)2 * LG_SPANS<T> * LG_ROWS * WT_K * sizeof(T);
    static std::atomic<uint64_t> allowed{0};
    rc = qm_allow_lds(reinterpret_cast<const void*>(moe_logits_mma_kernel<T>), lds, allowed);
    if (rc) return rc;
    hipLaunchKernelGGL(moe_logits_mma_kernel<T>, dim3((A.cols + 63) / 64 * ((A.rows + 63) / 64)), dim3(512), lds, stream, A, norms);
    QM_CHECK_LAUNCH();
  }
  if (rc) return rc;
  const bool apart = lists && (long)A.rows * top_k > (long)LISTS_ATOMIC * A.experts;
  if (apart) P.lists = QmRouteLists{};
  if (A.experts <= 64) rc = launch_topk<T, 1>(A, P, stream);
  else if (A.experts <= 128) rc = launch_topk<T, 2>(A, P, stream);
  else if (A.experts <= 256) rc = launch_topk<T, 4>(A, P, stream);
  else if (A.experts <= 512) rc = launch_topk<T, 8>(A, P, stream);
  else rc = launch_topk<T, 16>(A, P, stream);
  if (rc || !apart) return rc;
  hipLaunchKernelGGL(moe_lists_kernel, dim3(A.experts), dim3(LS_NT), 0, stream, ids, A.rows, top_k, *lists);
  QM_CHECK_LAUNCH();
  return QM_OK;
}

template int qm_route_logits<bf16_t>(const QmLogits<bf16_t>&, hipStream_t);
template int qm_route_logits<float>(const QmLogits<float>&, hipStream_t);
template int qm_route<bf16_t>(const QmLogits<bf16_t>&, int, int, int*, float*, int, int, const QmRouteLists*, float*, hipStream_t);
template int qm_route<float>(const QmLogits<float>&, int, int, int*, float*, int, int, const QmRouteLists*, float*, hipStream_t);

int qm_check_route(const char* what, int act_dtype, int rows, int hidden, int experts, int top_k, long ldx) {
  char msg[160];
  const int unit = act_dtype == QM_ACT_BF16 ? 8 : 4;
  const char* bad = nullptr;
  int code = QM_ERR_ARG;
  if (act_dtype != QM_ACT_BF16 && act_dtype != QM_ACT_F32) { bad = "act_dtype must be QM_ACT_F32 or QM_ACT_BF16"; code = QM_ERR_DTYPE; }
  else if (rows <= 0 || rows > 262140) bad = "rows must be 1..262140";
  else if (hidden <= 0 || hidden % 32 || hidden > (1 << 20)) bad = "hidden must be a positive multiple of 32 (at most 2^20)";
  else if (experts <= 0 || experts > RT_MAX_EXPERTS) { bad = "experts must be 1..1024"; code = QM_ERR_UNSUPPORTED; }
  else if (top_k <= 0 || top_k > RT_MAX_TOPK || top_k > experts) bad = "top_k must be 1..32 and at most experts";
  else if (ldx < hidden || ldx % unit) bad = "ldx must be at least hidden and whole 16-byte units";
  if (!bad) return QM_OK;
  snprintf(msg, sizeof(msg), "%s: %s", what, bad);
  return qm_fail(code, msg);
}

extern "C" size_t qm_moe_route_workspace(int rows, int experts) {
  if (rows <= 0 || experts <= 0 || experts > RT_MAX_EXPERTS) return 0;
  return qm_align256((size_t)rows * experts * sizeof(double)) + qm_align256(qm_route_norms(rows, experts));
}

extern "C" int qm_moe_route(int act_dtype, int rows, int hidden, int experts, int top_k, int normalize, const void* x,
                            long ldx, const void* router, int* ids, float* weights, void* workspace,
                            size_t workspace_bytes, hipStream_t stream) {
  const int rc = qm_check_route("qm_moe_route", act_dtype, rows, hidden, experts, top_k, ldx);
  if (rc) return rc;
  if (!x || !router || !ids || !weights || !workspace) return qm_fail(QM_ERR_ARG, "qm_moe_route: null pointer");
  if (!aligned16(x) || !aligned16(router) || !aligned16(workspace))
    return qm_fail(QM_ERR_ARG, "qm_moe_route: x, router and workspace must be 16-byte aligned");
  if (workspace_bytes < qm_moe_route_workspace(rows, experts))
    return qm_fail(QM_ERR_WORKSPACE, "qm_moe_route: workspace too small");
  double* logits = static_cast<double*>(workspace);
  float* norms = reinterpret_cast<float*>(static_cast<char*>(workspace) + qm_align256((size_t)rows * experts * sizeof(double)));
  if (act_dtype == QM_ACT_BF16) {
    const QmLogits<bf16_t> L = {static_cast<const bf16_t*>(x), ldx, static_cast<const bf16_t*>(router), nullptr, logits, rows,
                                hidden, experts, experts, nullptr};
    return qm_route(L, top_k, normalize, ids, weights, top_k, 0, nullptr, norms, stream);
  }
  const QmLogits<float> L = {static_cast<const float*>(x), ldx, static_cast<const float*>(router), nullptr, logits, rows,
                             hidden, experts, experts, nullptr};
  return qm_route(L, top_k, normalize, ids, weights, top_k, 0, nullptr, norms, stream);
}
