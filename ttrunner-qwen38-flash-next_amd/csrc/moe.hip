// Mixture-of-experts layer, gfx950: the routing of token rows to experts and the
// chosen experts' gated FFN (reference/model.py:387-417).
//
//   l[t][e] = sum_k x[t][k] R[e][k]            ids[t] = the top_k largest, ties to the lower index
//   w[t][j] = softmax(l[t])[ids[t][j]]         (over the chosen ones alone when normalize)
//   y[t]    = sum_j w[t][j] D_e (silu(G_e x[t]) * (U_e x[t]))
//           + sigmoid(x[t] . r) sum_s (shared expert s of x[t])
//
// Logits are sums of exact products in double: which experts a token takes then
// depends on its values alone, not on the number of rows beside it or the order
// of a sum, so a verify step routes as the single steps do.
//
// A pair is a (token, expert) choice; pair (top_k + shared) t + j is choice j of
// token t, the shared experts its last ones. The pair's weight multiplies the
// hidden row in float before that is rounded to the activations' type (the
// operand of the second product), so the second products add up unweighted, in
// the order of j.
#include <stdio.h>

#include "qwen4mix_internal.h"
#include "wtile.h"

namespace {

constexpr int RT_TB = 4;                 // token rows of one wave of the logits
constexpr int RT_MAX_EXPERTS = 1024;
constexpr int RT_MAX_TOPK = 32;

template <typename T> struct Unit;       // 16 bytes as floats
template <> struct Unit<bf16_t> {
  static constexpr int VE = 8;
  __device__ __forceinline__ static void get(const uint4& c, float (&v)[8]) {
    const unsigned d[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(d[i] << 16);
      v[2 * i + 1] = __uint_as_float(d[i] & 0xffff0000u);
    }
  }
};
template <> struct Unit<float> {
  static constexpr int VE = 4;
  __device__ __forceinline__ static void get(const uint4& c, float (&v)[4]) {
    v[0] = __uint_as_float(c.x); v[1] = __uint_as_float(c.y); v[2] = __uint_as_float(c.z); v[3] = __uint_as_float(c.w);
  }
};

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
  return v;
}

// logits[t][r], r < experts rows of the router and, when shared_router is given,
// one more row for it
template <typename T>
struct LogitArgs {
  const T* x;
  long ldx;
  const T* router;
  const T* shared_router;
  double* logits;
  int rows, hidden, experts, cols;
};

template <typename T>
__global__ __launch_bounds__(256) void moe_logits_kernel(LogitArgs<T> A) {
  constexpr int VE = Unit<T>::VE;
  const int lane = threadIdx.x & 63;
  const int r = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= A.cols) return;
  const int t0 = blockIdx.y * RT_TB;
  const T* w = r < A.experts ? A.router + (long)r * A.hidden : A.shared_router;
  double acc[RT_TB];
#pragma unroll
  for (int i = 0; i < RT_TB; ++i) acc[i] = 0.0;
  for (int u = lane; u < A.hidden / VE; u += 64) {
    float wv[VE];
    Unit<T>::get(*reinterpret_cast<const uint4*>(w + (long)u * VE), wv);
#pragma unroll
    for (int i = 0; i < RT_TB; ++i) {
      float xv[VE];
      Unit<T>::get(*reinterpret_cast<const uint4*>(A.x + (long)min(t0 + i, A.rows - 1) * A.ldx + (long)u * VE), xv);
#pragma unroll
      for (int e = 0; e < VE; ++e) acc[i] = fma((double)wv[e], (double)xv[e], acc[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < RT_TB; ++i) {
    const double s = wave_sum_f64(acc[i]);
    if (lane == 0 && t0 + i < A.rows) A.logits[(long)(t0 + i) * A.cols + r] = s;
  }
}

// A logit as an integer of the same order: NaN above everything, +0 and -0 equal.
__device__ __forceinline__ long long logit_key(double v) {
  if (v != v) return 0x7fffffffffffffffLL;
  const long long b = __double_as_longlong(v + 0.0);
  return b < 0 ? b ^ 0x7fffffffffffffffLL : b;
}

// One wave per token: lane l holds logits l, l + 64, ...; each round takes the
// largest of what is left, the lowest index among equals.
__global__ __launch_bounds__(256) void moe_topk_kernel(const double* logits, int rows, int cols, int experts, int top_k,
                                                       int normalize, int* ids, float* weights, int ld_w, int shared) {
  const int lane = threadIdx.x & 63;
  const int t = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= rows) return;
  constexpr int PER = RT_MAX_EXPERTS / 64;
  constexpr long long GONE = (long long)0x8000000000000000ULL;
  const double* l = logits + (long)t * cols;
  long long key[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = lane + 64 * i;
    key[i] = e < experts ? logit_key(l[e]) : GONE;
  }
  double top = 0.0;
  float mine = 0.f;                      // lane j: choice j's weight before the division
  int mine_id = 0;
  for (int j = 0; j < top_k; ++j) {
    long long best = GONE;
    int at = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (key[i] > best) { best = key[i]; at = lane + 64 * i; }
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) {
      const long long ob = __shfl_xor(best, m, 64);
      const int oa = __shfl_xor(at, m, 64);
      if (ob > best || (ob == best && oa < at)) { best = ob; at = oa; }
    }
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (lane + 64 * i == at) key[i] = GONE;
    const double v = l[at];
    if (j == 0) top = v;
    if (lane == j) { mine = expf((float)(v - top)); mine_id = at; }
  }
  float sum = 0.f;
  if (normalize) {
    sum = wave_sum(lane < top_k ? mine : 0.f);
  } else {
    for (int e = lane; e < experts; e += 64) sum += expf((float)(l[e] - top));
    sum = wave_sum(sum);
  }
  if (lane < top_k) {
    ids[(long)t * top_k + lane] = mine_id;
    weights[(long)t * ld_w + lane] = mine / sum;
  }
  if (lane < shared) {
    float g = 1.f;
    if (cols > experts) g = (float)(1.0 / (1.0 + exp(-l[experts])));
    weights[(long)t * ld_w + top_k + lane] = g;
  }
}

// Each expert's pairs in the tokens' order (a workgroup per expert)
__global__ __launch_bounds__(256) void moe_lists_kernel(const int* ids, int rows, int top_k, int ppt, int* counts,
                                                        int* lists) {
  __shared__ int s_wave[4];
  const int e = blockIdx.x, lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int n = rows * top_k;
  int* list = lists + (long)e * rows;
  int at = 0;
  for (int p0 = 0; p0 < n; p0 += 256) {
    const int p = p0 + threadIdx.x;
    const bool hit = p < n && ids[p] == e;
    const unsigned long long m = __builtin_amdgcn_ballot_w64(hit);
    if (lane == 0) s_wave[wid] = __popcll(m);
    __syncthreads();
    int before = at, all = 0;
    for (int w = 0; w < 4; ++w) {
      if (w < wid) before += s_wave[w];
      all += s_wave[w];
    }
    if (hit) list[before + __popcll(m & ((1ull << lane) - 1ull))] = p / top_k * ppt + p % top_k;
    at += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) counts[e] = at;
}

template <typename T>
struct MoeArgs {
  const T* x;
  long ldx;
  int rows, hidden, inter, experts, shared, top_k, ppt;
  WMat gate, up, down, s_gate, s_up, s_down;
  const int* counts;
  const int* lists;
  const float* pair_w;
  T* h;              // [pairs][inter]
  float* part;       // [pairs][hidden]
  T* out;            // [rows][hidden]
};

// rows (pairs) of the expert of grid row y; the shared experts come first
struct ExpertRows {
  int e;             // of its weights
  bool is_shared;
  int count;
  const int* list;   // null: every token's pair `first`
  int first;
};
template <typename T>
__device__ __forceinline__ ExpertRows expert_rows(const MoeArgs<T>& A, int y) {
  if (y < A.shared) return {y, true, A.rows, nullptr, A.top_k + y};
  const int e = y - A.shared;
  return {e, false, A.counts[e], A.lists + (long)e * A.rows, 0};
}
__device__ __forceinline__ int pair_of(const ExpertRows& r, int i, int ppt) {
  return r.list ? r.list[i] : i * ppt + r.first;
}
__device__ __forceinline__ WMat expert_mat(const WMat& m, int e, long tiles, int tile_bytes) {
  return {static_cast<const char*>(m.data) + (long)e * tiles * tile_bytes, m.scales ? m.scales + (long)e * tiles * 64 : nullptr};
}
template <typename WF> __device__ __forceinline__ constexpr int tile_bytes() {
  return sizeof(WF) && __is_same(WF, WMx4) ? 1024 : __is_same(WF, WBf16) ? 4096 : 8192;
}

// h = w silu(G x) (U x): a workgroup per (TN tiles of hidden units, expert), the
// waves split k, 16 MT pairs at a time
template <typename WF, typename T, int TN, int MT, int NW>
__global__ __launch_bounds__(64 * NW) void moe_up_kernel(MoeArgs<T> A) {
  using F = Fmt<WF, T>;
  __shared__ f32x4_t s_red[NW][2 * TN * MT][64];
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int g4 = lane >> 4, r16 = lane & 15;
  const ExpertRows R = expert_rows(A, blockIdx.y);
  const int t0 = blockIdx.x * TN;
  const int rt = wt_row_tiles(A.inter), kt = wt_k_tiles(A.hidden);
  const WMat gate = expert_mat(R.is_shared ? A.s_gate : A.gate, R.e, (long)rt * kt, tile_bytes<WF>());
  const WMat up = expert_mat(R.is_shared ? A.s_up : A.up, R.e, (long)rt * kt, tile_bytes<WF>());
  for (int m0 = 0; m0 < R.count; m0 += 16 * MT) {
    const T* xp[MT];
#pragma unroll
    for (int u = 0; u < MT; ++u)
      xp[u] = A.x + (long)(pair_of(R, min(m0 + 16 * u + r16, R.count - 1), A.ppt) / A.ppt) * A.ldx;
    f32x4_t acc[2 * TN][MT];
#pragma unroll
    for (int t = 0; t < 2 * TN; ++t)
#pragma unroll
      for (int u = 0; u < MT; ++u) acc[t][u] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    for (int ks = wid; ks < kt; ks += NW) {
      typename F::W w[2 * TN];
      typename F::X x[MT];
#pragma unroll
      for (int t = 0; t < TN; ++t) {
        const long tile = (long)min(t0 + t, rt - 1) * kt + ks;
        w[t] = F::load_w(gate, tile, lane);
        w[TN + t] = F::load_w(up, tile, lane);
      }
      const int kb = ks * WT_K + g4 * MX_BLOCK;
#pragma unroll
      for (int u = 0; u < MT; ++u) x[u] = F::load_x(kb < A.hidden ? xp[u] + kb : nullptr);
      F::step(acc, w, x);
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < 2 * TN; ++t)
#pragma unroll
      for (int u = 0; u < MT; ++u) s_red[wid][t * MT + u][lane] = acc[t][u];
    __syncthreads();
    for (int r = wid; r < TN * MT; r += NW) {
      f32x4_t a = s_red[0][r][lane], b = s_red[0][TN * MT + r][lane];
#pragma unroll
      for (int w = 1; w < NW; ++w) {
        a += s_red[w][r][lane];
        b += s_red[w][TN * MT + r][lane];
      }
      const int n = (t0 + r / MT) * 16 + 4 * g4, m = m0 + 16 * (r % MT) + r16;
      if (m < R.count && n < A.inter) {                      // inter is a multiple of 4
        const int p = pair_of(R, m, A.ppt);
        const float w = A.pair_w[p];
#pragma unroll
        for (int i = 0; i < 4; ++i) Act<T>::store(A.h, (long)p * A.inter + n + i, w * (silu_f(a[i]) * b[i]));
      }
    }
  }
}

// part[pair] = D h[pair]
template <typename WF, typename T, int TN, int MT, int NW>
__global__ __launch_bounds__(64 * NW) void moe_down_kernel(MoeArgs<T> A) {
  using F = Fmt<WF, T>;
  __shared__ f32x4_t s_red[NW][TN * MT][64];
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int g4 = lane >> 4, r16 = lane & 15;
  const ExpertRows R = expert_rows(A, blockIdx.y);
  const int t0 = blockIdx.x * TN;
  const int rt = wt_row_tiles(A.hidden), kt = wt_k_tiles(A.inter);
  const WMat down = expert_mat(R.is_shared ? A.s_down : A.down, R.e, (long)rt * kt, tile_bytes<WF>());
  for (int m0 = 0; m0 < R.count; m0 += 16 * MT) {
    const T* hp[MT];
#pragma unroll
    for (int u = 0; u < MT; ++u)
      hp[u] = A.h + (long)pair_of(R, min(m0 + 16 * u + r16, R.count - 1), A.ppt) * A.inter;
    f32x4_t acc[TN][MT];
#pragma unroll
    for (int t = 0; t < TN; ++t)
#pragma unroll
      for (int u = 0; u < MT; ++u) acc[t][u] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    for (int ks = wid; ks < kt; ks += NW) {
      typename F::W w[TN];
      typename F::X x[MT];
#pragma unroll
      for (int t = 0; t < TN; ++t) w[t] = F::load_w(down, (long)min(t0 + t, rt - 1) * kt + ks, lane);
      const int kb = ks * WT_K + g4 * MX_BLOCK;
#pragma unroll
      for (int u = 0; u < MT; ++u) x[u] = F::load_x(kb < A.inter ? hp[u] + kb : nullptr);
      F::step(acc, w, x);
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < TN; ++t)
#pragma unroll
      for (int u = 0; u < MT; ++u) s_red[wid][t * MT + u][lane] = acc[t][u];
    __syncthreads();
    for (int r = wid; r < TN * MT; r += NW) {
      f32x4_t a = s_red[0][r][lane];
#pragma unroll
      for (int w = 1; w < NW; ++w) a += s_red[w][r][lane];
      const int n = (t0 + r / MT) * 16 + 4 * g4, m = m0 + 16 * (r % MT) + r16;
      if (m < R.count && n < A.hidden)
        *reinterpret_cast<f32x4_t*>(A.part + (long)pair_of(R, m, A.ppt) * A.hidden + n) = a;
    }
  }
}

template <typename T>
__global__ __launch_bounds__(256) void moe_combine_kernel(MoeArgs<T> A) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  const int per = A.hidden / 4;
  if (i >= (long)A.rows * per) return;
  const long t = i / per;
  const int c = (int)(i % per) * 4;
  const float* p = A.part + t * A.ppt * A.hidden + c;
  f32x4_t v = {0.f, 0.f, 0.f, 0.f};
  for (int j = 0; j < A.ppt; ++j) v += *reinterpret_cast<const f32x4_t*>(p + (long)j * A.hidden);
#pragma unroll
  for (int e = 0; e < 4; ++e) Act<T>::store(A.out, t * A.hidden + c + e, v[e]);
}

// rows of bf16 or float weights into tiles (a wave per tile)
template <typename T>
__global__ __launch_bounds__(256) void tile_weight_kernel(int n, int k, int rt, int kt, long tiles, const T* w, char* out) {
  constexpr int VE = Unit<T>::VE, PIECES = 32 / VE;
  const int lane = threadIdx.x & 63;
  const long tile = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (tile >= tiles) return;
  const int ks = (int)(tile % kt);
  const long rest = tile / kt;
  const int r = (int)(rest % rt) * WT_ROWS + (lane & 15), k0 = ks * WT_K + (lane >> 4) * MX_BLOCK;
  const bool in = r < n && k0 < k;
  const T* src = w + ((rest / rt) * n + r) * (long)k + k0;
  char* dst = out + tile * (PIECES * 1024) + lane * 16;
#pragma unroll
  for (int s = 0; s < PIECES; ++s)
    *reinterpret_cast<uint4*>(dst + s * 1024) =
        in ? *reinterpret_cast<const uint4*>(src + s * VE) : make_uint4(0u, 0u, 0u, 0u);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename T>
int launch_logits(const LogitArgs<T>& A, hipStream_t stream) {
  hipLaunchKernelGGL(moe_logits_kernel<T>, dim3((A.cols + 3) / 4, (A.rows + RT_TB - 1) / RT_TB), dim3(256), 0, stream, A);
  QM_CHECK_LAUNCH();
  return QM_OK;
}

int check_route(const char* what, int act_dtype, int rows, int hidden, int experts, int top_k, long ldx) {
  static thread_local char msg[160];
  const int unit = act_dtype == QM_ACT_BF16 ? 8 : 4;
  const char* bad = nullptr;
  int code = QM_ERR_ARG;
  if (act_dtype != QM_ACT_BF16 && act_dtype != QM_ACT_F32) { bad = "act_dtype must be QM_ACT_F32 or QM_ACT_BF16"; code = QM_ERR_DTYPE; }
  else if (rows <= 0 || rows > 4 * 65535) bad = "rows must be 1..262140";
  else if (hidden <= 0 || hidden % 32 || hidden > (1 << 20)) bad = "hidden must be a positive multiple of 32 (at most 2^20)";
  else if (experts <= 0 || experts > RT_MAX_EXPERTS) { bad = "experts must be 1..1024"; code = QM_ERR_UNSUPPORTED; }
  else if (top_k <= 0 || top_k > RT_MAX_TOPK || top_k > experts) bad = "top_k must be 1..32 and at most experts";
  else if (ldx < hidden || ldx % unit) bad = "ldx must be at least hidden and whole 16-byte units";
  if (!bad) return QM_OK;
  snprintf(msg, sizeof(msg), "%s: %s", what, bad);
  return qm_fail(code, msg);
}

struct MoeLayout {
  size_t logits, ids, pair_w, counts, lists, h, part, bytes;
};
MoeLayout moe_layout(const qm_moe_geom& g) {
  const size_t es = g.act_dtype == QM_ACT_BF16 ? 2 : 4;
  const size_t t = g.rows, ppt = g.top_k + g.shared, pairs = t * ppt;
  MoeLayout l;
  size_t at = 0;
  auto take = [&at](size_t n) { const size_t p = at; at += qm_align256(n); return p; };
  l.logits = take(t * (g.experts + 1) * sizeof(double));
  l.ids = take(t * g.top_k * sizeof(int));
  l.pair_w = take(pairs * sizeof(float));
  l.counts = take(g.experts * sizeof(int));
  l.lists = take((size_t)g.experts * t * sizeof(int));
  l.h = take(pairs * g.inter * es);
  l.part = take(pairs * g.hidden * sizeof(float));
  l.bytes = at;
  return l;
}

int check_geom(const qm_moe_geom* g, long ldx) {
  if (!g) return qm_fail(QM_ERR_ARG, "qm_moe: null geometry");
  const int rc = check_route("qm_moe", g->act_dtype, g->rows, g->hidden, g->experts, g->top_k, ldx);
  if (rc) return rc;
  if (g->inter <= 0 || g->inter % 32 || g->inter > (1 << 20))
    return qm_fail(QM_ERR_ARG, "qm_moe: inter must be a positive multiple of 32 (at most 2^20)");
  if (g->shared < 0 || g->shared > 32) return qm_fail(QM_ERR_ARG, "qm_moe: shared must be 0..32");
  if (g->weight_format != QM_W_ACT && g->weight_format != QM_W_MX4)
    return qm_fail(QM_ERR_DTYPE, "qm_moe: weight_format must be QM_W_ACT or QM_W_MX4");
  return QM_OK;
}

template <typename WF, typename T>
int launch_ffn(const MoeArgs<T>& A, hipStream_t stream) {
  constexpr int TN = 1, MT = 2, NW = 8, TD = 2, ND = 4;
  hipLaunchKernelGGL((moe_up_kernel<WF, T, TN, MT, NW>), dim3((wt_row_tiles(A.inter) + TN - 1) / TN, A.shared + A.experts),
                     dim3(64 * NW), 0, stream, A);
  QM_CHECK_LAUNCH();
  hipLaunchKernelGGL((moe_down_kernel<WF, T, TD, MT, ND>),
                     dim3((wt_row_tiles(A.hidden) + TD - 1) / TD, A.shared + A.experts), dim3(64 * ND), 0, stream, A);
  QM_CHECK_LAUNCH();
  const long n = (long)A.rows * (A.hidden / 4);
  hipLaunchKernelGGL(moe_combine_kernel<T>, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream, A);
  QM_CHECK_LAUNCH();
  return QM_OK;
}

template <typename T, typename WPlain>
int run_moe(const qm_moe_geom& g, const qm_moe_weights& w, const void* x, long ldx, void* out, char* ws,
            hipStream_t stream) {
  const MoeLayout l = moe_layout(g);
  LogitArgs<T> L = {static_cast<const T*>(x), ldx, static_cast<const T*>(w.router), static_cast<const T*>(w.shared_router),
                    reinterpret_cast<double*>(ws + l.logits), g.rows, g.hidden, g.experts,
                    g.experts + (w.shared_router && g.shared ? 1 : 0)};
  int rc = launch_logits<T>(L, stream);
  if (rc) return rc;
  int* ids = reinterpret_cast<int*>(ws + l.ids);
  float* pair_w = reinterpret_cast<float*>(ws + l.pair_w);
  int* counts = reinterpret_cast<int*>(ws + l.counts);
  int* lists = reinterpret_cast<int*>(ws + l.lists);
  const int ppt = g.top_k + g.shared;
  hipLaunchKernelGGL(moe_topk_kernel, dim3((g.rows + 3) / 4), dim3(256), 0, stream, L.logits, g.rows, L.cols, g.experts,
                     g.top_k, g.normalize, ids, pair_w, ppt, g.shared);
  QM_CHECK_LAUNCH();
  hipLaunchKernelGGL(moe_lists_kernel, dim3(g.experts), dim3(256), 0, stream, ids, g.rows, g.top_k, ppt, counts, lists);
  QM_CHECK_LAUNCH();
  MoeArgs<T> A = {};
  A.x = L.x; A.ldx = ldx; A.rows = g.rows; A.hidden = g.hidden; A.inter = g.inter; A.experts = g.experts;
  A.shared = g.shared; A.top_k = g.top_k; A.ppt = ppt;
  const bool mx = g.weight_format == QM_W_MX4;
  auto mat = [mx](const void* d, const void* s) { return WMat{d, mx ? static_cast<const uint8_t*>(s) : nullptr}; };
  A.gate = mat(w.gate, w.gate_scales); A.up = mat(w.up, w.up_scales); A.down = mat(w.down, w.down_scales);
  A.s_gate = mat(w.shared_gate, w.shared_gate_scales); A.s_up = mat(w.shared_up, w.shared_up_scales);
  A.s_down = mat(w.shared_down, w.shared_down_scales);
  A.counts = counts; A.lists = lists; A.pair_w = pair_w;
  A.h = reinterpret_cast<T*>(ws + l.h);
  A.part = reinterpret_cast<float*>(ws + l.part);
  A.out = static_cast<T*>(out);
  return mx ? launch_ffn<WMx4, T>(A, stream) : launch_ffn<WPlain, T>(A, stream);
}

}  // namespace

extern "C" int qm_tile_weight(int act_dtype, int mats, int n, int k, const void* w, void* tiles, hipStream_t stream) {
  if (act_dtype != QM_ACT_BF16 && act_dtype != QM_ACT_F32)
    return qm_fail(QM_ERR_DTYPE, "qm_tile_weight: act_dtype must be QM_ACT_F32 or QM_ACT_BF16");
  if (mats <= 0 || n <= 0 || k <= 0 || k % 32 || n > (1 << 24) || k > (1 << 20))
    return qm_fail(QM_ERR_ARG, "qm_tile_weight: mats and n must be positive, k a positive multiple of 32 (n <= 2^24, k <= 2^20)");
  if (!w || !tiles) return qm_fail(QM_ERR_ARG, "qm_tile_weight: null pointer");
  if (!aligned16(w) || !aligned16(tiles)) return qm_fail(QM_ERR_ARG, "qm_tile_weight: w and tiles must be 16-byte aligned");
  const int rt = wt_row_tiles(n), kt = wt_k_tiles(k);
  const long total = (long)mats * rt * kt, nb = (total + 3) / 4;
  if (nb > 0x7fffffffL / 256) return qm_fail(QM_ERR_UNSUPPORTED, "qm_tile_weight: too many tiles for one launch");
  if (act_dtype == QM_ACT_BF16)
    hipLaunchKernelGGL(tile_weight_kernel<bf16_t>, dim3((unsigned)nb), dim3(256), 0, stream, n, k, rt, kt, total,
                       static_cast<const bf16_t*>(w), static_cast<char*>(tiles));
  else
    hipLaunchKernelGGL(tile_weight_kernel<float>, dim3((unsigned)nb), dim3(256), 0, stream, n, k, rt, kt, total,
                       static_cast<const float*>(w), static_cast<char*>(tiles));
  QM_CHECK_LAUNCH();
  return QM_OK;
}

extern "C" size_t qm_moe_route_workspace(int rows, int experts) {
  if (rows <= 0 || experts <= 0 || experts > RT_MAX_EXPERTS) return 0;
  return qm_align256((size_t)rows * experts * sizeof(double));
}

extern "C" int qm_moe_route(int act_dtype, int rows, int hidden, int experts, int top_k, int normalize, const void* x,
                            long ldx, const void* router, int* ids, float* weights, void* workspace,
                            size_t workspace_bytes, hipStream_t stream) {
  int rc = check_route("qm_moe_route", act_dtype, rows, hidden, experts, top_k, ldx);
  if (rc) return rc;
  if (!x || !router || !ids || !weights || !workspace) return qm_fail(QM_ERR_ARG, "qm_moe_route: null pointer");
  if (!aligned16(x) || !aligned16(router) || !aligned16(workspace))
    return qm_fail(QM_ERR_ARG, "qm_moe_route: x, router and workspace must be 16-byte aligned");
  if (workspace_bytes < qm_moe_route_workspace(rows, experts))
    return qm_fail(QM_ERR_WORKSPACE, "qm_moe_route: workspace too small");
  double* logits = static_cast<double*>(workspace);
  if (act_dtype == QM_ACT_BF16) {
    LogitArgs<bf16_t> L = {static_cast<const bf16_t*>(x), ldx, static_cast<const bf16_t*>(router), nullptr, logits, rows,
                           hidden, experts, experts};
    rc = launch_logits<bf16_t>(L, stream);
  } else {
    LogitArgs<float> L = {static_cast<const float*>(x), ldx, static_cast<const float*>(router), nullptr, logits, rows,
                          hidden, experts, experts};
    rc = launch_logits<float>(L, stream);
  }
  if (rc) return rc;
  hipLaunchKernelGGL(moe_topk_kernel, dim3((rows + 3) / 4), dim3(256), 0, stream, logits, rows, experts, experts, top_k,
                     normalize, ids, weights, top_k, 0);
  QM_CHECK_LAUNCH();
  return QM_OK;
}

extern "C" size_t qm_moe_workspace(const qm_moe_geom* g) {
  if (check_geom(g, g ? g->hidden : 0)) return 0;
  return moe_layout(*g).bytes;
}

extern "C" int qm_moe(const qm_moe_geom* g, const qm_moe_weights* w, const void* x, long ldx, void* out, void* workspace,
                      size_t workspace_bytes, hipStream_t stream) {
  const int rc = check_geom(g, ldx);
  if (rc) return rc;
  if (!w || !x || !out || !workspace) return qm_fail(QM_ERR_ARG, "qm_moe: null pointer");
  const void* need[] = {w->router, w->gate, w->up, w->down, w->shared_gate, w->shared_up, w->shared_down};
  const void* scales[] = {w->gate_scales, w->up_scales, w->down_scales, w->shared_gate_scales, w->shared_up_scales,
                          w->shared_down_scales};
  for (int i = 0; i < (g->shared ? 7 : 4); ++i)
    if (!need[i] || !aligned16(need[i])) return qm_fail(QM_ERR_ARG, "qm_moe: a weight is null or not 16-byte aligned");
  if (g->weight_format == QM_W_MX4)
    for (int i = 0; i < (g->shared ? 6 : 3); ++i)
      if (!scales[i]) return qm_fail(QM_ERR_ARG, "qm_moe: null scales");
  if (!aligned16(x) || !aligned16(out) || !aligned16(workspace) || (w->shared_router && !aligned16(w->shared_router)))
    return qm_fail(QM_ERR_ARG, "qm_moe: x, out, workspace and shared_router must be 16-byte aligned");
  const MoeLayout l = moe_layout(*g);
  if (workspace_bytes < l.bytes) return qm_fail(QM_ERR_WORKSPACE, "qm_moe: workspace too small (see qm_moe_workspace)");
  char* ws = static_cast<char*>(workspace);
  if (g->act_dtype == QM_ACT_BF16) return run_moe<bf16_t, WBf16>(*g, *w, x, ldx, out, ws, stream);
  return run_moe<float, WF32>(*g, *w, x, ldx, out, ws, stream);
}
