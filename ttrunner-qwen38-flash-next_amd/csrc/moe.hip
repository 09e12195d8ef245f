// Mixture-of-experts layer, gfx950: the chosen experts' gated FFN
// (reference/model.py:387-417), routed as route.hip does.
//
//   y[t]    = sum_j w[t][j] D_e (silu(G_e x[t]) * (U_e x[t])),   e = ids[t][j]
//           + sigmoid(x[t] . r) sum_s (shared expert s of x[t])
//
// A pair is a (token, expert) choice; pair (top_k + shared) t + j is choice j of
// token t, the shared experts its last ones. The pair's weight multiplies the
// hidden row in float before that is rounded to the activations' type, so the second
// products add up unweighted, in the order of j. That rounding is the second
// product's bf16 operand: one MFMA a piece and half of a float row's bytes; it adds as
// much error as the output's own rounding (relative error of the layer 2.3e-3 where
// float hidden rows would leave 1.7e-3). Float activations keep float hidden rows.
#include "moe_internal.h"
#include "moe_topk.h"
#include "wgemm.h"

namespace {

template <typename T>
struct MoeArgs {
  const T* x;
  long ldx;
  int rows, hidden, inter, experts, shared, top_k, ppt;
  WMat gate, up, down, s_gate, s_up, s_down;
  const int* counts;
  const int* lists;
  const int* n_tiles;
  const int2* tiles;   // row tiles of the many-row kernels
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
// ---------------------------------------------------------------------------
// A few tokens (at most FEW): the logits, the up products and the down products,
// three launches over the chosen experts' weights alone.
//
// An operand holds 16 activation rows: all tokens' rows stand in it, whichever
// expert is multiplied, and a column counts where its token chose the expert. A
// slot is a shared expert or one of the distinct chosen ones, in the order of
// their numbers. A single token's workgroups rank its logits for themselves (a
// launch of its own for that takes longer); for several tokens one workgroup
// does and leaves the table of slots.
//
// What bounds it is the weights' way from memory. 8 of 128 experts of 2048 x 512 and
// a shared one: one token, bf16, 57 MB: logits 3.1 us, up 10 to 11.6 (2 of them the
// ranking), down 6; 9 tokens, 4-bit, 96 MB: 4.2, table 4.6, up 15 (4.2 TB/s), down
// 11.5. Against the many-token kernels: 8 tokens, 4-bit, 34 for 39 us, 16 tokens 46 and
// 46, bf16 98 for 108.
// ---------------------------------------------------------------------------
constexpr int FEW = 16;
// Waves of a workgroup. Down products of 9 tokens, 4-bit: 16 waves with four units in
// flight each 14.8 us, 8 with eight 16.7 (one workgroup a tile).
constexpr int FEW_UP_NW = 8, FEW_DOWN_NW = 16;

template <typename T>
struct FewArgs {
  MoeArgs<T> m;
  const double* logits;
  int cols, normalize;
  int* n_slots;        // of the table
  int* slot_expert;    // [slot] expert; of a shared one -1 - its number
  int* slot_pair;      // [slot][16] the pair of each column, -1 where none
  float* slot_w;       // [slot][16] its weight
  int split;           // workgroups of an output tile in the down products
  float* down_part;    // [output tile][split][16 outputs][16] their sums
  unsigned* down_done; // [output tile] how many have theirs there, cleared before
};

// choice `lane` of a token and its weight, by one wave. The exponential is a float of a
// difference taken in double, and so is the sum of up to 32 (or all) of them: a weight
// is off by some 1e-7 of it, far below the rounding that the hidden row sees.
template <int PER>
__device__ __forceinline__ int wave_choose(const double* l, int experts, int top_k, int normalize, int lane, float& weight) {
  long long key;
  int id;
  if (!wave_topk<PER>(l, experts, top_k, 0.0, lane, key, id, [](const int (&)[RT_EXACT]) { return 0.0; }))
    wave_topk_exact(l, experts, top_k, lane, key, id);
  const double v0 = key_logit(lane_key(key, 0));
  const float mine = lane < top_k ? expf((float)(key_logit(key) - v0)) : 0.f;
  float sum = mine;
  if (!normalize) {
    sum = 0.f;
    for (int i = lane; i < experts; i += 64) sum += expf((float)(l[i] - v0));
  }
  weight = mine / wave_sum(sum);
  return id;
}
template <typename T> __device__ __forceinline__ float shared_weight(const FewArgs<T>& A, int t) {
  return A.cols > A.m.experts ? sigmoid_f((float)A.logits[(long)t * A.cols + A.m.experts]) : 1.f;
}

template <typename T> __device__ __forceinline__ void clear_down(const FewArgs<T>& A, int i, int threads) {
  if (A.split > 1)
    for (; i < wt_row_tiles(A.m.hidden); i += threads) A.down_done[i] = 0u;
}

// The table of slots, by one workgroup with a wave per token
template <typename T, int PER>
__global__ __launch_bounds__(64 * FEW) void moe_few_plan_kernel(FewArgs<T> A) {
  __shared__ int s_ids[FEW][RT_MAX_TOPK];
  __shared__ float s_w[FEW][RT_MAX_TOPK];
  __shared__ unsigned s_map[RT_MAX_EXPERTS / 32];
  __shared__ int s_before[RT_MAX_EXPERTS / 32 + 1];
  const MoeArgs<T>& M = A.m;
  const int lane = threadIdx.x & 63, t = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (threadIdx.x < RT_MAX_EXPERTS / 32) s_map[threadIdx.x] = 0u;
  __syncthreads();
  if (t < M.rows) {
    float w;
    const int id = wave_choose<PER>(A.logits + (long)t * A.cols, M.experts, M.top_k, A.normalize, lane, w);
    if (lane < M.top_k) {
      s_ids[t][lane] = id;
      s_w[t][lane] = w;
      atomicOr(&s_map[id >> 5], 1u << (id & 31));
    }
  }
  // every column of every slot none, before the choices fill theirs
  const int most = M.shared + min(M.rows * M.top_k, M.experts);
  for (int i = threadIdx.x; i < most * 16; i += 64 * FEW) A.slot_pair[i] = -1;
  clear_down(A, threadIdx.x, 64 * FEW);
  __syncthreads();
  if (threadIdx.x == 0) {
    int n = M.shared;
    for (int i = 0; i < RT_MAX_EXPERTS / 32; ++i) {
      s_before[i] = n;
      n += __popc(s_map[i]);
    }
    *A.n_slots = n;
  }
  __syncthreads();
  if (t < M.rows && lane < M.top_k) {
    const int e = s_ids[t][lane], slot = s_before[e >> 5] + __popc(s_map[e >> 5] & ((1u << (e & 31)) - 1u));
    A.slot_expert[slot] = e;                                 // the same value from every token that chose it
    A.slot_pair[slot * 16 + t] = t * M.ppt + lane;
    A.slot_w[slot * 16 + t] = s_w[t][lane];
  }
  if (t < M.rows && lane < M.shared) {
    A.slot_expert[lane] = -1 - lane;
    A.slot_pair[lane * 16 + t] = t * M.ppt + M.top_k + lane;
    A.slot_w[lane * 16 + t] = shared_weight(A, t);
  }
}

// h of a slot: a workgroup per 16 TN hidden units and slot, the waves split k (a
// wave's loads are whole lines of tiles; the partial results meet in LDS). TN: 4-bit
// weights are few bytes beside the activations' operands, so two row tiles share
// them (16 tokens of 8 of 128 experts, us with one / two: 4-bit 22.6 / 18.8, bf16
// 54.8 / 61.2).
template <typename WF, typename T, int PER, bool ONE, int TN>
__global__ __launch_bounds__(64 * FEW_UP_NW) void moe_few_up_kernel(FewArgs<T> A) {
  using F = Fmt<WF, T>;
  constexpr int NW = FEW_UP_NW, KP = 2;                      // k tiles in flight
  __shared__ f32x4_t s_red[NW][2 * TN][64];
  __shared__ int s_id[RT_MAX_TOPK];
  __shared__ float s_w[RT_MAX_TOPK];
  const MoeArgs<T>& M = A.m;
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g4 = lane >> 4, r16 = lane & 15;
  const int kt = wt_k_tiles(M.hidden), rt = wt_row_tiles(M.inter), slot = blockIdx.y;
  const T* row = M.x + (long)min(r16, M.rows - 1) * M.ldx;
  Acts<F, T> pre[KP];                                        // before it is known which expert
  if constexpr (ONE) {
#pragma unroll
    for (int p = 0; p < KP; ++p) pre[p].load(row, min(wid + p * NW, kt - 1), M.hidden, g4);
  }
  int e, pair = -1;
  float weight = 0.f;
  if constexpr (ONE) {
    if (slot < M.shared) {
      e = -1 - slot;
      weight = shared_weight(A, 0);
    } else {
      if (wid == 0) {
        float w;
        const int id = wave_choose<PER>(A.logits, M.experts, M.top_k, A.normalize, lane, w);
        if (lane < M.top_k) { s_id[lane] = id; s_w[lane] = w; }
      }
      __syncthreads();
      e = __builtin_amdgcn_readfirstlane(s_id[slot - M.shared]);
      weight = s_w[slot - M.shared];
    }
    if (r16 == 0) pair = slot < M.shared ? M.top_k + slot : slot - M.shared;
    if (blockIdx.x == 0 && threadIdx.x < 16) {               // for the down products
      A.slot_pair[slot * 16 + threadIdx.x] = pair;
      if (threadIdx.x == 0) A.slot_expert[slot] = e;
      if (threadIdx.x == 0 && slot == 0) *A.n_slots = gridDim.y;
      if (slot == 0) clear_down(A, threadIdx.x, 16);
    }
  } else {
    // (one round trip: what stands behind the last slot is read but not used)
    const int n = *A.n_slots;
    e = A.slot_expert[slot];
    pair = A.slot_pair[slot * 16 + r16];
    weight = A.slot_w[slot * 16 + r16];
    if (slot >= n) return;
  }
  const WMat gate = expert_mat(e < 0 ? M.s_gate : M.gate, e < 0 ? -1 - e : e, (long)rt * kt, F::TILE);
  const WMat up = expert_mat(e < 0 ? M.s_up : M.up, e < 0 ? -1 - e : e, (long)rt * kt, F::TILE);
  f32x4_t acc[2 * TN][1];
  clear(acc);
  for (int k0 = wid; k0 < kt; k0 += NW * KP) {
    typename F::W w[KP][2 * TN];
    Acts<F, T> x[KP][1];
#pragma unroll
    for (int p = 0; p < KP; ++p) {
      const int ks = min(k0 + p * NW, kt - 1);
#pragma unroll
      for (int t = 0; t < TN; ++t) {
        const long tile = (long)min((int)blockIdx.x * TN + t, rt - 1) * kt + ks;
        w[p][t] = F::load_w(gate, tile, lane);
        w[p][TN + t] = F::load_w(up, tile, lane);
      }
      // (several tokens: the columns that did not choose the expert load nothing)
      if (ONE && k0 == wid) x[p][0] = pre[p];
      else x[p][0].load(row, ks, ONE || pair >= 0 ? M.hidden : 0, g4);
    }
#pragma unroll
    for (int p = 0; p < KP; ++p)
      if (k0 + p * NW < kt) step_tile<F, T>(acc, w[p], x[p]);
  }
#pragma unroll
  for (int t = 0; t < 2 * TN; ++t) s_red[wid][t][lane] = acc[t][0];
  __syncthreads();
  if (wid >= TN || pair < 0) return;
  f32x4_t a = s_red[0][wid][lane], b = s_red[0][TN + wid][lane];
#pragma unroll
  for (int w = 1; w < NW; ++w) {
    a += s_red[w][wid][lane];
    b += s_red[w][TN + wid][lane];
  }
  const int n = (blockIdx.x * TN + wid) * 16 + 4 * g4;
  if (n >= M.inter) return;
  f32x4_t v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = weight * (silu_f(a[i]) * b[i]);
  store_act4(M.h + (long)pair * M.inter + n, v);
}

// out: a workgroup per 16 outputs, or `split` of them; the waves share the (slot,
// k tile) units. Of several workgroups the last to finish adds their sums, in the
// order of their numbers.
template <typename WF, typename T>
__global__ __launch_bounds__(64 * FEW_DOWN_NW) void moe_few_down_kernel(FewArgs<T> A) {
  using F = Fmt<WF, T>;
  // units in flight, as many as 128 registers hold
  constexpr int NW = FEW_DOWN_NW, U = F::SCALED ? (sizeof(T) == 2 ? 4 : 2) : sizeof(T) == 2 ? 3 : 1;
  __shared__ f32x4_t s_red[NW][64];
  const MoeArgs<T>& M = A.m;
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g4 = lane >> 4, r16 = lane & 15;
  const int kt = wt_k_tiles(M.inter), rt = wt_row_tiles(M.hidden);
  const int units = *A.n_slots * kt, stride = NW * A.split, first = NW * blockIdx.y + wid;
  f32x4_t total = {0.f, 0.f, 0.f, 0.f};
  // a batch's slots are looked up while the one before is multiplied, the first
  // while their number is on its way (what stands behind the last is not used)
  const int most = M.shared + min(M.rows * M.top_k, M.experts);
  int expert[U], pair[U], at[U];
  int slot = first / kt, ks = first % kt;                    // of the next unit to look up
  const int slot_step = stride / kt, ks_step = stride % kt;
  auto look_up = [&]() {
#pragma unroll
    for (int p = 0; p < U; ++p) {
      const int s = min(slot, most - 1);
      expert[p] = A.slot_expert[s];
      pair[p] = A.slot_pair[s * 16 + r16];
      at[p] = ks;
      slot += slot_step;
      ks += ks_step;
      if (ks >= kt) { ks -= kt; ++slot; }
    }
  };
  look_up();
  for (int u0 = first; u0 < units; u0 += stride * U) {
    typename F::W w[U][1];
    Acts<F, T> x[U][1];
    bool mine[U];
#pragma unroll
    for (int p = 0; p < U; ++p) {
      const bool in = u0 + p * stride < units;
      const int e = in ? expert[p] : 0;
      const WMat down = expert_mat(e < 0 ? M.s_down : M.down, e < 0 ? -1 - e : e, (long)rt * kt, F::TILE);
      w[p][0] = F::load_w(down, (long)blockIdx.x * kt + at[p], lane);
      // (columns that did not choose the expert load nothing: most of them)
      mine[p] = in && pair[p] >= 0;
      x[p][0].load(M.h + (long)(mine[p] ? pair[p] : 0) * M.inter, at[p], mine[p] ? M.inter : 0, g4);
    }
    look_up();
#pragma unroll
    for (int p = 0; p < U; ++p) {
      if (u0 + p * stride >= units) continue;
      f32x4_t acc[1][1];
      clear(acc);
      step_tile<F, T>(acc, w[p], x[p]);
      // a token that did not choose the expert takes nothing from it, whatever it is
#pragma unroll
      for (int i = 0; i < 4; ++i) total[i] += mine[p] ? acc[0][0][i] : 0.f;
    }
  }
  s_red[wid][lane] = total;
  __syncthreads();
  if (wid != 0) return;
  f32x4_t v = s_red[0][lane];
#pragma unroll
  for (int w = 1; w < NW; ++w) v += s_red[w][lane];
  if (A.split > 1) {
    float* parts = A.down_part + ((long)blockIdx.x * A.split * 64 + lane) * 4;
    unsigned* mine = reinterpret_cast<unsigned*>(parts + blockIdx.y * 256);
#pragma unroll
    for (int i = 0; i < 4; ++i) st_flag(mine + i, __float_as_uint(v[i]));
    wait_all_memory();                                       // the wave's stores, before they are counted
    unsigned before = 0u;
    if (lane == 0) before = __hip_atomic_fetch_add(A.down_done + blockIdx.x, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if ((int)__builtin_amdgcn_readfirstlane(before) != A.split - 1) return;
    v = f32x4_t{0.f, 0.f, 0.f, 0.f};
    for (int p = 0; p < A.split; ++p)
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] += __uint_as_float(ld_flag(reinterpret_cast<const unsigned*>(parts + p * 256) + i));
  }
  const int n = blockIdx.x * 16 + 4 * g4;
  if (r16 < M.rows && n < M.hidden) store_act4(M.out + (long)r16 * M.hidden + n, v);
}

// ---------------------------------------------------------------------------
// Many tokens: routing, the experts' lists of pairs, the up products, the down
// products of every pair, and their sum per token.
//
// 2000 tokens, 8 of 64 experts of 2048 x 768 and a shared one, bf16: routing 30 us, up
// 163, down 124, sum 25. The up products read 400 MB of weights and do 113 GFLOP (a
// quarter more with the experts' last tiles filled up): 620 MB from behind the L2 at
// 3.9 TB/s and 870 TFLOP/s at once, neither alone at its limit. 128 tokens, 4-bit, 8 of
// 128 of 2048 x 512: up 30 us, down 19, the weights at 4.6 and 3.8 TB/s.
// ---------------------------------------------------------------------------
// A workgroup (wgemm.h) per row tile of the table and range of weight rows, the
// ranges of a tile side by side on an XCD. Of a wave's TN row tiles the first half
// are gate rows, the others the up rows of the same hidden units.
template <typename WF, typename T, int TN, int TM, int WN, int WM, int S, bool STREAM>
__global__ __launch_bounds__(64 * WN * WM, 2) void moe_up_gemm_kernel(MoeArgs<T> A) {
  using G = SpanGemm<WF, T, TN, TM, WN, WM, S, STREAM>;
  constexpr int HN = TN / 2;
  extern __shared__ __attribute__((aligned(16))) char s_buf[];
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rt = wt_row_tiles(A.inter), kt = wt_k_tiles(A.hidden);
  const int nt = (rt + HN * WN - 1) / (HN * WN), items = *A.n_tiles * nt;
  if ((int)blockIdx.x >= items) return;
  const int item = xcd_run(blockIdx.x, items);
  const int2 tile = A.tiles[item / nt];
  const ExpertRows R = expert_rows(A, tile.x);
  const int t0 = item % nt * WN * HN;
  const WMat gate = expert_mat(R.is_shared ? A.s_gate : A.gate, R.e, (long)rt * kt, G::F::TILE);
  const WMat up = expert_mat(R.is_shared ? A.s_up : A.up, R.e, (long)rt * kt, G::F::TILE);
  auto first = [&](int q) { return (long)min(t0 + q / TN * HN + q % HN, rt - 1) * kt; };
  auto row = [&](int i) { return A.x + (long)(pair_of(R, min(tile.y + i, R.count - 1), A.ppt) / A.ppt) * A.ldx; };
  auto weight = [&](int q) { return static_cast<const char*>(q % TN < HN ? gate.data : up.data) + first(q) * G::F::TILE; };
  const typename G::Src src =
      G::source(wid, lane, row, weight, [&](int q) { return (q % TN < HN ? gate.scales : up.scales) + first(q) * 64; });
  f32x4_t acc[TN][TM];
  clear(acc);
  G::run(acc, s_buf, src, A.hidden, R.count - tile.y);
#pragma unroll
  for (int u = 0; u < TM; ++u) {
    const int m = tile.y + (wid % WM) * 16 * TM + 16 * u + (lane & 15);
    if (m >= R.count) continue;
    const int p = pair_of(R, m, A.ppt);
    const float w = A.pair_w[p];
#pragma unroll
    for (int t = 0; t < HN; ++t) {
      const int n = (t0 + wid / WM * HN + t) * 16 + 4 * (lane >> 4);
      if (n >= A.inter) continue;
      f32x4_t v;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = w * (silu_f(acc[t][u][i]) * acc[HN + t][u][i]);
      store_act4(A.h + (long)p * A.inter + n, v);
    }
  }
}

template <typename WF, typename T, int TN, int TM, int WN, int WM, int S, bool STREAM>
__global__ __launch_bounds__(64 * WN * WM, 2) void moe_down_gemm_kernel(MoeArgs<T> A) {
  using G = SpanGemm<WF, T, TN, TM, WN, WM, S, STREAM>;
  extern __shared__ __attribute__((aligned(16))) char s_buf[];
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rt = wt_row_tiles(A.hidden), kt = wt_k_tiles(A.inter);
  const int nt = (rt + TN * WN - 1) / (TN * WN), items = *A.n_tiles * nt;
  if ((int)blockIdx.x >= items) return;
  const int item = xcd_run(blockIdx.x, items);
  const int2 tile = A.tiles[item / nt];
  const ExpertRows R = expert_rows(A, tile.x);
  const int t0 = item % nt * WN * TN;
  const WMat down = expert_mat(R.is_shared ? A.s_down : A.down, R.e, (long)rt * kt, G::F::TILE);
  auto first = [&](int q) { return (long)min(t0 + q, rt - 1) * kt; };
  auto row = [&](int i) { return A.h + (long)pair_of(R, min(tile.y + i, R.count - 1), A.ppt) * A.inter; };
  auto weight = [&](int q) { return static_cast<const char*>(down.data) + first(q) * G::F::TILE; };
  const typename G::Src src = G::source(wid, lane, row, weight, [&](int q) { return down.scales + first(q) * 64; });
  f32x4_t acc[TN][TM];
  clear(acc);
  G::run(acc, s_buf, src, A.inter, R.count - tile.y);
#pragma unroll
  for (int u = 0; u < TM; ++u) {
    const int m = tile.y + (wid % WM) * 16 * TM + 16 * u + (lane & 15);
    if (m >= R.count) continue;
    float* o = A.part + (long)pair_of(R, m, A.ppt) * A.hidden;
#pragma unroll
    for (int t = 0; t < TN; ++t) {
      const int n = (t0 + wid / WM * TN + t) * 16 + 4 * (lane >> 4);
      if (n < A.hidden) store_act4(o + n, acc[t][u]);
    }
  }
}

// y[t] = the sum of its pairs' products, in their order (a thread per 16 bytes of
// the output): a stream (2000 tokens of 9 pairs, 156 MB, 25 us). The products stay in float: in bf16 their rounding would add as much
// error again as the hidden rows' (2000 tokens of 9 pairs: relative error 2.9e-3
// for 2.4e-3, and 21 us of 339 saved).
template <typename T>
__global__ __launch_bounds__(256) void moe_combine_kernel(MoeArgs<T> A) {
  constexpr int VE = 16 / sizeof(T);
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  const int per = A.hidden / VE;
  if (i >= (long)A.rows * per) return;
  const long t = i / per;
  const int c = (int)(i % per) * VE;
  const float* p = A.part + t * A.ppt * A.hidden + c;
  f32x4_t v[VE / 4];
#pragma unroll
  for (int e = 0; e < VE / 4; ++e) v[e] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  for (int j = 0; j < A.ppt; ++j)
#pragma unroll
    for (int e = 0; e < VE / 4; ++e) v[e] += *reinterpret_cast<const f32x4_t*>(p + (long)j * A.hidden + 4 * e);
#pragma unroll
  for (int e = 0; e < VE / 4; ++e) store_act4(A.out + t * A.hidden + c + 4 * e, v[e]);
}

// rows of bf16 or float weights into tiles (a wave per tile): once, when the weights
// are made (128 experts of 2048 x 512, 268 MB there and back, 92 us)
template <typename T>
__global__ __launch_bounds__(256) void tile_weight_kernel(int n, int k, int rt, int kt, long tiles, const T* w, char* out) {
  constexpr int VE = 16 / sizeof(T), PIECES = 32 / VE;
  const int lane = threadIdx.x & 63;
  const long tile = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (tile >= tiles) return;
  const int ks = (int)(tile % kt);
  const long rest = tile / kt;
  const int r = (int)(rest % rt) * WT_ROWS + (lane & 15);
  const T* src = w + ((rest / rt) * n + r) * (long)k;
  char* dst = out + tile * (PIECES * 1024) + lane * 16;
#pragma unroll
  for (int s = 0; s < PIECES; ++s) {
    // piece s / HALVES of 8 k, its half s % HALVES
    constexpr int HALVES = 8 / VE;
    const int k0 = ks * WT_K + 32 * (s / HALVES) + 8 * (lane >> 4) + s % HALVES * VE;
    *reinterpret_cast<uint4*>(dst + s * 1024) =
        r < n && k0 < k ? *reinterpret_cast<const uint4*>(src + k0) : make_uint4(0u, 0u, 0u, 0u);
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

struct MoeLayout {
  size_t logits, norms, ids, pair_w, counts, lists, meta, tiles, h, part, done, bytes;
  long max_tiles;      // of row tiles of bm rows
  int bm;
};

// Activation rows of a tile of the many-token kernels, by the rows that an expert
// has on average (us a layer, 8 experts of a token):
//   bf16 weights, 128 experts of 2048 x 512, tiles of 32 / 64 / 128 rows: 8 rows 152 /
//     169 / 170, 25 rows 206 / 195 / 204, 62 rows 262 / 234 / 228; 64 of 2048 x 768:
//     250 rows 493 / 357 / 312
//   4-bit weights, 32 / 64: 8 rows 67 / 82, 31 rows 109 / 112, 125 rows 209 / 212, 375
//     rows (2048 x 768) 341 / 339, 750 rows 642 / 620
//   float activations, 25 rows, 16 / 32: float weights 419 / 400, 4-bit ones 193 / 217;
//     125 rows: 1308 / 1168, 614 / 677
int rows_per_tile(const qm_moe_geom& g) {
  const double avg = (double)g.rows * g.top_k / g.experts;
  const bool mx = g.weight_format == QM_W_MX4;
  if (g.act_dtype != QM_ACT_BF16) return mx ? 16 : 32;
  if (mx) return avg < 512 ? 32 : 64;
  return avg < 20 ? 32 : avg < 48 ? 64 : 128;
}
// Workgroups of an output tile in the few tokens' down products: two where the tiles
// alone leave half of the CUs without one and a wave has some six units of work (us,
// 8 of 128 experts of 2048 x 512, with one / two: 4-bit 2 tokens 6.3 / 8.0, 3 tokens
// 9.5 / 8.0, 9 tokens 15.2 / 11.2; bf16 9 tokens 29.6 / 24.8; 4096 x 1024, 256
// tiles, 8 tokens 32.6 / 39.0; four are slower everywhere)
int down_split(const qm_moe_geom& g) {
  const long choices = (long)g.rows * g.top_k, slots = g.shared + (choices < g.experts ? choices : g.experts);
  return wt_row_tiles(g.hidden) <= 128 && slots * wt_k_tiles(g.inter) >= 6 * FEW_DOWN_NW ? 2 : 1;
}
// The few-token kernels take the table of slots where the others keep the lists.
MoeLayout moe_layout(const qm_moe_geom& g) {
  const size_t es = g.act_dtype == QM_ACT_BF16 ? 2 : 4;
  const size_t t = g.rows, ppt = g.top_k + g.shared, pairs = t * ppt;
  const size_t choices = t * g.top_k, hot = choices < (size_t)g.experts ? choices : (size_t)g.experts;
  MoeLayout l = {};
  size_t at = 0;
  auto take = [&at](size_t n) { const size_t p = at; at += qm_align256(n); return p; };
  l.logits = take(t * (g.experts + 1) * sizeof(double));
  l.meta = take(2 * sizeof(int));
  l.h = take(pairs * g.inter * es);
  if (g.rows <= FEW) {
    l.counts = take((g.shared + hot) * sizeof(int));          // slot_expert
    l.lists = take((g.shared + hot) * 16 * sizeof(int));      // slot_pair
    l.pair_w = take((g.shared + hot) * 16 * sizeof(float));   // slot_w
    const size_t split = down_split(g);
    l.part = take(split > 1 ? wt_row_tiles(g.hidden) * split * 256 * sizeof(float) : 0);
    l.done = take(split > 1 ? wt_row_tiles(g.hidden) * sizeof(unsigned) : 0);
  } else {
    l.bm = rows_per_tile(g);
    // every expert's last tile may be part-filled
    l.max_tiles = (long)(choices / l.bm + hot + g.shared * ((t + l.bm - 1) / l.bm));
    l.norms = take(qm_route_norms(g.rows, g.experts));
    l.ids = take(choices * sizeof(int));
    l.pair_w = take(pairs * sizeof(float));
    l.counts = take((g.experts + 1) * sizeof(int));           // and the number of finished workgroups
    l.lists = take((size_t)g.experts * t * sizeof(int));
    l.tiles = take(l.max_tiles * sizeof(int2));
    l.part = take(pairs * g.hidden * sizeof(float));
  }
  l.bytes = at;
  return l;
}

int check_geom(const qm_moe_geom* g, long ldx) {
  if (!g) return qm_fail(QM_ERR_ARG, "qm_moe: null geometry");
  const int rc = qm_check_route("qm_moe", g->act_dtype, g->rows, g->hidden, g->experts, g->top_k, ldx);
  if (rc) return rc;
  if (g->inter <= 0 || g->inter % 32 || g->inter > (1 << 20))
    return qm_fail(QM_ERR_ARG, "qm_moe: inter must be a positive multiple of 32 (at most 2^20)");
  if (g->shared < 0 || g->shared > 32) return qm_fail(QM_ERR_ARG, "qm_moe: shared must be 0..32");
  if (g->weight_format != QM_W_ACT && g->weight_format != QM_W_MX4)
    return qm_fail(QM_ERR_DTYPE, "qm_moe: weight_format must be QM_W_ACT or QM_W_MX4");
  return QM_OK;
}

template <typename T>
int launch_combine(const MoeArgs<T>& A, hipStream_t stream) {
  const long n = (long)A.rows * (A.hidden / (16 / (int)sizeof(T)));
  hipLaunchKernelGGL(moe_combine_kernel<T>, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream, A);
  QM_CHECK_LAUNCH();
  return QM_OK;
}

template <typename WF, typename T, int TN, int TM, int WN, int WM, int S, bool STREAM = false>
int launch_gemms(const MoeArgs<T>& A, long max_tiles, hipStream_t stream) {
  using G = SpanGemm<WF, T, TN, TM, WN, WM, S, STREAM>;
  constexpr int NT = 64 * WN * WM;
  const int hn = TN / 2 * WN, dn = TN * WN;
  const long up = max_tiles * ((wt_row_tiles(A.inter) + hn - 1) / hn), down = max_tiles * ((wt_row_tiles(A.hidden) + dn - 1) / dn);
  if (up > 0x7fffffffL / NT || down > 0x7fffffffL / NT) return qm_fail(QM_ERR_UNSUPPORTED, "qm_moe: too many tiles for one launch");
  static std::atomic<uint64_t> up_ok{0}, down_ok{0};
  int rc = qm_allow_lds(reinterpret_cast<const void*>(moe_up_gemm_kernel<WF, T, TN, TM, WN, WM, S, STREAM>), G::LDS_BYTES, up_ok);
  if (!rc)
    rc = qm_allow_lds(reinterpret_cast<const void*>(moe_down_gemm_kernel<WF, T, TN, TM, WN, WM, S, STREAM>), G::LDS_BYTES, down_ok);
  if (rc) return rc;
  hipLaunchKernelGGL((moe_up_gemm_kernel<WF, T, TN, TM, WN, WM, S, STREAM>), dim3((unsigned)up), dim3(NT), G::LDS_BYTES, stream, A);
  QM_CHECK_LAUNCH();
  hipLaunchKernelGGL((moe_down_gemm_kernel<WF, T, TN, TM, WN, WM, S, STREAM>), dim3((unsigned)down), dim3(NT), G::LDS_BYTES, stream, A);
  QM_CHECK_LAUNCH();
  return launch_combine(A, stream);
}

template <typename WF, typename T>
int launch_ffn(const MoeArgs<T>& A, int bm, bool once, long max_tiles, hipStream_t stream) {
  if constexpr (sizeof(T) == 4) {
    if constexpr (Fmt<WF, T>::SCALED) return launch_gemms<WF, T, 4, 1, 2, 1, 2>(A, max_tiles, stream);
    else return launch_gemms<WF, T, 2, 2, 4, 1, 2>(A, max_tiles, stream);
  } else if constexpr (Fmt<WF, T>::SCALED) {
    if (bm == 64) return launch_gemms<WF, T, 4, 2, 4, 2, 2>(A, max_tiles, stream);
    return once ? launch_gemms<WF, T, 2, 2, 8, 1, 2, true>(A, max_tiles, stream)
                : launch_gemms<WF, T, 2, 2, 8, 1, 2>(A, max_tiles, stream);
  } else {
    if (bm == 128) return launch_gemms<WF, T, 2, 4, 4, 2, 2>(A, max_tiles, stream);
    if (bm == 64) return launch_gemms<WF, T, 2, 4, 4, 1, 3>(A, max_tiles, stream);
    return once ? launch_gemms<WF, T, 2, 2, 4, 1, 3, true>(A, max_tiles, stream)
                : launch_gemms<WF, T, 2, 2, 4, 1, 3>(A, max_tiles, stream);
  }
}

template <typename WF, typename T, int PER>
int launch_few_per(const FewArgs<T>& A, int max_slots, hipStream_t stream) {
  constexpr int TN = Fmt<WF, T>::SCALED ? 2 : 1;
  const int rt = wt_row_tiles(A.m.inter);
  if (A.m.rows == 1) {
    hipLaunchKernelGGL((moe_few_up_kernel<WF, T, PER, true, 1>), dim3(rt, max_slots), dim3(64 * FEW_UP_NW), 0, stream, A);
  } else {
    hipLaunchKernelGGL((moe_few_plan_kernel<T, PER>), dim3(1), dim3(64 * FEW), 0, stream, A);
    QM_CHECK_LAUNCH();
    hipLaunchKernelGGL((moe_few_up_kernel<WF, T, 1, false, TN>), dim3((rt + TN - 1) / TN, max_slots), dim3(64 * FEW_UP_NW), 0,
                       stream, A);
  }
  QM_CHECK_LAUNCH();
  hipLaunchKernelGGL((moe_few_down_kernel<WF, T>), dim3(wt_row_tiles(A.m.hidden), A.split), dim3(64 * FEW_DOWN_NW), 0, stream, A);
  QM_CHECK_LAUNCH();
  return QM_OK;
}

template <typename WF, typename T>
int launch_few(const FewArgs<T>& A, hipStream_t stream) {
  const int choices = A.m.rows * A.m.top_k, slots = A.m.shared + (choices < A.m.experts ? choices : A.m.experts);
  if (A.m.experts <= 64) return launch_few_per<WF, T, 1>(A, slots, stream);
  if (A.m.experts <= 128) return launch_few_per<WF, T, 2>(A, slots, stream);
  if (A.m.experts <= 256) return launch_few_per<WF, T, 4>(A, slots, stream);
  if (A.m.experts <= 512) return launch_few_per<WF, T, 8>(A, slots, stream);
  return launch_few_per<WF, T, 16>(A, slots, stream);
}

template <typename T, typename WPlain>
int run_moe(const qm_moe_geom& g, const qm_moe_weights& w, const void* x, long ldx, void* out, char* ws,
            hipStream_t stream) {
  const MoeLayout l = moe_layout(g);
  int* counts = reinterpret_cast<int*>(ws + l.counts);
  const QmLogits<T> L = {static_cast<const T*>(x), ldx, static_cast<const T*>(w.router),
                         static_cast<const T*>(w.shared_router), reinterpret_cast<double*>(ws + l.logits), g.rows, g.hidden,
                         g.experts, g.experts + (w.shared_router && g.shared ? 1 : 0), g.rows <= FEW ? nullptr : counts};
  const bool mx = g.weight_format == QM_W_MX4;
  auto mat = [mx](const void* d, const void* s) { return WMat{d, mx ? static_cast<const uint8_t*>(s) : nullptr}; };
  int* meta = reinterpret_cast<int*>(ws + l.meta);
  MoeArgs<T> A = {};
  A.x = L.x; A.ldx = ldx; A.rows = g.rows; A.hidden = g.hidden; A.inter = g.inter; A.experts = g.experts;
  A.shared = g.shared; A.top_k = g.top_k; A.ppt = g.top_k + g.shared;
  A.gate = mat(w.gate, w.gate_scales); A.up = mat(w.up, w.up_scales); A.down = mat(w.down, w.down_scales);
  A.s_gate = mat(w.shared_gate, w.shared_gate_scales); A.s_up = mat(w.shared_up, w.shared_up_scales);
  A.s_down = mat(w.shared_down, w.shared_down_scales);
  A.h = reinterpret_cast<T*>(ws + l.h);
  A.out = static_cast<T*>(out);
  if (g.rows <= FEW) {
    const FewArgs<T> P = {A, L.logits, L.cols, g.normalize, meta, counts,
                          reinterpret_cast<int*>(ws + l.lists), reinterpret_cast<float*>(ws + l.pair_w), down_split(g),
                          reinterpret_cast<float*>(ws + l.part), reinterpret_cast<unsigned*>(ws + l.done)};
    const int rc = qm_route_logits(L, stream);
    if (rc) return rc;
    return mx ? launch_few<WMx4, T>(P, stream) : launch_few<WPlain, T>(P, stream);
  }
  int* ids = reinterpret_cast<int*>(ws + l.ids);
  float* pair_w = reinterpret_cast<float*>(ws + l.pair_w);
  int* lists = reinterpret_cast<int*>(ws + l.lists);
  int2* tiles = reinterpret_cast<int2*>(ws + l.tiles);
  const QmRouteLists lists_out = {counts, lists, meta + 1, tiles, A.ppt, g.shared, l.bm};
  const int rc = qm_route(L, g.top_k, g.normalize, ids, pair_w, A.ppt, g.shared, &lists_out,
                          reinterpret_cast<float*>(ws + l.norms), stream);
  if (rc) return rc;
  A.counts = counts; A.lists = lists; A.pair_w = pair_w; A.n_tiles = meta + 1; A.tiles = tiles;
  A.part = reinterpret_cast<float*>(ws + l.part);
  // Up to 16 rows of an expert, on average, its weights are read about once and not
  // kept in the L2 (128 tokens over 128 experts: bf16 157 -> 147 us, 4-bit 53 -> 50;
  // 25 rows 60 -> 63, 62 rows 98 -> 106)
  const bool once = (double)g.rows * g.top_k <= 16.0 * g.experts;
  return mx ? launch_ffn<WMx4, T>(A, l.bm, once, l.max_tiles, stream)
            : launch_ffn<WPlain, T>(A, l.bm, once, l.max_tiles, stream);
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
      if (!scales[i] || reinterpret_cast<uintptr_t>(scales[i]) & 3)
        return qm_fail(QM_ERR_ARG, "qm_moe: scales are null or not 4-byte aligned");
  if (!aligned16(x) || !aligned16(out) || !aligned16(workspace) || (w->shared_router && !aligned16(w->shared_router)))
    return qm_fail(QM_ERR_ARG, "qm_moe: x, out, workspace and shared_router must be 16-byte aligned");
  const MoeLayout l = moe_layout(*g);
  if (workspace_bytes < l.bytes) return qm_fail(QM_ERR_WORKSPACE, "qm_moe: workspace too small (see qm_moe_workspace)");
  char* ws = static_cast<char*>(workspace);
  if (g->act_dtype == QM_ACT_BF16) return run_moe<bf16_t, WBf16>(*g, *w, x, ldx, out, ws, stream);
  return run_moe<float, WF32>(*g, *w, x, ldx, out, ws, stream);
}
