// The largest logits of a token, found by one wave. Shared by the routing kernels
// (route.hip) and the few-token layer (moe.hip), which ranks for itself.
#pragma once

#include "common.h"

constexpr int RT_MAX_EXPERTS = 1024;
constexpr int RT_MAX_TOPK = 32;
constexpr int RT_EXACT = 2;

// A logit as an integer of the same order: NaN above everything, +0 and -0 equal.
__device__ __forceinline__ long long logit_key(double v) {
  if (v != v) return 0x7fffffffffffffffLL;
  const long long b = __double_as_longlong(v + 0.0);
  return b < 0 ? b ^ 0x7fffffffffffffffLL : b;
}
constexpr long long KEY_GONE = (long long)0x8000000000000000ULL;   // below every logit's

// lane i's key, uniform
__device__ __forceinline__ long long lane_key(long long k, int i) {
  const unsigned lo = (unsigned)__builtin_amdgcn_readlane((int)k, i);
  return (long long)(((unsigned long long)(unsigned)__builtin_amdgcn_readlane((int)(k >> 32), i) << 32) | lo);
}

// max / min over the wave, uniform (DPP steps in a row of 16, then the rows)
template <int CTRL> __device__ __forceinline__ int dpp_i(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xF, 0xF, true);
}
__device__ __forceinline__ int wave_max_i32(int v) {
  v = max(v, dpp_i<0xB1>(v));
  v = max(v, dpp_i<0x4E>(v));
  v = max(v, dpp_i<0x141>(v));
  v = max(v, dpp_i<0x140>(v));
  return max(max(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)),
             max(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
}
__device__ __forceinline__ int wave_min_i32(int v) { return ~wave_max_i32(~v); }

// The logits of up to 64 PER experts: lane l holds experts l, l + 64, ..., as floats
// in an integer's order (NaN above everything), and the largest of its own. take()
// gives the largest of all that are left, the lowest index among equals, and
// removes it. Rounding to float may make two logits equal or order none wrongly:
// who needs the order of the doubles looks again where two come close.
__device__ __forceinline__ int float_key(float v) {
  if (v != v) return 0x7fffffff;
  const int b = __float_as_int(v + 0.f);
  return b < 0 ? b ^ 0x7fffffff : b;
}
__device__ __forceinline__ float key_float(int k) { return __int_as_float(k == 0x7fffffff ? 0x7fc00000 : k < 0 ? k ^ 0x7fffffff : k); }
constexpr int KEY32_GONE = (int)0x80000000;                  // below every logit's

template <int PER>
struct WaveTop {
  int key[PER];
  int best, best_i;
  __device__ __forceinline__ void pick() {
    best = key[0];
    best_i = 0;
#pragma unroll
    for (int i = 1; i < PER; ++i)
      if (key[i] > best) { best = key[i]; best_i = i; }
  }
  __device__ __forceinline__ void load(const double* l, int experts, int lane) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = lane + 64 * i;
      key[i] = e < experts ? float_key((float)l[e]) : KEY32_GONE;
    }
    pick();
  }
  __device__ __forceinline__ int take(int lane, int& k) {
    k = wave_max_i32(best);
    const bool mine = best == k;
    const unsigned long long m = __builtin_amdgcn_ballot_w64(mine);
    int at = best_i * 64 + lane;
    if (__popcll(m) == 1) at = __builtin_amdgcn_readlane(at, __ffsll(m) - 1);
    else at = wave_min_i32(mine ? at : 0x7fffffff);
#pragma unroll
    for (int i = 0; i < PER; ++i) key[i] = at == lane + 64 * i ? KEY32_GONE : key[i];
    pick();
    return at;
  }
};

// The top_k largest logits of a token in the doubles' order, one per lane (key, id
// of lane j < top_k), by one wave. The logits in l are off by up to `off` each (0:
// they are the doubles); exact(e[2]) gives the sums in double of two experts to
// lanes 0 and 1. False, with nothing chosen, when more of them come close than a
// wave holds.
template <int PER, typename Exact>
__device__ __forceinline__ bool wave_topk(const double* l, int experts, int top_k, double off, int lane, long long& key,
                                          int& id, Exact exact) {
  WaveTop<PER> top;
  top.load(l, experts, lane);
  id = 0x7fffffff;
  int mine = KEY32_GONE, n = 0;
  float bar = 0.f, largest = 0.f;
  // logits further apart than this are in the right order: both may be off, and
  // both were rounded to float (half a step, of the largest of them)
  float close = 0.f;
  for (; n < experts; ++n) {
    int k;
    const int at = top.take(lane, k);
    const float v = key_float(k);
    if (n == 0) {
      largest = fabsf(v);
      close = (float)(2.0 * off * (1.0 + 0x1p-20)) + largest * 0x1p-22f + 0x1p-120f;
    }
    if (n == top_k - 1) {
      // magnitudes below the top may be larger (negative logits)
      close = fmaxf(close, (float)(2.0 * off * (1.0 + 0x1p-20)) + fabsf(v) * 0x1p-22f + 0x1p-120f);
      bar = v - 2.f * close;
    }
    if (n >= top_k && v < bar) break;
    if (n == 64) return false;             // more candidates than lanes (or NaN among them)
    if (lane == n) { mine = k; id = at; }
  }
  const float v = key_float(mine), above = __shfl_up(v, 1, 64), below = __shfl_down(v, 1, 64);
  const bool again = lane < n && ((lane > 0 && !(above - v > close)) || (lane + 1 < n && !(v - below > close)));
  key = lane < n ? logit_key(l[id]) : KEY_GONE;
  unsigned long long m = __builtin_amdgcn_ballot_w64(again);
  if (m == 0ull) return true;
  while (off > 0.0 && m) {
    // the last of them again where there is no other
    int at[RT_EXACT], e[RT_EXACT];
#pragma unroll
    for (int c = 0; c < RT_EXACT; ++c) {
      at[c] = m ? __ffsll(m) - 1 : at[c - 1 < 0 ? 0 : c - 1];
      m &= m - 1;
      e[c] = __builtin_amdgcn_readlane(id, at[c]);
    }
    const long long k = logit_key(exact(e));
#pragma unroll
    for (int c = 0; c < RT_EXACT; ++c) {
      const long long kc = lane_key(k, c);
      if (lane == at[c]) key = kc;
    }
  }
  // their order again
  int rank = 0;
  for (int i = 0; i < n; ++i) {
    const long long ok = lane_key(key, i);
    const int oi = __builtin_amdgcn_readlane(id, i);
    rank += ok > key || (ok == key && oi < id);
  }
  if (lane >= n) rank = lane;              // a permutation of the lanes
  const int lo = __builtin_amdgcn_ds_permute(4 * rank, (int)key), hi = __builtin_amdgcn_ds_permute(4 * rank, (int)(key >> 32));
  key = (long long)(((unsigned long long)(unsigned)hi << 32) | (unsigned)lo);
  id = __builtin_amdgcn_ds_permute(4 * rank, id);
  return true;
}

// The same when every logit is in double already: a plain selection by rounds.
__device__ __forceinline__ void wave_topk_exact(const double* l, int experts, int top_k, int lane, long long& key, int& id) {
  unsigned gone = 0;                       // of the lane's experts
  key = KEY_GONE;
  id = 0x7fffffff;
  for (int j = 0; j < top_k; ++j) {
    long long best = KEY_GONE;
    int at = 0x7fffffff;
    for (int i = 0; lane + 64 * i < experts; ++i) {
      const long long k = gone >> i & 1u ? KEY_GONE : logit_key(l[lane + 64 * i]);
      if (k > best) { best = k; at = lane + 64 * i; }
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
      const long long ok = __shfl_xor(best, d, 64);
      const int oa = __shfl_xor(at, d, 64);
      if (ok > best || (ok == best && oa < at)) { best = ok; at = oa; }
    }
    if (lane == (at & 63)) gone |= 1u << (at >> 6);
    if (lane == j) { key = best; id = at; }
  }
}

// the logit a key stands for (NaN as some NaN)
__device__ __forceinline__ double key_logit(long long k) {
  if (k == 0x7fffffffffffffffLL) return __longlong_as_double(0x7ff8000000000000LL);
  return __longlong_as_double(k < 0 ? k ^ 0x7fffffffffffffffLL : k);
}
