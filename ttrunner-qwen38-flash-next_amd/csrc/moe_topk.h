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

// the logit a key stands for (NaN as some NaN)
__device__ __forceinline__ double key_logit(long long k) {
  if (k == 0x7fffffffffffffffLL) return __longlong_as_double(0x7ff8000000000000LL);
  return __longlong_as_double(k < 0 ? k ^ 0x7fffffffffffffffLL : k);
}

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
// a float as an integer of the same order (NaN above everything)
__device__ __forceinline__ int float_key(float v) {
  if (v != v) return 0x7fffffff;
  const int b = __float_as_int(v + 0.f);
  return b < 0 ? b ^ 0x7fffffff : b;
}
__device__ __forceinline__ float key_float(int k) { return __int_as_float(k < 0 ? k ^ 0x7fffffff : k); }
constexpr int KEY32_GONE = (int)0x80000000;                  // below every logit's

// how many lanes below this one have their bit set
__device__ __forceinline__ int bits_below(unsigned long long m) {
  return __builtin_amdgcn_mbcnt_hi((unsigned)(m >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)m, 0u));
}
__device__ __forceinline__ long long push_key(int to, long long k) {
  const int lo = __builtin_amdgcn_ds_permute(4 * to, (int)k), hi = __builtin_amdgcn_ds_permute(4 * to, (int)(k >> 32));
  return (long long)(((unsigned long long)(unsigned)hi << 32) | (unsigned)lo);
}

// The top_k largest logits of a token in the doubles' order, one per lane (key, id
// of lane j < top_k), by one wave; of up to 64 PER experts lane l looks at l, l + 64,
// ... The logits in l are off by up to `off` each (0: they are the doubles);
// exact(e[2]) gives the sums in double of two experts to lanes 0 and 1. False, with
// nothing chosen, when a logit is NaN or more than 63 come close.
//
// A search over the upper halves of the logits as floats finds where the top_k-th
// lies, sixteen counts over the wave; who may be above it goes to a lane of its own
// (a dozen, mostly) and is ranked there. (Taking the largest top_k times over has three
// times the instructions: 17.5 us for 14.3, 4001 tokens over 256 experts.)
template <int PER, typename Exact>
__device__ __forceinline__ bool wave_topk(const double* l, int experts, int top_k, double off, int lane, long long& key,
                                          int& id, Exact exact) {
  int k32[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) k32[i] = lane + 64 * i < experts ? float_key((float)l[lane + 64 * i]) : KEY32_GONE;
  int best = k32[0];
#pragma unroll
  for (int i = 1; i < PER; ++i) best = max(best, k32[i]);
  best = wave_max_i32(best);
  if (best == 0x7fffffff) return false;
  int border = KEY32_GONE;                 // top_k keys at least are not below it
#pragma unroll
  for (int b = 31; b >= 16; --b) {
    const int up = (int)((unsigned)border + (1u << b));
    int count = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) count += __popcll(__builtin_amdgcn_ballot_w64(k32[i] >= up));
    if (count >= top_k) border = up;
  }
  // Logits further apart than this are in the right order: both may be off, and both
  // were rounded to float (half a step of the larger).
  const float first = key_float(best), low = key_float(border);
  const float close = (float)(2.0 * off * (1.0 + 0x1p-20)) + fmaxf(fabsf(first), fabsf(low)) * 0x1p-22f + 0x1p-120f;
  const float bar = low - 2.f * close;
  const int bar_key = bar == bar ? float_key(bar) : KEY32_GONE + 1;   // (infinite ones: all of them)
  int n = 0;
  id = 0x7fffffff;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const bool in = k32[i] >= bar_key;
    const unsigned long long m = __builtin_amdgcn_ballot_w64(in);
    const int more = __popcll(m), to = in ? n + bits_below(m) : 63;
    const int got = __builtin_amdgcn_ds_permute(4 * to, lane + 64 * i);
    if (lane >= n && lane < n + more) id = got;
    n += more;
  }
  if (n > 63) return false;                // (lane 63 is where the others went)
  key = lane < n ? logit_key(l[id]) : KEY_GONE;
  int rank = 0;                            // (the lanes are in the order of the ids)
  for (int i = 0; i < n; ++i) {
    const long long other = lane_key(key, i);
    rank += lane > i ? other >= key : other > key;
  }
  if (lane >= n) rank = lane;              // a permutation of the lanes
  key = push_key(rank, key);
  id = __builtin_amdgcn_ds_permute(4 * rank, id);
  if (!(off > 0.0)) return true;
  const double v = key_logit(key), above = __shfl_up(v, 1, 64), below = __shfl_down(v, 1, 64);
  const bool again = lane < n && ((lane > 0 && !(above - v > (double)close)) || (lane + 1 < n && !(v - below > (double)close)));
  unsigned long long m = __builtin_amdgcn_ballot_w64(again);
  if (m == 0ull) return true;
  while (m) {
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
  rank = 0;
  for (int i = 0; i < n; ++i) {
    const long long other = lane_key(key, i);
    const int oi = __builtin_amdgcn_readlane(id, i);
    rank += other > key || (other == key && oi < id);
  }
  if (lane >= n) rank = lane;
  key = push_key(rank, key);
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
