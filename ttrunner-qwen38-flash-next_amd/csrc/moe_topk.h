// The largest logits of a token, found by one wave. Shared by the routing kernels
// (route.hip) and the few-token layer (moe.hip), which ranks for itself.
#pragma once

#include "common.h"

constexpr int RT_MAX_EXPERTS = 1024;
constexpr int RT_MAX_TOPK = 32;

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
__device__ __forceinline__ unsigned wave_max_u32(unsigned v) { return (unsigned)wave_max_i32((int)(v ^ 0x80000000u)) ^ 0x80000000u; }

// The logits of up to 64 PER experts: lane l holds experts l, l + 64, ... and the
// largest of its own. take() gives the largest of all that are left, the lowest
// index among equals, and removes it.
template <int PER>
struct WaveTop {
  long long key[PER];
  int b_hi, b_i;
  unsigned b_lo;
  __device__ __forceinline__ void pick() {
    long long best = key[0];
    b_i = 0;
#pragma unroll
    for (int i = 1; i < PER; ++i)
      if (key[i] > best) { best = key[i]; b_i = i; }
    b_hi = (int)(best >> 32);
    b_lo = (unsigned)best;
  }
  __device__ __forceinline__ void load(const double* l, int experts, int lane) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = lane + 64 * i;
      key[i] = e < experts ? logit_key(l[e]) : KEY_GONE;
    }
    pick();
  }
  __device__ __forceinline__ int take(int lane, long long& best) {
    const int hi = wave_max_i32(b_hi);
    const unsigned lo = wave_max_u32(b_hi == hi ? b_lo : 0u);
    const bool mine = b_hi == hi && b_lo == lo;
    const unsigned long long m = __builtin_amdgcn_ballot_w64(mine);
    int at = b_i * 64 + lane;
    if (__popcll(m) == 1) at = __builtin_amdgcn_readlane(at, __ffsll(m) - 1);
    else at = wave_min_i32(mine ? at : 0x7fffffff);
    best = (long long)(((unsigned long long)(unsigned)hi << 32) | lo);
#pragma unroll
    for (int i = 0; i < PER; ++i) key[i] = at == lane + 64 * i ? KEY_GONE : key[i];
    pick();
    return at;
  }
};

// the logit a key stands for (NaN as some NaN)
__device__ __forceinline__ double key_logit(long long k) {
  if (k == 0x7fffffffffffffffLL) return __longlong_as_double(0x7ff8000000000000LL);
  return __longlong_as_double(k < 0 ? k ^ 0x7fffffffffffffffLL : k);
}
