// All-reduces over aligned teams of L lanes of a wave (L a power of two up to 64) by lane-permute instructions: neighbours,
// pairs, the quads of a half row (mirror of 8), the halves of a row (mirror of 16), rows, halves of the wave.  Each step's two
// partners combine the same two values, so every lane of a team ends with the same bits.
#pragma once

#include "common.hpp"

namespace d2dmoe {

// The larger (smaller) of two numbers in one instruction: the middle one of them and an infinity, which the empty asm hides,
// since the compiler makes fmaxf of it otherwise, and of that up to three instructions (operands made quiet first).  A NaN loses
// in max1, as in fmaxf; min1 takes none.
__device__ __forceinline__ float max1(float a, float b) {
  float end = INFINITY;
  asm("" : "+s"(end));
  return __builtin_amdgcn_fmed3f(a, b, end);
}
__device__ __forceinline__ float min1(float a, float b) {
  float end = -INFINITY;
  asm("" : "+s"(end));
  return __builtin_amdgcn_fmed3f(a, b, end);
}

template <int CTRL>
__device__ inline uint32_t dpp(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true); }

template <int L, typename Op>
__device__ inline uint32_t team_reduce(uint32_t v, Op op) {
  if constexpr (L >= 2) v = op(v, dpp<0xB1>(v));
  if constexpr (L >= 4) v = op(v, dpp<0x4E>(v));
  if constexpr (L >= 8) v = op(v, dpp<0x141>(v));
  if constexpr (L >= 16) v = op(v, dpp<0x140>(v));
  if constexpr (L >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = op(r[0], r[1]);
  }
  if constexpr (L >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = op(r[0], r[1]);
  }
  return v;
}
template <int L>
__device__ inline uint32_t team_max_u(uint32_t v) { return team_reduce<L>(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; }); }
template <int L>
__device__ inline float team_max(float v) {
  return __uint_as_float(team_reduce<L>(__float_as_uint(v), [](uint32_t a, uint32_t b) { return __float_as_uint(max1(__uint_as_float(a), __uint_as_float(b))); }));
}
template <int L>
__device__ inline float team_sum(float v) {
  return __uint_as_float(team_reduce<L>(__float_as_uint(v), [](uint32_t a, uint32_t b) { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); }));
}
template <int L>
__device__ inline double team_sum(double v) {
#pragma unroll
  for (int off = 1; off < L; off <<= 1) v += __shfl_xor(v, off, kWave);
  return v;
}
template <int L>
__device__ inline bool team_any(bool v) {
  const int base = (threadIdx.x & 63) & ~(L - 1);
  const uint64_t mask = (L == 64) ? ~0ull : ((1ull << (L & 63)) - 1) << base;
  return (__ballot(v) & mask) != 0ull;
}

}  // namespace d2dmoe
