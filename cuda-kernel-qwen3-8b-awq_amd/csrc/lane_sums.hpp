// Sums and maxima over the lanes of a wavefront without a trip through LDS: a shuffle between any two lanes takes that trip, about
// 50 cycles of latency each; exchanges within 16 lanes are operands of the addition itself (DPP), and gfx950 swaps rows of 16
// and of 32 lanes between two registers.
#pragma once
#include "common.hpp"

namespace lanes {

template <int CTRL>
__device__ __forceinline__ float from(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
struct Add {
  __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
};
struct Max {
  __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
};

// over groups of N lanes next to each other, in every lane: lane ^ 1, lane ^ 2, then the mirror images within 8 and 16 lanes (whose
// groups of 4 and 8 hold one value by then), then rows of 16 and 32
template <int N, typename F>
__device__ __forceinline__ float over(float v, F f) {
  static_assert(N >= 2 && N <= 64 && (N & (N - 1)) == 0, "a power of two");
  v = f(v, from<0xB1>(v));
  if constexpr (N >= 4) v = f(v, from<0x4E>(v));
  if constexpr (N >= 8) v = f(v, from<0x141>(v));
  if constexpr (N >= 16) v = f(v, from<0x140>(v));
  if constexpr (N >= 32) {  // (the waits are the data hazard slots the compiler would insert if it saw the instruction)
    float a = v, b = v;
    asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b));
    v = f(a, b);
  }
  if constexpr (N >= 64) {
    float a = v, b = v;
    asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b));
    v = f(a, b);
  }
  return v;
}
// over the lanes 16 apart, in every lane
template <typename F>
__device__ __forceinline__ float over_rows(float v, F f) {
  float a = v, b = v;
  asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b));
  a = b = f(a, b);
  asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b));
  return f(a, b);
}
template <int N = 64>
__device__ __forceinline__ float sum(float v) {
  return over<N>(v, Add());
}
template <int N = 64>
__device__ __forceinline__ float maximum(float v) {
  return over<N>(v, Max());
}

// n lanes next to each other (8, 16, 32 or 64, the same in the whole wavefront), in every lane
__device__ __forceinline__ float sum_of(float v, int n) {
  v = sum<8>(v);
  if (n > 8) v += from<0x140>(v);
  if (n > 16) {
    float a = v, b = v;
    asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b));
    v = a + b;
  }
  if (n > 32) {
    float a = v, b = v;
    asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b));
    v = a + b;
  }
  return v;
}
// the lanes n, 2 n, .. apart (n: 8, 16 or 32), in every lane
__device__ __forceinline__ float sum_apart(float v, int n) {
  if (n <= 8) v += from<0x128>(v);  // rotated by 8 within 16
  float a = v, b = v;
  if (n <= 16) {
    asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b));
    v = a + b;
    a = b = v;
  }
  asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b));
  return a + b;
}

// in every lane the sum over the lanes up to it, itself included (4 or 8 bytes): within rows of 16, then the rows ahead
template <int CTRL, int ROWS, typename T>
__device__ __forceinline__ T ahead(T v) {  // 0 where there is none
  static_assert(sizeof(T) == 4 || sizeof(T) == 8, "one or two registers");
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false));
  } else {
    const unsigned long long u = __builtin_bit_cast(unsigned long long, v);
    const unsigned int lo = (unsigned int)__builtin_amdgcn_update_dpp(0, (int)(unsigned int)u, CTRL, ROWS, 0xf, false);
    const unsigned int hi = (unsigned int)__builtin_amdgcn_update_dpp(0, (int)(unsigned int)(u >> 32), CTRL, ROWS, 0xf, false);
    return __builtin_bit_cast(T, (unsigned long long)hi << 32 | lo);
  }
}
template <typename T>
__device__ __forceinline__ T upto(T v) {
  v += ahead<0x111, 0xf>(v);
  v += ahead<0x112, 0xf>(v);
  v += ahead<0x114, 0xf>(v);
  v += ahead<0x118, 0xf>(v);
  v += ahead<0x142, 0xa>(v);  // lane 15 of the row ahead, for rows 1 and 3
  v += ahead<0x143, 0xc>(v);  // lane 31, for rows 2 and 3
  return v;
}

}  // namespace lanes
