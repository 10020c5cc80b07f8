// What the kernels of the dense layers with an epilogue share: activations, and the tiles of rows in the experts' order.
#pragma once
#include <cstdint>
#include <cuda_runtime.h>
#include "fasteq_b200.h"
#include "fasteq_device.cuh"

namespace fasteq {
namespace product {

enum Act : int { kIdentity = 0, kSilu = 1, kTanh = 2, kSigmoid = 3, kAbs = 4 };

// exp(x) within two units of the last place: 2^t for the rounded t = x log2(e), times 1 + what the rounding left of the exponent (a
// product in two parts, as in Cody and Waite's argument reduction).  A third of the instructions of expf.
__device__ __forceinline__ float exponential(float x) {
  constexpr float L = 1.44269502f, L_LOW = 1.92596303e-8f, LN2 = 0.693147181f;
  const float t = x * L, left = fmaf(x, L_LOW, fmaf(x, L, -t));
  float e;
  asm("ex2.approx.f32 %0, %1;" : "=f"(e) : "f"(t));
  return fabsf(t) < 200.f ? fmaf(e, left * LN2, e) : e;      // beyond: 0 or infinity, which `left` (infinite itself there, or not a number) must not touch
}
__device__ __forceinline__ double exponential(double x) { return exp(x); }
__device__ __forceinline__ float reciprocal(float x) {
  float r;
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ double reciprocal(double x) { return 1.0 / x; }

// act(z) and act'(z)
template <int ACT, typename T> __device__ __forceinline__ T activate(T z, T& slope) {
  if (ACT == kSilu) {
    const T s = reciprocal(T(1) + exponential(-z));
    slope = s * (T(1) + z * (T(1) - s));
    return z * s;
  }
  if (ACT == kTanh) {
    const T t = tanh(z);
    slope = T(1) - t * t;
    return t;
  }
  if (ACT == kSigmoid) {
    const T s = reciprocal(T(1) + exponential(-z));
    slope = s * (T(1) - s);
    return s;
  }
  if (ACT == kAbs) {
    slope = T((z > T(0)) - (z < T(0)));
    return fabs(z);
  }
  slope = T(1);
  return z;
}
template <typename T> __device__ __forceinline__ T activate(int act, T z, T& slope) {
  return act == kSilu ? activate<kSilu>(z, slope) : act == kTanh ? activate<kTanh>(z, slope) : act == kSigmoid ? activate<kSigmoid>(z, slope)
       : act == kAbs ? activate<kAbs>(z, slope) : activate<kIdentity>(z, slope);
}

// Rows of group e: [first(e), first(e + 1)); group `experts` holds those of no expert.
struct Groups {
  const int* offsets;                   // null: one group of all rows
  int experts, inner;
  long long rows;
  __device__ __forceinline__ long long first(int e) const {
    if (e > experts) return rows;
    if (!offsets) return e == 0 ? 0 : rows;
    return (long long)offsets[e] * inner;
  }
};

// Tiles of SIZE rows, numbered so that a tile's group follows from the offsets alone: group e begins at number first(e) / SIZE + e, which
// leaves it at least ceil(rows of e / SIZE) numbers (some stay empty: at most one per group).
template <int SIZE> __host__ __device__ inline long long tile_numbers(long long rows, int groups) { return rows / SIZE + groups; }
template <int SIZE> __device__ __forceinline__ long long first_number(const Groups& g, int e) { return g.first(e) / SIZE + e; }
// the group of tile number b, its first row and its rows (0: an empty number)
template <int SIZE> __device__ __forceinline__ int tile_of(const Groups& g, int n_groups, long long b, long long* m0, int* n_rows) {
  int lo = 0, hi = n_groups - 1;
  while (lo < hi) {                     // the last group that begins at or before b
    const int mid = (lo + hi + 1) >> 1;
    if (first_number<SIZE>(g, mid) <= b) lo = mid; else hi = mid - 1;
  }
  const long long begin = g.first(lo), end = g.first(lo + 1);
  *m0 = begin + (b - (begin / SIZE + lo)) * SIZE;
  const long long left = end - *m0;
  *n_rows = left <= 0 ? 0 : left < SIZE ? (int)left : SIZE;
  return lo;
}

}  // namespace product
}  // namespace fasteq
