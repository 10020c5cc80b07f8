// What the kernels of the dense layers with an epilogue share: activations, and the tiles of rows in the experts' order.
#pragma once
#include <cstdint>
#include <cuda_runtime.h>
#include "fasteq_b200.h"
#include "fasteq_device.cuh"

namespace fasteq {
namespace product {

enum Act : int { kIdentity = 0, kSilu = 1, kTanh = 2, kSigmoid = 3, kAbs = 4 };

// act(z) and act'(z)
template <typename T> __device__ __forceinline__ T activate(int act, T z, T& slope) {
  if (act == kSilu) {
    const T e = T(1) + exp(-z), s = T(1) / e;
    slope = s * (T(1) + z * (T(1) - s));
    return z / e;                       // z s rounds once more
  }
  if (act == kTanh) {
    const T t = tanh(z);
    slope = T(1) - t * t;
    return t;
  }
  if (act == kSigmoid) {
    const T s = T(1) / (T(1) + exp(-z));
    slope = s * (T(1) - s);
    return s;
  }
  if (act == kAbs) {
    slope = T((z > T(0)) - (z < T(0)));
    return fabs(z);
  }
  slope = T(1);
  return z;
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
