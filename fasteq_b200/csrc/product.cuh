// What the kernels of the dense layers with an epilogue share: activations, and the tiles of rows in the experts' order.
#pragma once
#include <cstdint>
#include <cuda_runtime.h>
#include "fasteq_b200.h"
#include "fasteq_device.cuh"

namespace fasteq {
namespace product {

enum Act : int { kIdentity = 0, kSilu = 1, kTanh = 2, kSigmoid = 3, kAbs = 4 };

// 2^t within two units of the last place (0 below 2^-126), and 1 / x within one (x from 1 to 2^126)
__device__ __forceinline__ float power_of_two(float t) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
  return e;
}
__device__ __forceinline__ float reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
constexpr float kLog2e = 1.44269502f;
// 1 / (1 + exp(-z)) and what it lacks to one, 1 / (1 + exp(z)), each with relative accuracy: exp(-z) = 2^t (1 + c), t = -z log2(e) rounded, c what that
// rounding lost and what log2(e) lost as a constant (1.93e-8).  Up to |z| = kNear, where nothing overflows or is flushed, two values side by side (644,552 rows of
// 64 to 64 channels with SiLU: 78.1 us, one by one 80.9 us; without c 72.4 us, and off by |z| half steps).
constexpr float kNear = 80.f;
__device__ __forceinline__ float2 sigmoid_near(float2 z, float2& rest) {
  const float2 t = vmul(z, make_float2(-kLog2e, -kLog2e)), lost = vfma(z, make_float2(kLog2e, kLog2e), t);
  const float2 c = vfma(lost, make_float2(-0.693147182f, -0.693147182f), vmul(z, make_float2(-1.334976e-8f, -1.334976e-8f)));
  const float2 first = make_float2(power_of_two(t.x), power_of_two(t.y)), e = vfma(first, c, first), d = vadd(e, make_float2(1.f, 1.f));
  const float2 s = make_float2(reciprocal(d.x), reciprocal(d.y));
  rest = vmul(e, s);
  return s;
}
// For any z: beyond kNear e = exp(-|z|) is below 2^-115 and the two are e and one, e down to the subnormal numbers (0 from 110 on, NaN of NaN).
__device__ __forceinline__ float sigmoid(float z, float& rest) {
  if (fabsf(z) <= kNear) {
    float2 r;
    const float2 s = sigmoid_near(make_float2(z, z), r);
    rest = r.x;
    return s.x;
  }
  float a, e;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(a) : "f"(fabsf(z)), "f"(110.f));
  const float t = a * -kLog2e;
  asm("ex2.approx.f32 %0, %1;" : "=f"(e) : "f"(t));
  e = fmaf(e, fmaf(fmaf(a, kLog2e, t), -0.693147182f, a * -1.334976e-8f), e);
  rest = z < 0.f ? 1.f : e;
  return z < 0.f ? e : 1.f + e;
}
// In FP64 exp(-a) = 2^n exp(r), -a = n ln 2 + r (ln 2 in two parts, the first of 33 bits, so that its product with n is exact), exp(r) by its Taylor polynomial
// of degree 13 (|r| <= 0.347: 4e-18 left out); no branch, so that a thread's values run side by side.  2^n in two factors, the second of which rounds into the
// subnormal numbers.  From a = 750 on it is 0.
__device__ __forceinline__ double exp_minus(double a) {
  const double t = a > 750.0 ? -750.0 : -a, n = rint(t * 0x1.71547652b82fep+0);
  const double r = fma(n, -0x1.473de6af278edp-34, fma(n, -0x1.62e42fef00000p-1, t));
  double p = 1.0 / 6227020800.0;
  p = fma(p, r, 1.0 / 479001600.0);
  p = fma(p, r, 1.0 / 39916800.0);
  p = fma(p, r, 1.0 / 3628800.0);
  p = fma(p, r, 1.0 / 362880.0);
  p = fma(p, r, 1.0 / 40320.0);
  p = fma(p, r, 1.0 / 5040.0);
  p = fma(p, r, 1.0 / 720.0);
  p = fma(p, r, 1.0 / 120.0);
  p = fma(p, r, 1.0 / 24.0);
  p = fma(p, r, 1.0 / 6.0);
  p = fma(p, r, 1.0 / 2.0);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  const int k = (int)n, most = max(k, -1000);
  return __hiloint2double(__double2hiint(p) + most * (1 << 20), __double2loint(p)) * __hiloint2double((1023 + k - most) << 20, 0);
}
// 1 / d in FP64, by Newton's iteration, each step squaring the error of the first 20 bits
__device__ __forceinline__ double reciprocal(double d) {
  double y;
  asm("rcp.approx.ftz.f64 %0, %1;" : "=d"(y) : "d"(d));
  y = fma(y, fma(-d, y, 1.0), y);
  return fma(y, fma(-d, y, 1.0), y);
}
// of both, the smaller is e / (1 + e), the larger 1 / (1 + e), e = exp(-|z|)
__device__ __forceinline__ double sigmoid(double z, double& rest) {
  const double e = exp_minus(fabs(z)), q = reciprocal(1.0 + e), small = e * q;
  rest = z < 0.0 ? q : small;
  return z < 0.0 ? small : q;
}

// tanh(z): up to |z| = 0.8 its Pade approximant of degrees 5 and 4 (8e-9 off at most), beyond 1 - 2 / (exp(2 |z|) + 1), which is nowhere above one (so that
// the slope is nowhere negative) and one itself from |z| = 10 on
__device__ __forceinline__ float hyperbolic_tangent(float z) {
  const float a = fabsf(z), e = power_of_two(a * (2.f * kLog2e)), q = z * z;
  const bool small = a <= 0.8f;
  const float r = reciprocal(small ? fmaf(q, fmaf(q, 15.f, 420.f), 945.f) : e + 1.f);
  return small ? z * fmaf(q, 105.f + q, 945.f) * r : copysignf(fmaf(-2.f, r, 1.f), z);
}
__device__ __forceinline__ double hyperbolic_tangent(double z) { return tanh(z); }

// act(z) and act'(z)
template <int ACT, typename T> __device__ __forceinline__ T activate(T z, T& slope) {
  if (ACT == kSilu) {
    T rest;
    const T s = sigmoid(z, rest);
    slope = s * (T(1) + z * rest);
    return z * s;
  }
  if (ACT == kTanh) {
    const T t = hyperbolic_tangent(z);
    slope = T(1) - t * t;
    return t;
  }
  if (ACT == kSigmoid) {
    T rest;
    const T s = sigmoid(z, rest);
    slope = s * rest;
    return s;
  }
  if (ACT == kAbs) {
    slope = T((z > T(0)) - (z < T(0)));
    return fabs(z);
  }
  slope = T(1);
  return z;
}
// of two values, |z| <= kNear
template <int ACT> __device__ __forceinline__ float2 activate_near(float2 z, float2& slope) {
  if (ACT == kSilu || ACT == kSigmoid) {
    float2 rest;
    const float2 s = sigmoid_near(z, rest);
    slope = vmul(s, ACT == kSilu ? vfma(z, rest, make_float2(1.f, 1.f)) : rest);
    return ACT == kSilu ? vmul(z, s) : s;
  }
  return make_float2(activate<ACT>(z.x, slope.x), activate<ACT>(z.y, slope.y));
}
template <typename T> __device__ __forceinline__ T activate(int act, T z, T& slope) {
  return act == kSilu ? activate<kSilu>(z, slope) : act == kTanh ? activate<kTanh>(z, slope) : act == kSigmoid ? activate<kSigmoid>(z, slope)
       : act == kAbs ? activate<kAbs>(z, slope) : activate<kIdentity>(z, slope);
}

// Rows of group e: [first(e), first(e + 1)); group `experts` holds those of no expert.  Offsets are the caller's memory: whatever they hold, the tiles and
// chunks made of them stay within the rows.
struct Groups {
  const int* offsets;                   // null: one group of all rows
  int experts, inner;
  long long rows;
  __device__ __forceinline__ long long first(int e) const {
    if (e > experts) return rows;
    if (!offsets) return e == 0 ? 0 : rows;
    const long long row = (long long)offsets[e] * inner;
    return row < 0 ? 0 : row > rows ? rows : row;
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
  *n_rows = left <= 0 || *m0 < begin ? 0 : left < SIZE ? (int)left : SIZE;
  return lo;
}

// The same with a size known at run time, found by a warp together (two loads a lane for up to 1024 groups): for the chunks of the weight gradient.
struct Chunk {
  int e, rows;                          // group, rows (0: an empty number)
  long long m0, begin, count;           // first row; the group's first row and number of chunks
};
__device__ __forceinline__ Chunk chunk_of(const Groups& g, int n_groups, int size, long long b) {
  const int lane = threadIdx.x & 31, step = (n_groups + 31) / 32;
  auto begins = [&](int e) { return e < n_groups && g.first(e) / size + e <= b; };
  int e = max(__popc(__ballot_sync(0xffffffffu, begins(lane * step))) - 1, 0) * step;
  if (step > 1) e += max(__popc(__ballot_sync(0xffffffffu, lane < step && begins(e + lane))) - 1, 0);
  Chunk c;
  c.e = e;
  c.begin = g.first(e);
  const long long end = g.first(e + 1), left = end - c.begin - (b - (c.begin / size + e)) * size;
  c.count = (end - c.begin + size - 1) / size;
  c.m0 = end - left;
  c.rows = left <= 0 || c.m0 < c.begin ? 0 : left < size ? (int)left : size;
  return c;
}
// Where a chunk's partial sums go, of chunks(rows, size): groups of several chunks have more than their share of 2 rows / size, so that
// counting those from 2 begin / size leaves each its own.  A group of one chunk needs none, its sums are the result.
__host__ __device__ inline long long partial_slots(long long rows, int size) { return 2 * rows / size + 1; }
__device__ __forceinline__ long long partial_slot(const Chunk& c, int size) { return 2 * c.begin / size + (c.m0 - c.begin) / size; }

}  // namespace product
}  // namespace fasteq
