// FP64 products of the dense layers on the FP64 tensor cores (mma.sync.m8n8k4; tcgen05 has no FP64 kind): forward, grad_x and the weight gradient
// are one loop over tiles of 64 x 64 outputs with operands from shared memory, [outer][k] or [k][outer] as they lie in memory.
//   forward  x [rows, K]    W [N, K]       both [outer][k]
//   grad_x   g [rows, N]    W [N, K]       [outer][k], [k][outer]
//   grad_w   g [rows, N]    x [rows, K]    both [k][outer], k running over an expert's rows
// Four warps of 32 x 32 outputs; 16-wide k-steps through three stages of cp.async (16 bytes where extents and addresses are even, else 8).  A fragment's
// lanes read 4 x 4 neighbours of 8 bytes in a half warp, so rows 4 (mod 16) values apart meet no bank twice: pitches of 20 and 68.
// Bound: the FP64 pipe, 64 multiply-adds per clock and SM.
#pragma once
#include "product.cuh"

namespace fasteq {
namespace pf64 {

using product::Chunk;
using product::Groups;

constexpr int TILE = 64, BK = 16, NT = 128, STAGES = 3, OUTER_PITCH = BK + 4, K_PITCH = TILE + 4;
constexpr int OPERAND = TILE * OUTER_PITCH;          // doubles of an operand's stage, either way round
constexpr int SMEM = STAGES * 2 * OPERAND * 8;
static_assert(SMEM >= TILE * (TILE + 2) * 8, "the turned tile of the forward");

__device__ __forceinline__ void copy_async(double* dst, const double* src, bool pair, int there) {      // there: 0, 1 or 2 values
  if (pair) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(there * 8) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(there * 8) : "memory");
}
__device__ __forceinline__ void commit_async() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void wait_async() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Every thread's copies of a k-step: f(smem offset, outer, k, values).  OUTER: [outer][k] in memory.
template <bool OUTER, typename F> __device__ __forceinline__ void each_copy(bool pair, F f) {
  const int t = threadIdx.x;
  if (OUTER) {
    if (pair) {
#pragma unroll
      for (int i = 0; i < 4; ++i) { const int m = t / 8 + 16 * i, k = t % 8 * 2; f(m * OUTER_PITCH + k, m, k); }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) { const int m = t / 16 + 8 * i, k = t % 16; f(m * OUTER_PITCH + k, m, k); }
    }
  } else if (pair) {
#pragma unroll
    for (int i = 0; i < 4; ++i) { const int k = t / 32 + 4 * i, m = t % 32 * 2; f(k * K_PITCH + m, m, k); }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) { const int k = t / 64 + 2 * i, m = t % 64; f(k * K_PITCH + m, m, k); }
  }
}
// a k-step of an operand of `outer` x `depth` values from `src`, `ld` between its rows; zeros beyond
template <bool OUTER> __device__ __forceinline__ void load_step(double* dst, const double* src, long long ld, int outer, int k0, int depth, bool pair) {
  each_copy<OUTER>(pair, [&](int at, int m, int k) {
    const int along = OUTER ? depth - k0 - k : outer - m;          // values left in the direction they lie in
    const bool other = OUTER ? m < outer : k0 + k < depth;
    const int there = other && along > 0 ? (pair && along > 1 ? 2 : 1) : 0;
    copy_async(dst + at, there ? src + (OUTER ? m * ld + k0 + k : (long long)(k0 + k) * ld + m) : src, pair, there);
  });
}

struct Operand {
  const double* src;
  long long ld;
  int outer;                           // values there are in the tile
  bool pair;
};

// sum[i][j]: the 8 x 8 blocks of this warp's 32 x 32 outputs; column: sums over k of operand A's outer index `threadIdx.x` (COLUMNS)
template <bool A_OUTER, bool B_OUTER, bool COLUMNS>
__device__ __forceinline__ void multiply(double* smem, const Operand& a, const Operand& b, int depth, double (&sum)[4][4][2], double& column) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, m0 = (warp >> 1) * 32, n0 = (warp & 1) * 32, steps = (depth + BK - 1) / BK;
  constexpr int STAGE = 2 * OPERAND;
  auto load = [&](int step) {
    double* st = smem + step % STAGES * STAGE;
    if (step < steps) {
      load_step<A_OUTER>(st, a.src, a.ld, a.outer, step * BK, depth, a.pair);
      load_step<B_OUTER>(st + OPERAND, b.src, b.ld, b.outer, step * BK, depth, b.pair);
    }
    commit_async();
  };
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) load(s);
  for (int step = 0; step < steps; ++step) {
    double* st = smem + step % STAGES * STAGE;
    wait_async<STAGES - 2>();
    __syncthreads();
    load(step + STAGES - 1);             // into the stage that the step before has read
#pragma unroll
    for (int k = 0; k < BK; k += 4) {
      double x[4], y[4];
      const int kk = k + (lane & 3), mm = m0 + (lane >> 2), nn = n0 + (lane >> 2);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = st[A_OUTER ? (mm + 8 * i) * OUTER_PITCH + kk : kk * K_PITCH + mm + 8 * i];
        y[i] = st[OPERAND + (B_OUTER ? (nn + 8 * i) * OUTER_PITCH + kk : kk * K_PITCH + nn + 8 * i)];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          asm volatile("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0, %1}, {%2}, {%3}, {%0, %1};"
                       : "+d"(sum[i][j][0]), "+d"(sum[i][j][1]) : "d"(x[i]), "d"(y[j]));
    }
    if (COLUMNS && threadIdx.x < TILE) {
      double part = 0.0;                 // two levels: a long sum's error is its additions'
#pragma unroll
      for (int k = 0; k < BK; ++k) part += st[A_OUTER ? threadIdx.x * OUTER_PITCH + k : k * K_PITCH + threadIdx.x];
      column += part;
    }
  }
  wait_async<0>();
}
// f(row, column, value) of this thread's outputs, column even: two neighbours
template <typename F> __device__ __forceinline__ void each_output(const double (&sum)[4][4][2], F f) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, m = (warp >> 1) * 32 + (lane >> 2), n = (warp & 1) * 32 + (lane & 3) * 2;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) f(m + 8 * i, n + 8 * j, sum[i][j]);
}

// Every second row of a column of the turned tile, four at a time: their activations' chains and their residuals' loads run side by side (12,288 rows
// of 256 to 256 channels with SiLU, residual and slope: 111 us one by one with branches, 80 us).
constexpr int PITCH = TILE + 2;
template <int ACT> __device__ __forceinline__ void finish_rows(const double* z, double b, const double* more, double* to, double* kept, int rows, int N) {
  constexpr int STEP = NT / TILE;
#pragma unroll 1
  for (int r0 = threadIdx.x / TILE; r0 < rows; r0 += 4 * STEP) {
    double y[4], d[4], m[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = more && r0 + i * STEP < rows ? more[(size_t)(r0 + i * STEP) * N] : 0.0;
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = product::activate<ACT>(z[min(r0 + i * STEP, TILE - 1) * PITCH] + b, d[i]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (r0 + i * STEP >= rows) break;
      to[(size_t)(r0 + i * STEP) * N] = y[i] + m[i];
      if (kept) kept[(size_t)(r0 + i * STEP) * N] = d[i];
    }
  }
}

// One tile of C = epilogue(A op(W)); see product_kernel.  The forward turns its tile in shared memory and walks it in a loop: one copy of the
// activations' code, whole lines stored.
template <bool FORWARD>
__global__ void __launch_bounds__(NT, 3) product_f64_kernel(Groups groups, const double* A, const double* W, const double* bias, const double* residual, int K, int N, int act,
                                                            int tiles_n, bool pair_a, bool pair_w, double* C, double* slope_out) {
  extern __shared__ __align__(16) double smem_f64[];
  wait_for_previous_kernel();
  long long m0;
  int m_rows;
  const int e = product::tile_of<TILE>(groups, groups.experts + 1, blockIdx.x / tiles_n, &m0, &m_rows), n0 = (int)(blockIdx.x % tiles_n) * TILE;
  if (m_rows == 0) return;
  double sum[4][4][2] = {}, none = 0.0;
  const bool routed = e < groups.experts;
  if (routed) {
    const double* w = W + (size_t)e * N * K;
    const Operand a{A + m0 * K, K, m_rows, pair_a}, b{FORWARD ? w + (size_t)n0 * K : w + n0, FORWARD ? K : N, min(TILE, N - n0), pair_w};
    multiply<true, FORWARD, false>(smem_f64, a, b, K, sum, none);
  }
  if (!FORWARD) {
    each_output(sum, [&](int r, int c, const double (&v)[2]) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (r < m_rows && n0 + c + h < N) C[(size_t)(m0 + r) * N + n0 + c + h] = v[h];
    });
    return;
  }
  __syncthreads();                       // the last step has been read
  each_output(sum, [&](int r, int c, const double (&v)[2]) { *reinterpret_cast<double2*>(smem_f64 + r * PITCH + c) = make_double2(v[0], v[1]); });
  __syncthreads();
  const int c = threadIdx.x % TILE, n = n0 + c;
  if (n >= N) return;
  const double b = bias && routed ? bias[(size_t)e * N + n] : 0.0;
  const size_t from = (size_t)m0 * N + n;
  const double* more = residual ? residual + from : nullptr;
  double *to = C + from, *kept = slope_out ? slope_out + from : nullptr;
  if (!routed) {
    for (int r = threadIdx.x / TILE; r < m_rows; r += NT / TILE) {
      to[(size_t)r * N] = 0.0;
      if (kept) kept[(size_t)r * N] = 0.0;
    }
    return;
  }
  const double* z = smem_f64 + c;
  switch (act) {
    case product::kSilu: return finish_rows<product::kSilu>(z, b, more, to, kept, m_rows, N);
    case product::kTanh: return finish_rows<product::kTanh>(z, b, more, to, kept, m_rows, N);
    case product::kSigmoid: return finish_rows<product::kSigmoid>(z, b, more, to, kept, m_rows, N);
    case product::kAbs: return finish_rows<product::kAbs>(z, b, more, to, kept, m_rows, N);
    default: return finish_rows<product::kIdentity>(z, b, more, to, kept, m_rows, N);
  }
}

// A chunk of an expert's rows and a tile of its matrix; see product_wgrad_kernel
__global__ void __launch_bounds__(NT, 3) product_wgrad_f64_kernel(Groups groups, const double* X, const double* G, int K, int N, int size, int tiles_k, int tiles, bool pair_x,
                                                                  bool pair_g, double* gw, double* gb, double* partial) {
  extern __shared__ __align__(16) double smem_f64[];
  wait_for_previous_kernel();
  const Chunk c = product::chunk_of(groups, groups.experts, size, blockIdx.x / tiles);
  if (c.rows == 0) return;
  const int tile = (int)(blockIdx.x % tiles), n0 = tile / tiles_k * TILE, k0 = tile % tiles_k * TILE;
  double sum[4][4][2] = {}, column = 0.0;
  const Operand a{G + c.m0 * N + n0, N, min(TILE, N - n0), pair_g}, b{X + c.m0 * K + k0, K, min(TILE, K - k0), pair_x};
  if (k0 == 0) multiply<false, false, true>(smem_f64, a, b, c.rows, sum, column);
  else multiply<false, false, false>(smem_f64, a, b, c.rows, sum, column);
  const size_t nk = (size_t)N * K;
  const bool only = c.count == 1;
  double* dst = only ? gw + (size_t)c.e * nk : partial + (size_t)product::partial_slot(c, size) * (nk + N);
  each_output(sum, [&](int r, int col, const double (&v)[2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (n0 + r < N && k0 + col + h < K) dst[(size_t)(n0 + r) * K + k0 + col + h] = v[h];
  });
  if (k0 == 0 && threadIdx.x < TILE && n0 + (int)threadIdx.x < N && (gb || !only)) (only ? gb + (size_t)c.e * N : dst + nk)[n0 + threadIdx.x] = column;
}

}  // namespace pf64
}  // namespace fasteq
