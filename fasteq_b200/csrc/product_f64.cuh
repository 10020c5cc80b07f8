// FP64 products of the dense layers on the FP64 tensor cores (mma.sync.m8n8k4; tcgen05 has no FP64 kind): forward, grad_x and the weight gradient
// are one loop over tiles of TM x TN outputs with operands from shared memory, [outer][k] or [k][outer] as they lie in memory.
//   forward  x [rows, K]    W [N, K]       both [outer][k]
//   grad_x   g [rows, N]    W [N, K]       [outer][k], [k][outer]
//   grad_w   g [rows, N]    x [rows, K]    both [k][outer], k running over an expert's rows
// Four warps share a tile; 16-wide k-steps through three stages of cp.async (16 bytes where extents and addresses are even, else 8).  A fragment's
// lanes read 4 x 4 neighbours of 8 bytes in a half warp, so rows 4 or 12 (mod 16) values apart meet no bank twice: pitches of 20 and the extent plus 4.
// Bound: the FP64 pipe, 64 multiply-adds per clock and SM.  Few columns get narrow tiles, or that pipe and the activations' threads would work on columns that are not there:
// with 64 x 64 tiles alone 224,531 rows of 8 to 8 channels with tanh and all gradients took 202 us, 63 us with these
// (elementary operations 116 us); of 512 to 8 1,332 and 731 us (859 us).
#pragma once
#include <type_traits>
#include "product.cuh"

namespace fasteq {
namespace pf64 {

using product::Chunk;
using product::Groups;

constexpr int ROWS = 64, BK = 16, NT = 128, STAGES = 3, OUTER_PITCH = BK + 4;
// doubles of an operand's stage
template <bool OUTER> constexpr int operand_size(int tile) { return OUTER ? tile * OUTER_PITCH : BK * (tile + 4); }
template <int TM, int TN, bool A_OUTER, bool B_OUTER> struct Shape {
  static constexpr int WM = TM == 64 ? (TN == 64 ? 2 : 4) : (TN == 64 ? 1 : 2), WN = 4 / WM;      // warps
  static constexpr int I = TM / WM / 8, J = TN / WN / 8;                                          // a warp's blocks of 8 x 8
  static constexpr int B_AT = operand_size<A_OUTER>(TM), STAGE = B_AT + operand_size<B_OUTER>(TN);
  static constexpr int TURNED = ROWS * (TN + 2);                                                  // the forward's tile on its way out
  static constexpr int SMEM = 8 * (STAGES * STAGE > TURNED ? STAGES * STAGE : TURNED);
};
// columns of a tile for N of them
inline int tile_for(int N) { return N <= 8 ? 8 : N <= 16 ? 16 : N <= 32 ? 32 : 64; }

__device__ __forceinline__ void copy_async(double* dst, const double* src, bool pair, int there) {      // there: 0, 1 or 2 values
  if (pair) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(there * 8) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(there * 8) : "memory");
}
__device__ __forceinline__ void commit_async() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void wait_async() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Every thread's copies of a k-step: f(smem offset, outer, k).  OUTER: [outer][k] in memory.
template <bool OUTER, int TILE, typename F> __device__ __forceinline__ void each_copy(bool pair, F f) {
  auto each = [&](auto values) {
    constexpr int V = decltype(values)::value, COPIES = TILE * BK / V, ALONG = (OUTER ? BK : TILE) / V;
#pragma unroll
    for (int c = 0; c < (COPIES + NT - 1) / NT; ++c) {
      const int i = c * NT + (int)threadIdx.x, far = i / ALONG, near = i % ALONG * V;
      if (COPIES % NT && i >= COPIES) break;
      if (OUTER) f(far * OUTER_PITCH + near, far, near); else f(far * (TILE + 4) + near, near, far);
    }
  };
  if (pair) each(std::integral_constant<int, 2>{}); else each(std::integral_constant<int, 1>{});
}
// a k-step of an operand of `outer` x `depth` values from `src`, `ld` between its rows; zeros beyond
template <bool OUTER, int TILE> __device__ __forceinline__ void load_step(double* dst, const double* src, long long ld, int outer, int k0, int depth, bool pair) {
  each_copy<OUTER, TILE>(pair, [&](int at, int m, int k) {
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

// sum[i][j]: this warp's blocks; column: sums over k of operand A's outer index `threadIdx.x` (COLUMNS)
template <int TM, int TN, bool A_OUTER, bool B_OUTER, bool COLUMNS>
__device__ __forceinline__ void multiply(double* smem, const Operand& a, const Operand& b, int depth,
                                         double (&sum)[Shape<TM, TN, A_OUTER, B_OUTER>::I][Shape<TM, TN, A_OUTER, B_OUTER>::J][2], double& column) {
  using S = Shape<TM, TN, A_OUTER, B_OUTER>;
  constexpr int I = S::I, J = S::J, A_PITCH = A_OUTER ? OUTER_PITCH : TM + 4, B_PITCH = B_OUTER ? OUTER_PITCH : TN + 4;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, m0 = warp / S::WN * I * 8, n0 = warp % S::WN * J * 8, steps = (depth + BK - 1) / BK;
  auto load = [&](int step) {
    double* st = smem + step % STAGES * S::STAGE;
    if (step < steps) {
      load_step<A_OUTER, TM>(st, a.src, a.ld, a.outer, step * BK, depth, a.pair);
      load_step<B_OUTER, TN>(st + S::B_AT, b.src, b.ld, b.outer, step * BK, depth, b.pair);
    }
    commit_async();
  };
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) load(s);
  for (int step = 0; step < steps; ++step) {
    double* st = smem + step % STAGES * S::STAGE;
    wait_async<STAGES - 2>();
    __syncthreads();
    load(step + STAGES - 1);             // into the stage that the step before has read
#pragma unroll
    for (int k = 0; k < BK; k += 4) {
      double x[I], y[J];
      const int kk = k + (lane & 3), mm = m0 + (lane >> 2), nn = n0 + (lane >> 2);
#pragma unroll
      for (int i = 0; i < I; ++i) x[i] = st[A_OUTER ? (mm + 8 * i) * A_PITCH + kk : kk * A_PITCH + mm + 8 * i];
#pragma unroll
      for (int j = 0; j < J; ++j) y[j] = st[S::B_AT + (B_OUTER ? (nn + 8 * j) * B_PITCH + kk : kk * B_PITCH + nn + 8 * j)];
#pragma unroll
      for (int i = 0; i < I; ++i)
#pragma unroll
        for (int j = 0; j < J; ++j)
          asm volatile("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0, %1}, {%2}, {%3}, {%0, %1};"
                       : "+d"(sum[i][j][0]), "+d"(sum[i][j][1]) : "d"(x[i]), "d"(y[j]));
    }
    if (COLUMNS && threadIdx.x < TM) {
      double part = 0.0;                 // two levels: a long sum's error is its additions'
#pragma unroll
      for (int k = 0; k < BK; ++k) part += st[A_OUTER ? threadIdx.x * A_PITCH + k : k * A_PITCH + threadIdx.x];
      column += part;
    }
  }
  wait_async<0>();
}
// f(row, column, value) of this thread's outputs, column even: two neighbours
template <int WN, int I, int J, typename F> __device__ __forceinline__ void each_output(const double (&sum)[I][J][2], F f) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, m = warp / WN * I * 8 + (lane >> 2), n = warp % WN * J * 8 + (lane & 3) * 2;
#pragma unroll
  for (int i = 0; i < I; ++i)
#pragma unroll
    for (int j = 0; j < J; ++j) f(m + 8 * i, n + 8 * j, sum[i][j]);
}

// A thread's rows of a column of the turned tile, four at a time: their activations' chains and their residuals' loads run side by side (12,288 rows
// of 256 to 256 channels with SiLU, residual and slope: 111 us one by one with branches, 78 us).
template <int ACT, int TN> __device__ __forceinline__ void finish_rows(const double* z, double b, const double* more, double* to, double* kept, int rows, int N) {
  constexpr int STEP = NT / TN, PITCH = TN + 2;
#pragma unroll 1
  for (int r0 = threadIdx.x / TN; r0 < rows; r0 += 4 * STEP) {
    double y[4], d[4], m[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = more && r0 + i * STEP < rows ? more[(size_t)(r0 + i * STEP) * N] : 0.0;
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = product::activate<ACT>(z[min(r0 + i * STEP, ROWS - 1) * PITCH] + b, d[i]);
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
template <bool FORWARD, int TN>
__global__ void __launch_bounds__(NT, TN == 64 ? 3 : 5) product_f64_kernel(Groups groups, const double* A, const double* W, const double* bias, const double* residual, int K, int N, int act,
                                                            int tiles_n, bool pair_a, bool pair_w, double* C, double* slope_out) {
  extern __shared__ __align__(16) double smem_f64[];
  wait_for_previous_kernel();
  long long m0;
  int m_rows;
  using S = Shape<ROWS, TN, true, FORWARD>;
  constexpr int PITCH = TN + 2;
  const int e = product::tile_of<ROWS>(groups, groups.experts + 1, blockIdx.x / tiles_n, &m0, &m_rows), n0 = (int)(blockIdx.x % tiles_n) * TN;
  if (m_rows == 0) return;
  double sum[S::I][S::J][2] = {}, none = 0.0;
  const bool routed = e < groups.experts;
  if (routed) {
    const double* w = W + (size_t)e * N * K;
    const Operand a{A + m0 * K, K, m_rows, pair_a}, b{FORWARD ? w + (size_t)n0 * K : w + n0, FORWARD ? K : N, min(TN, N - n0), pair_w};
    multiply<ROWS, TN, true, FORWARD, false>(smem_f64, a, b, K, sum, none);
  }
  if (!FORWARD) {
    each_output<S::WN>(sum, [&](int r, int c, const double (&v)[2]) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (r < m_rows && n0 + c + h < N) C[(size_t)(m0 + r) * N + n0 + c + h] = v[h];
    });
    return;
  }
  __syncthreads();                       // the last step has been read
  each_output<S::WN>(sum, [&](int r, int c, const double (&v)[2]) { *reinterpret_cast<double2*>(smem_f64 + r * PITCH + c) = make_double2(v[0], v[1]); });
  __syncthreads();
  const int c = threadIdx.x % TN, n = n0 + c;
  if (n >= N) return;
  const double b = bias && routed ? bias[(size_t)e * N + n] : 0.0;
  const size_t from = (size_t)m0 * N + n;
  const double* more = residual ? residual + from : nullptr;
  double *to = C + from, *kept = slope_out ? slope_out + from : nullptr;
  if (!routed) {
    for (int r = threadIdx.x / TN; r < m_rows; r += NT / TN) {
      to[(size_t)r * N] = 0.0;
      if (kept) kept[(size_t)r * N] = 0.0;
    }
    return;
  }
  const double* z = smem_f64 + c;
  switch (act) {
    case product::kSilu: return finish_rows<product::kSilu, TN>(z, b, more, to, kept, m_rows, N);
    case product::kTanh: return finish_rows<product::kTanh, TN>(z, b, more, to, kept, m_rows, N);
    case product::kSigmoid: return finish_rows<product::kSigmoid, TN>(z, b, more, to, kept, m_rows, N);
    case product::kAbs: return finish_rows<product::kAbs, TN>(z, b, more, to, kept, m_rows, N);
    default: return finish_rows<product::kIdentity, TN>(z, b, more, to, kept, m_rows, N);
  }
}

// A chunk of an expert's rows and a tile of its matrix; see product_wgrad_kernel
template <int TM, int TN>
__global__ void __launch_bounds__(NT, TM * TN == 4096 ? 3 : 5) product_wgrad_f64_kernel(Groups groups, const double* X, const double* G, int K, int N, int size, int tiles_k, int tiles, bool pair_x,
                                                                  bool pair_g, double* gw, double* gb, double* partial) {
  extern __shared__ __align__(16) double smem_f64[];
  wait_for_previous_kernel();
  const Chunk c = product::chunk_of(groups, groups.experts, size, blockIdx.x / tiles);
  if (c.rows == 0) return;
  const int tile = (int)(blockIdx.x % tiles), n0 = tile / tiles_k * TM, k0 = tile % tiles_k * TN;
  using S = Shape<TM, TN, false, false>;
  double sum[S::I][S::J][2] = {}, column = 0.0;
  const Operand a{G + c.m0 * N + n0, N, min(TM, N - n0), pair_g}, b{X + c.m0 * K + k0, K, min(TN, K - k0), pair_x};
  if (k0 == 0) multiply<TM, TN, false, false, true>(smem_f64, a, b, c.rows, sum, column);
  else multiply<TM, TN, false, false, false>(smem_f64, a, b, c.rows, sum, column);
  const size_t nk = (size_t)N * K;
  const bool only = c.count == 1;
  double* dst = only ? gw + (size_t)c.e * nk : partial + (size_t)product::partial_slot(c, size) * (nk + N);
  each_output<S::WN>(sum, [&](int r, int col, const double (&v)[2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (n0 + r < N && k0 + col + h < K) dst[(size_t)(n0 + r) * K + k0 + col + h] = v[h];
  });
  if (k0 == 0 && threadIdx.x < TM && n0 + (int)threadIdx.x < N && (gb || !only)) (only ? gb + (size_t)c.e * N : dst + nk)[n0 + threadIdx.x] = column;
}

}  // namespace pf64
}  // namespace fasteq
