// Dense layers with an epilogue, one matrix for all rows or one per expert (rows in the experts' order):
//   z = x W[e]^T + bias[e],  y = act(z) + residual;   gz = grad_y act'(z):  grad_x = gz W[e],  grad_w[e] = gz^T x,  grad_bias[e] = sum gz
// FP32 goes to the tensor cores (product_tc.cuh, product_wgrad_tc.cuh), FP64 to the FP64 ones (product_f64.cuh).  Here are the entries, and FMA kernels for what
// those do not take (addresses that are not 16-byte aligned, no channels to sum over, extents beyond their 32-bit counts): 64 x 64 tiles of 4 x 4 sums a
// thread, bound by shared-memory reads.  12,288 rows of 128 to 256 channels, forward / grad_x / weights: 43 / 55 / 60 us, on the tensor
// cores 16 / 16 / 18 us.
#include <algorithm>
#include <atomic>
#include <mutex>
#include <cstdint>
#include <cuda_runtime.h>
#include "fasteq_b200.h"
#include "core_common.h"
#include "fasteq_device.cuh"
#include "launch.cuh"
#include "product.cuh"
#include "product_tc.cuh"
#include "product_wgrad_tc.cuh"
#include "product_f64.cuh"
#include "gemm_tf32x3.h"

using namespace fasteq;
using namespace fasteq::product;

namespace {

constexpr int TILE = 64, BK = 16, PITCH = TILE + 4, THREADS = 256;
static_assert(FASTEQ_MAX_CHANNELS == TILE * 65535, "tiles of columns in a grid's second extent");

// One tile of C = epilogue(A op(W)).  A [rows, K], times `slope` where it is given.  FORWARD: W [N, K], bias, act and residual;
// else W [K, N] (grad_x: K the layer's outputs, N its inputs).
template <typename T, bool FORWARD>
__global__ void __launch_bounds__(THREADS) product_kernel(Groups groups, const T* A, const T* slope, const T* W, const T* bias, const T* residual,
                                                          int K, int N, int ldd, int act, T* C, T* slope_out) {
  __shared__ __align__(16) T sa[BK][PITCH], sw[BK][PITCH];
  wait_for_previous_kernel();
  long long m0;
  int m_rows;
  const int e = tile_of<TILE>(groups, groups.experts + 1, blockIdx.x, &m0, &m_rows);
  if (m_rows == 0) return;
  const int n0 = blockIdx.y * TILE, t = threadIdx.x, tm = (t / 16) * 4, tn = (t % 16) * 4;
  T sum[4][4] = {};
  if (e < groups.experts) {
    const T* w = W + (size_t)e * N * K;
    for (int k0 = 0; k0 < K; k0 += BK) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = t % 16, m = t / 16 + 16 * i;
        const long long at = (m0 + m) * K + k0 + k;
        T v = T(0);
        if (m < m_rows && k0 + k < K) v = slope ? A[at] * slope[(m0 + m) * ldd + k0 + k] : A[at];
        sa[k][m] = v;
        if (FORWARD) {
          sw[k][m] = n0 + m < N && k0 + k < K ? w[(size_t)(n0 + m) * K + k0 + k] : T(0);
        } else {
          const int n = t % 64, kk = t / 64 + 4 * i;
          sw[kk][n] = n0 + n < N && k0 + kk < K ? w[(size_t)(k0 + kk) * N + n0 + n] : T(0);
        }
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < BK; ++k) {
        T a[4], b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) { a[i] = sa[k][tm + i]; b[i] = sw[k][tn + i]; }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) sum[i][j] = vfma(a[i], b[j], sum[i][j]);
      }
      __syncthreads();
    }
  }
  for (int i = 0; i < 4; ++i) {
    if (tm + i >= m_rows) break;
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + tn + j;
      if (n >= N) break;
      const size_t at = (size_t)(m0 + tm + i) * N + n;
      T v = sum[i][j], d = T(1);
      if (FORWARD && e < groups.experts) {
        if (bias) v += bias[(size_t)e * N + n];
        v = activate(act, v, d);
        if (residual) v += residual[at];
      } else if (FORWARD) {
        d = T(0);
      }
      C[at] = v;
      if (FORWARD && slope_out) slope_out[(size_t)(m0 + tm + i) * ldd + n] = d;
    }
  }
}

// ------------------------------------------------------------------------------------------------ weight gradient
// A chunk of `size` of an expert's rows and a tile of its matrix per CTA.  An expert of one chunk has its sums then; the partial sums [slot][N * K | N]
// of the others a second kernel adds in order.
template <typename T>
__global__ void __launch_bounds__(THREADS) product_wgrad_kernel(Groups groups, const T* X, const T* G, const T* slope, int K, int N, int ldd, int size, T* gw,
                                                                T* gb, T* partial) {
  __shared__ __align__(16) T sg[BK][PITCH], sx[BK][PITCH];
  wait_for_previous_kernel();
  const Chunk c = chunk_of(groups, groups.experts, size, blockIdx.x);
  if (c.rows == 0) return;
  const int tiles_k = max(1, (K + TILE - 1) / TILE), n0 = ((int)blockIdx.y / tiles_k) * TILE, k0 = ((int)blockIdx.y % tiles_k) * TILE;
  const int t = threadIdx.x, tn = (t / 16) * 4, tk = (t % 16) * 4;
  T sum[4][4] = {}, column = T(0);
  for (int r0 = 0; r0 < c.rows; r0 += BK) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int col = t % 64, r = t / 64 + 4 * i;
      const bool there = r0 + r < c.rows;
      const long long row = c.m0 + r0 + r;
      T g = T(0);
      if (there && n0 + col < N) {
        const long long at = row * N + n0 + col;
        g = slope ? G[at] * slope[row * ldd + n0 + col] : G[at];
      }
      sg[r][col] = g;
      sx[r][col] = there && k0 + col < K ? X[row * K + k0 + col] : T(0);
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < BK; ++r) {
      T a[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) { a[i] = sg[r][tn + i]; b[i] = sx[r][tk + i]; }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[i][j] = vfma(a[i], b[j], sum[i][j]);
      if (k0 == 0 && t < TILE) column += sg[r][t];
    }
    __syncthreads();
  }
  const size_t nk = (size_t)N * K;
  const bool only = c.count == 1;
  T* dst = only ? gw + (size_t)c.e * nk : partial + (size_t)partial_slot(c, size) * (nk + N);
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j)
      if (n0 + tn + i < N && k0 + tk + j < K) dst[(size_t)(n0 + tn + i) * K + k0 + tk + j] = sum[i][j];
  if (k0 == 0 && t < TILE && n0 + t < N && (gb || !only)) (only ? gb + (size_t)c.e * N : dst + nk)[n0 + t] = column;
}

// Experts of no or of several chunks: 32 packs of V values at a time to a CTA, eight threads to each, which take every eighth chunk and are added in
// order.
template <typename T, int V> __global__ void __launch_bounds__(256) product_reduce_kernel(Groups groups, const T* partial, int K, int N, int size, T* gw, T* gb) {
  struct alignas(sizeof(T) * V) Pack { T v[V]; };
  __shared__ Pack part[8][32];
  wait_for_previous_kernel();
  const int e = blockIdx.y;
  const size_t nk = (size_t)N * K, all = nk + N;
  const long long begin = groups.first(e), n = (groups.first(e + 1) - begin + size - 1) / size;
  if (n == 1) return;
  const T* from = partial + (size_t)(2 * begin / size) * all;
  for (size_t i0 = (size_t)blockIdx.x * 32 * V; i0 < all; i0 += (size_t)gridDim.x * 32 * V) {
    const size_t i = i0 + threadIdx.x * V;
    Pack s{};
    if (i < all) {
#pragma unroll 4
      for (long long c = threadIdx.y; c < n; c += 8) {
        const Pack v = *reinterpret_cast<const Pack*>(from + (size_t)c * all + i);
#pragma unroll
        for (int k = 0; k < V; ++k) s.v[k] += v.v[k];
      }
    }
    part[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y == 0 && i < all) {
#pragma unroll
      for (int j = 1; j < 8; ++j)
#pragma unroll
        for (int k = 0; k < V; ++k) s.v[k] += part[j][threadIdx.x].v[k];
      if (i < nk) *reinterpret_cast<Pack*>(gw + (size_t)e * nk + i) = s;
      else if (gb) *reinterpret_cast<Pack*>(gb + (size_t)e * N + (i - nk)) = s;
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------------ entries
int check(const fasteq_product_problem* p, const int32_t* offsets) {
  if (!p || (p->dtype != FASTEQ_F32 && p->dtype != FASTEQ_F64) || p->k < 0 || p->n < 0 || p->rows < 0 || p->experts < 1 || p->inner < 1 ||
      p->act < 0 || p->act > 4 || (!offsets && p->experts != 1))
    return FASTEQ_INVALID;
  if (p->experts > FASTEQ_MAX_EXPERTS || p->rows / p->inner > 0x7fff0000LL || p->rows / TILE > 0x7fff0000LL || p->n > FASTEQ_MAX_CHANNELS || p->k > FASTEQ_MAX_CHANNELS)
    return FASTEQ_UNSUPPORTED;
  return FASTEQ_OK;
}
Groups groups_of(const fasteq_product_problem* p, const int32_t* offsets) { return Groups{offsets, p->experts, p->inner, (long long)p->rows}; }

// columns between the rows of what the forward leaves for the gradients (TMA wants multiples of 16 bytes)
int slope_pitch(const fasteq_product_problem* p) { return p->dtype == FASTEQ_F32 ? (p->n + 3) & ~3 : p->n; }

template <typename T>
int forward(const fasteq_product_problem* p, const void* x, const void* w, const void* bias, const void* residual, const int32_t* offsets, void* y,
            void* slope, cudaStream_t s) {
  const dim3 grid((unsigned)tile_numbers<TILE>(p->rows, p->experts + 1), (unsigned)((p->n + TILE - 1) / TILE));
  const cudaError_t e = launch_dependent(product_kernel<T, true>, grid, THREADS, 0, s, groups_of(p, offsets), (const T*)x, (const T*)nullptr, (const T*)w,
                                         (const T*)bias, (const T*)residual, p->k, p->n, slope_pitch(p), p->act, (T*)y, (T*)slope);
  return e == cudaSuccess ? FASTEQ_OK : cuda_fail(e);
}
template <typename T>
int dgrad(const fasteq_product_problem* p, const void* g, const void* slope, const void* w, const int32_t* offsets, void* gx, cudaStream_t s) {
  const dim3 grid((unsigned)tile_numbers<TILE>(p->rows, p->experts + 1), (unsigned)((p->k + TILE - 1) / TILE));
  const cudaError_t e = launch_dependent(product_kernel<T, false>, grid, THREADS, 0, s, groups_of(p, offsets), (const T*)g, (const T*)slope, (const T*)w,
                                         (const T*)nullptr, (const T*)nullptr, p->n, p->k, slope_pitch(p), 0, (T*)gx, (T*)nullptr);
  return e == cudaSuccess ? FASTEQ_OK : cuda_fail(e);
}
// What a launch needs to know of the current device, asked once: a microsecond or two a call otherwise.
struct Device {
  std::atomic<bool> known{false};
  int sms = 0;
  int* status = nullptr;                  // the tensor-core kernels' status word
};
constexpr int MAX_DEVICES = 64;
cudaError_t current_device(int* index, Device** device) {
  static Device devices[MAX_DEVICES];
  cudaError_t e = cudaGetDevice(index);
  if (e != cudaSuccess) return e;
  if (*index >= MAX_DEVICES) return cudaErrorInvalidDevice;
  Device& d = devices[*index];
  if (!d.known.load(std::memory_order_acquire)) {
    int sms = 0;
    int* status = nullptr;
    e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, *index);
    if (e == cudaSuccess) e = tc::status_word(&status);
    if (e != cudaSuccess) return e;
    static std::mutex lock;
    std::lock_guard<std::mutex> g(lock);
    if (!d.known.load(std::memory_order_relaxed)) {      // the first thread writes; others may be reading already
      d.sms = sms;
      d.status = status;
      d.known.store(true, std::memory_order_release);
    }
  }
  *device = &d;
  return cudaSuccess;
}
// lets a kernel have all of an SM's shared memory on a device, once
template <auto KERNEL> cudaError_t allow_shared_memory(int device) {
  static std::atomic<uint64_t> done{0};
  if (done.load(std::memory_order_relaxed) >> device & 1) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
  if (e == cudaSuccess) done.fetch_or(uint64_t(1) << device, std::memory_order_relaxed);
  return e;
}

// CTAs of a launch over tiles of rows and columns
bool in_32_bits(const fasteq_product_problem* p, int tile) {
  const long long tiles_k = (p->k + tile - 1) / tile, tiles_n = (p->n + tile - 1) / tile, rows = p->rows / tile + p->experts + 1;
  return rows * std::max(tiles_k, tiles_n) <= 0x7fffffffLL && tiles_k * tiles_n <= 0x7fffffffLL && tiles_k * tiles_n * (p->rows / 64 + p->experts) <= 0x7fffffffLL;
}
bool even(int extent, std::initializer_list<const void*> pointers) {
  uintptr_t all = 0;
  for (const void* q : pointers) all |= reinterpret_cast<uintptr_t>(q);
  return extent % 2 == 0 && (all & 15u) == 0;
}
template <bool FORWARD, int TN>
int launch_f64(const fasteq_product_problem* p, const void* A, const void* w, const void* bias, const void* residual, const int32_t* offsets, void* C, void* slope_out,
               cudaStream_t s) {
  const int K = FORWARD ? p->k : p->n, N = FORWARD ? p->n : p->k, tiles_n = (N + TN - 1) / TN;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = allow_shared_memory<pf64::product_f64_kernel<FORWARD, TN>>(dev);
  if (e == cudaSuccess)
    e = launch_dependent(pf64::product_f64_kernel<FORWARD, TN>, (unsigned)(tile_numbers<pf64::ROWS>(p->rows, p->experts + 1) * tiles_n), pf64::NT,
                         pf64::Shape<pf64::ROWS, TN, true, FORWARD>::SMEM, s, groups_of(p, offsets), (const double*)A, (const double*)w, (const double*)bias,
                         (const double*)residual, K, N, p->act, tiles_n, even(K, {A}), even(p->k, {w}), (double*)C, (double*)slope_out);
  return e == cudaSuccess ? FASTEQ_OK : cuda_fail(e);
}
template <bool FORWARD>
int product_f64(const fasteq_product_problem* p, const void* A, const void* w, const void* bias, const void* residual, const int32_t* offsets, void* C, void* slope_out,
                cudaStream_t s) {
  switch (pf64::tile_for(FORWARD ? p->n : p->k)) {
    case 8: return launch_f64<FORWARD, 8>(p, A, w, bias, residual, offsets, C, slope_out, s);
    case 16: return launch_f64<FORWARD, 16>(p, A, w, bias, residual, offsets, C, slope_out, s);
    case 32: return launch_f64<FORWARD, 32>(p, A, w, bias, residual, offsets, C, slope_out, s);
    default: return launch_f64<FORWARD, 64>(p, A, w, bias, residual, offsets, C, slope_out, s);
  }
}

// Rows of a chunk: as many as give every SM `per_sm` tiles of rows x matrix, in one wave (24,576 rows of 128 x 256 in FP32: 148 CTAs 18.4 us, 196 CTAs
// 28.4, 100 CTAs 23.8).  Every expert may add a chunk to those; many experts take half of the places at most.  At least 64 rows (1,000 rows of 128 x 256 with
// the sums' way out: FP32 16.1 us, 18.4 with 256 rows at least; FP64 31.7 and 39.8).  Experts of 256 rows or fewer on average stay whole, and need no
// partial sums (ten experts of 100 rows, 128 x 256, FP64: 27.5 us, 42.1 in pieces of 64; of 400 rows 68.9 and 50.4).
int chunk_rows(const fasteq_product_problem* p, int tile_n, int tile_k, int per_sm) {
  const long long tiles = (long long)((p->n + tile_n - 1) / tile_n) * std::max(1, (p->k + tile_k - 1) / tile_k), places = std::max<long long>(1, 148 * per_sm / tiles);
  const long long chunks = std::max<long long>(std::max<long long>(places - (p->experts > 1 ? p->experts : 0), places / 2), 1);
  const long long rows = ((p->rows + chunks - 1) / chunks + 31) / 32 * 32;
  const long long least = p->experts > 1 && p->rows <= 256LL * p->experts ? 256 : 64;
  return (int)std::min<long long>(1 << 24, std::max<long long>(least, rows));
}
int chunk_rows(const fasteq_product_problem* p, bool tensor_cores) { return tensor_cores ? chunk_rows(p, pwg::TM, pwg::TN, 1) : chunk_rows(p, TILE, TILE, 3); }

template <typename T> int reduce(const fasteq_product_problem* p, const Groups& groups, int size, void* gw, void* gb, void* scratch, cudaStream_t s) {
  if (p->experts == 1 && p->rows <= size && !groups.offsets) return FASTEQ_OK;
  constexpr int V = 16 / sizeof(T);
  const uintptr_t all = reinterpret_cast<uintptr_t>(gw) | reinterpret_cast<uintptr_t>(gb) | reinterpret_cast<uintptr_t>(scratch);
  const bool wide = p->n % V == 0 && all % 16 == 0;
  const size_t blocks = ((size_t)p->n * p->k + p->n + 32 * (wide ? V : 1) - 1) / (32 * (wide ? V : 1));
  const cudaError_t e = launch_dependent(wide ? product_reduce_kernel<T, V> : product_reduce_kernel<T, 1>,
                                         dim3((unsigned)std::min<size_t>(blocks, std::max(1, 4096 / p->experts)), (unsigned)p->experts), dim3(32, 8), 0, s, groups,
                                         (const T*)scratch, p->k, p->n, size, (T*)gw, (T*)gb);
  return e == cudaSuccess ? FASTEQ_OK : cuda_fail(e);
}

template <int TM, int TN>
int launch_wgrad_f64(const fasteq_product_problem* p, int size, const void* x, const void* g, const int32_t* offsets, void* gw, void* gb, void* scratch, cudaStream_t s) {
  const Groups groups = groups_of(p, offsets);
  const int tiles_k = (p->k + TN - 1) / TN, tiles = tiles_k * ((p->n + TM - 1) / TM);
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = allow_shared_memory<pf64::product_wgrad_f64_kernel<TM, TN>>(dev);
  if (e == cudaSuccess)
    e = launch_dependent(pf64::product_wgrad_f64_kernel<TM, TN>, (unsigned)((p->rows / size + p->experts) * tiles), pf64::NT, pf64::Shape<TM, TN, false, false>::SMEM, s, groups,
                         (const double*)x, (const double*)g, p->k, p->n, size, tiles_k, tiles, even(p->k, {x}), even(p->n, {g}), (double*)gw, (double*)gb, (double*)scratch);
  return e == cudaSuccess ? reduce<double>(p, groups, size, gw, gb, scratch, s) : cuda_fail(e);
}
int wgrad_f64(const fasteq_product_problem* p, int size, const void* x, const void* g, const int32_t* offsets, void* gw, void* gb, void* scratch, cudaStream_t s) {
  if (p->n <= 16) return p->k <= 16 ? launch_wgrad_f64<16, 16>(p, size, x, g, offsets, gw, gb, scratch, s) : launch_wgrad_f64<16, 64>(p, size, x, g, offsets, gw, gb, scratch, s);
  return p->k <= 16 ? launch_wgrad_f64<64, 16>(p, size, x, g, offsets, gw, gb, scratch, s) : launch_wgrad_f64<64, 64>(p, size, x, g, offsets, gw, gb, scratch, s);
}

template <typename T>
int wgrad(const fasteq_product_problem* p, int size, const void* x, const void* g, const void* slope, const int32_t* offsets, void* gw, void* gb, void* scratch,
          cudaStream_t s) {
  const Groups groups = groups_of(p, offsets);
  const long long tiles = (long long)((p->n + TILE - 1) / TILE) * std::max(1, (p->k + TILE - 1) / TILE);
  if (tiles > 65535) return FASTEQ_UNSUPPORTED;
  const cudaError_t e = launch_dependent(product_wgrad_kernel<T>, dim3((unsigned)(p->rows / size + p->experts), (unsigned)tiles), THREADS, 0, s, groups, (const T*)x,
                                         (const T*)g, (const T*)slope, p->k, p->n, slope_pitch(p), size, (T*)gw, (T*)gb, (T*)scratch);
  return e == cudaSuccess ? reduce<T>(p, groups, size, gw, gb, scratch, s) : cuda_fail(e);
}

// ------------------------------------------------------------------------------------------------ tensor cores
bool wide(int extent, std::initializer_list<const void*> pointers) {
  uintptr_t all = 0;
  for (const void* q : pointers) all |= reinterpret_cast<uintptr_t>(q);
  return extent % 4 == 0 && (all & 15u) == 0;
}

// Units of the tensor-core kernel (at most), which counts them, and a CTA's blocks, in 32 bits.
long long most_units(const fasteq_product_problem* p, int K, int N) {
  const long long units = (p->rows / ptc::BM + p->experts) * ((N + ptc::BN - 1) / ptc::BN);
  return units > 0x3fffffffLL || units * ((K + ptc::KB - 1) / ptc::KB) > 0x3fffffffLL ? -1 : units;
}
bool on_tensor_cores(const fasteq_product_problem* p) {
  return p->dtype == FASTEQ_F32 && p->k > 0 && p->n > 0 && p->rows > 0 && p->rows <= 0x7fffffffLL && most_units(p, p->k, p->n) > 0 && most_units(p, p->n, p->k) > 0;
}

// dst [rows, pitch] = src [rows, columns] (times slope, rows of ldd), zeros behind: rows that TMA cannot take as they lie, and FP64's gz
template <typename T, int V> __global__ void __launch_bounds__(256) align_rows_kernel(const T* src, const T* slope, int columns, int ldd, int pitch, long long rows, T* dst) {
  struct alignas(sizeof(T) * V) Pack { T v[V]; };
  wait_for_previous_kernel();
  for (long long r = (long long)blockIdx.x * blockDim.y + threadIdx.y; r < rows; r += (long long)gridDim.x * blockDim.y)
    for (int k = threadIdx.x * V; k < pitch; k += blockDim.x * V) {
      Pack x{};
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (k + i < columns) x.v[i] = src[r * columns + k + i];
        if (slope && k + i < columns) x.v[i] *= slope[r * ldd + k + i];
      }
      *reinterpret_cast<Pack*>(dst + r * pitch + k) = x;
    }
}
template <typename T> cudaError_t align_rows(const void* src, const void* slope, int columns, int ldd, int pitch, long long rows, void* dst, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const bool packs = pitch % V == 0;
  const int tx = std::min(32, packs ? pitch / V : pitch);      // not a power of two: 80,533 rows of 33 values 6.1 us, with 16 lanes a row 8.3 us
  const dim3 block((unsigned)tx, (unsigned)(256 / tx));
  return launch_dependent(packs ? align_rows_kernel<T, V> : align_rows_kernel<T, 1>, (unsigned)std::min<long long>((rows + block.y - 1) / block.y, 148 * 32), block, 0, s,
                          (const T*)src, (const T*)slope, columns, ldd, pitch, rows, (T*)dst);
}

// A call's scratch: the aligned copies, the weights split beforehand (none where a CTA keeps them), the weight gradient's partial sums.
struct Scratch {
  int64_t x = 0, g = 0, split = 0, partial = 0;
  int64_t total() const { return x + g + split + partial; }
};
int64_t round16(int64_t v) { return (v + 15) & ~(int64_t)15; }
Scratch scratch_of(const fasteq_product_problem* p, bool backward) {
  Scratch r;
  const bool tensor = on_tensor_cores(p);
  const int64_t size = p->dtype == FASTEQ_F32 ? 4 : 8;
  if (tensor) {
    const int K = backward ? p->n : p->k, N = backward ? p->k : p->n, n_kb = (K + ptc::KB - 1) / ptc::KB;
    const int slots = std::min(ptc::Cfg<false>::slots(p->experts), ptc::Cfg<true>::slots(p->experts));
    if (p->k % 4) r.x = round16(p->rows * ((p->k + 3) & ~3) * size);
    if (backward && p->n % 4) r.g = round16(p->rows * ((p->n + 3) & ~3) * size);
    if (n_kb > slots) r.split = (int64_t)p->experts * ((N + ptc::BN - 1) / ptc::BN) * n_kb * ptc::B_BYTES;
  }
  if (backward && p->dtype == FASTEQ_F64 && p->k > 0 && p->act != kIdentity) r.g = round16(p->rows * p->n * size);
  if (backward && p->rows > 0) {
    const int rows = chunk_rows(p, tensor);
    if (p->rows > rows) r.partial = partial_slots(p->rows, rows) * ((int64_t)p->n * p->k + p->n) * size;
  }
  return r;
}

template <bool FORWARD, bool SLOPE, int ACT>
int launch_tc(const fasteq_product_problem* p, ptc::Args& a, int dev, int sms, const CUtensorMap (&tm)[4], cudaStream_t s) {
  a.slots = ptc::Cfg<SLOPE>::slots(p->experts);
  const int smem = ptc::Cfg<SLOPE>::smem(a.slots, p->experts);
  cudaError_t e = allow_shared_memory<ptc::product_tc_kernel<FORWARD, SLOPE, ACT>>(dev);
  if (e == cudaSuccess)
    e = launch_dependent(ptc::product_tc_kernel<FORWARD, SLOPE, ACT>, (unsigned)std::min<long long>(sms, most_units(p, a.K, a.N)), ptc::NT, smem, s, a, tm[0], tm[1],
                         tm[2], tm[3]);
  return e == cudaSuccess ? FASTEQ_OK : cuda_fail(e);
}

// K and N as the kernel sees them (grad_x: exchanged); A and slope with rows of lda and ldd, 16-byte aligned
template <bool FORWARD>
int run_tc(const fasteq_product_problem* p, const void* A, int lda, const void* slope, const void* W, const void* bias, const void* residual,
           const int32_t* offsets, void* C, void* slope_out, void* split, cudaStream_t s) {
  ptc::Args a{};
  a.groups = groups_of(p, offsets);
  a.A = (const float*)A; a.slope = (const float*)slope; a.W = (const float*)W; a.bias = (const float*)bias; a.residual = (const float*)residual;
  a.C = (float*)C; a.slope_out = (float*)slope_out;
  a.K = FORWARD ? p->k : p->n; a.N = FORWARD ? p->n : p->k; a.lda = lda; a.ldd = slope_pitch(p);
  a.w_wide = wide(p->k, {W}); a.c_wide = wide(a.N, {C, residual});
  int dev = 0;
  Device* device = nullptr;
  cudaError_t e = current_device(&dev, &device);
  if (e != cudaSuccess) return cuda_fail(e);
  a.status = device->status;
  const int sms = device->sms;
  if (e == cudaSuccess && split) {
    const int n_tiles = (a.N + ptc::BN - 1) / ptc::BN, n_kb = (a.K + ptc::KB - 1) / ptc::KB;
    e = launch_dependent(ptc::split_weights_kernel<FORWARD>, (unsigned)((int64_t)p->experts * n_tiles * n_kb), 256, 0, s, a.W, (unsigned char*)split, a.N, a.K, n_tiles,
                         n_kb, a.w_wide);
    a.split = (const unsigned char*)split;
  }
  if (e != cudaSuccess) return cuda_fail(e);
  CUtensorMap tm[4] = {};               // A, its slope; C, its slope
  int rc = FASTEQ_OK;
  auto map = [&](int i, const float* base, int columns, int pitch, uint32_t box_rows) {
    if (rc == FASTEQ_OK && base) rc = tc::make_map(&tm[i], base, (uint64_t)columns, 1, (uint64_t)p->rows, (uint64_t)pitch, (uint64_t)pitch, 32, 1, box_rows);
  };
  map(0, a.A, a.K, a.lda, ptc::BM);
  map(1, a.slope, a.K, a.ldd, ptc::BM);
  if (a.c_wide) map(2, a.C, a.N, a.N, 32);
  map(3, a.slope_out, a.N, a.ldd, 32);
  if (rc != FASTEQ_OK) return rc;
  if (!FORWARD) return slope ? launch_tc<false, true, kIdentity>(p, a, dev, sms, tm, s) : launch_tc<false, false, kIdentity>(p, a, dev, sms, tm, s);
  switch (p->act) {
    case kSilu: return launch_tc<true, false, kSilu>(p, a, dev, sms, tm, s);
    case kTanh: return launch_tc<true, false, kTanh>(p, a, dev, sms, tm, s);
    case kSigmoid: return launch_tc<true, false, kSigmoid>(p, a, dev, sms, tm, s);
    case kAbs: return launch_tc<true, false, kAbs>(p, a, dev, sms, tm, s);
    default: return launch_tc<true, false, kIdentity>(p, a, dev, sms, tm, s);
  }
}

template <bool SLOPE>
int wgrad_tc(const fasteq_product_problem* p, const void* x, int ldx, const void* g, int ldg, const void* slope, const int32_t* offsets, void* gw, void* gb,
             void* partial, cudaStream_t s) {
  pwg::ArgsW a{};
  a.groups = groups_of(p, offsets);
  a.x = (const float*)x; a.g = (const float*)g; a.slope = (const float*)slope;
  a.gw = (float*)gw; a.gb = (float*)gb; a.partial = (float*)partial;
  a.K = p->k; a.N = p->n; a.ldx = ldx; a.ldg = ldg; a.ldd = slope_pitch(p); a.size = chunk_rows(p, true);
  a.tiles_k = (p->k + pwg::TN - 1) / pwg::TN;
  a.tiles = a.tiles_k * ((p->n + pwg::TM - 1) / pwg::TM);
  a.wide = wide(p->k, {gw}) && p->n % 4 == 0;
  CUtensorMap tm[3] = {};
  int rc = FASTEQ_OK;
  auto map = [&](int i, const float* base, int columns, int pitch, uint32_t box) {
    if (rc == FASTEQ_OK && base) rc = tc::make_map_pitched(&tm[i], base, columns, pitch, p->rows, box, pwg::ROWS);
  };
  map(0, a.g, p->n, ldg, pwg::TM); map(1, a.slope, p->n, a.ldd, pwg::TM); map(2, a.x, p->k, ldx, pwg::TN);
  if (rc != FASTEQ_OK) return rc;
  int dev = 0;
  Device* device = nullptr;
  cudaError_t e = current_device(&dev, &device);
  if (e == cudaSuccess) a.status = device->status;
  if (e == cudaSuccess) e = allow_shared_memory<pwg::product_wgrad_tc_kernel<SLOPE>>(dev);
  if (e == cudaSuccess)
    e = launch_dependent(pwg::product_wgrad_tc_kernel<SLOPE>, (unsigned)((p->rows / a.size + p->experts) * a.tiles), pwg::NTW, pwg::CfgW<SLOPE>::SMEM, s, a, tm[0], tm[1],
                         tm[2]);
  return e == cudaSuccess ? reduce<float>(p, a.groups, a.size, gw, gb, partial, s) : cuda_fail(e);
}

}  // namespace

extern "C" int fasteq_product_scratch(const fasteq_product_problem* p, int32_t backward, int64_t* bytes) {
  static const int32_t some = 0;
  if (!bytes) return FASTEQ_INVALID;
  if (const int rc = check(p, &some)) return rc;
  *bytes = scratch_of(p, backward != 0).total();
  return FASTEQ_OK;
}

extern "C" int fasteq_product_forward(const fasteq_product_problem* p, const void* x, const void* w, const void* bias, const void* residual,
                                      const int32_t* offsets, void* y, void* slope, void* scratch, int64_t scratch_bytes, fasteq_stream_t stream) {
  if (const int rc = check(p, offsets)) return rc;
  if (p->rows == 0 || p->n == 0) return FASTEQ_OK;
  if (p->act == kIdentity) slope = nullptr;
  const Scratch need = scratch_of(p, false);
  if (need.total() > 0 && !wide(0, {scratch})) return FASTEQ_INVALID;
  if (!y || (p->k > 0 && (!x || !w)) || (need.total() > 0 && (!scratch || scratch_bytes < need.total()))) return FASTEQ_INVALID;
  cudaStream_t s = (cudaStream_t)stream;
  if (on_tensor_cores(p) && (need.x || wide(0, {x})) && wide(0, {slope})) {
    char* at = (char*)scratch;
    if (need.x) {
      const cudaError_t e = align_rows<float>(x, nullptr, p->k, 0, (p->k + 3) & ~3, p->rows, at, s);
      if (e != cudaSuccess) return cuda_fail(e);
      x = at;
      at += need.x;
    }
    return run_tc<true>(p, x, (p->k + 3) & ~3, nullptr, w, bias, residual, offsets, y, slope, need.split ? at : nullptr, s);
  }
  if (p->dtype == FASTEQ_F32) return forward<float>(p, x, w, bias, residual, offsets, y, slope, s);
  if (p->k == 0 || !in_32_bits(p, TILE)) return forward<double>(p, x, w, bias, residual, offsets, y, slope, s);
  return product_f64<true>(p, x, w, bias, residual, offsets, y, slope, s);
}

extern "C" int fasteq_product_backward(const fasteq_product_problem* p, const void* x, const void* w, const void* grad_y, const void* slope,
                                       const int32_t* offsets, void* grad_x, void* grad_w, void* grad_bias, void* scratch, int64_t scratch_bytes,
                                       fasteq_stream_t stream) {
  if (const int rc = check(p, offsets)) return rc;
  if (!grad_x && !grad_w && !grad_bias) return FASTEQ_OK;
  if (p->act == kIdentity) slope = nullptr;
  if (grad_bias && !grad_w && p->k > 0) return FASTEQ_INVALID;
  const bool sums = grad_w || grad_bias, there = p->rows > 0 && p->n > 0;
  const Scratch need = scratch_of(p, true);
  if (need.total() > 0 && (!scratch || !wide(0, {scratch}) || scratch_bytes < need.total())) return FASTEQ_INVALID;
  if (there && (!grad_y || (p->act != kIdentity && !slope) || (grad_x && p->k > 0 && !w) || (sums && p->k > 0 && !x))) return FASTEQ_INVALID;
  cudaStream_t s = (cudaStream_t)stream;
  const size_t size = p->dtype == FASTEQ_F32 ? 4 : 8;
  cudaError_t e = cudaSuccess;
  if (!there) {                           // no rows, or no columns to sum over
    if (grad_x && p->rows > 0 && p->k > 0) e = cudaMemsetAsync(grad_x, 0, (size_t)p->rows * p->k * size, s);
    if (e == cudaSuccess && grad_w && p->n > 0 && p->k > 0) e = cudaMemsetAsync(grad_w, 0, (size_t)p->experts * p->n * p->k * size, s);
    if (e == cudaSuccess && grad_bias && p->n > 0) e = cudaMemsetAsync(grad_bias, 0, (size_t)p->experts * p->n * size, s);
    return e == cudaSuccess ? FASTEQ_OK : cuda_fail(e);
  }
  char *x_at = (char*)scratch, *g_at = x_at + need.x, *split_at = g_at + need.g, *partial_at = split_at + need.split;
  int rc = FASTEQ_OK;
  if (on_tensor_cores(p) && (need.g || wide(0, {grad_y})) && (need.x || !sums || wide(0, {x})) && wide(0, {slope})) {
    const int ldg = (p->n + 3) & ~3, ldx = (p->k + 3) & ~3;
    if (need.g) {                         // with the slope multiplied in, then
      e = align_rows<float>(grad_y, slope, p->n, ldg, ldg, p->rows, g_at, s);
      grad_y = g_at;
      slope = nullptr;
    }
    if (sums && need.x && e == cudaSuccess) {
      e = align_rows<float>(x, nullptr, p->k, 0, ldx, p->rows, x_at, s);
      x = x_at;
    }
    if (e != cudaSuccess) return cuda_fail(e);
    if (grad_x) rc = run_tc<false>(p, grad_y, ldg, slope, w, nullptr, nullptr, offsets, grad_x, nullptr, need.split ? split_at : nullptr, s);
    if (rc == FASTEQ_OK && sums)
      rc = slope ? wgrad_tc<true>(p, x, ldx, grad_y, ldg, slope, offsets, grad_w, grad_bias, partial_at, s)
                 : wgrad_tc<false>(p, x, ldx, grad_y, ldg, slope, offsets, grad_w, grad_bias, partial_at, s);
    return rc;
  }
  const int rows = chunk_rows(p, on_tensor_cores(p));      // as the scratch was counted with
  if (p->dtype == FASTEQ_F64 && p->k > 0 && in_32_bits(p, TILE)) {
    if (slope) {
      e = align_rows<double>(grad_y, slope, p->n, p->n, p->n, p->rows, g_at, s);
      if (e != cudaSuccess) return cuda_fail(e);
      grad_y = g_at;
    }
    if (grad_x) rc = product_f64<false>(p, grad_y, w, nullptr, nullptr, offsets, grad_x, nullptr, s);
    if (rc == FASTEQ_OK && sums) rc = wgrad_f64(p, rows, x, grad_y, offsets, grad_w, grad_bias, partial_at, s);
    return rc;
  }
  const bool f32 = p->dtype == FASTEQ_F32;
  if (grad_x && p->k > 0) rc = f32 ? dgrad<float>(p, grad_y, slope, w, offsets, grad_x, s) : dgrad<double>(p, grad_y, slope, w, offsets, grad_x, s);
  if (rc == FASTEQ_OK && sums)
    rc = f32 ? wgrad<float>(p, rows, x, grad_y, slope, offsets, grad_w, grad_bias, partial_at, s) : wgrad<double>(p, rows, x, grad_y, slope, offsets, grad_w, grad_bias, partial_at, s);
  return rc;
}
