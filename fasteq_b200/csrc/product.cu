// Dense layers with an epilogue, one matrix for all rows or one per expert (rows in the experts' order):
//   z = x W[e]^T + bias[e],  y = act(z) + residual;   gz = grad_y act'(z):  grad_x = gz W[e],  grad_w[e] = gz^T x,  grad_bias[e] = sum gz
// FMA kernels for every extent, FP32 and FP64: 64 x 64 tiles of 4 x 4 sums a thread.
#include <algorithm>
#include <cstdint>
#include <cuda_runtime.h>
#include "fasteq_b200.h"
#include "core_common.h"
#include "fasteq_device.cuh"
#include "launch.cuh"
#include "product.cuh"
#include "product_tc.cuh"
#include "gemm_tf32x3.h"

using namespace fasteq;
using namespace fasteq::product;

namespace {

constexpr int TILE = 64, BK = 16, PITCH = TILE + 4, THREADS = 256;

// One tile of C = epilogue(A op(W)).  A [rows, K], times `slope` where it is given.  FORWARD: W [N, K], bias, act and residual;
// else W [K, N] (grad_x: K the layer's outputs, N its inputs).
template <typename T, bool FORWARD>
__global__ void __launch_bounds__(THREADS) product_kernel(Groups groups, const T* A, const T* slope, const T* W, const T* bias, const T* residual,
                                                          int K, int N, int act, T* C, T* slope_out) {
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
        if (m < m_rows && k0 + k < K) v = slope ? A[at] * slope[at] : A[at];
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
      if (FORWARD && slope_out) slope_out[at] = d;
    }
  }
}

// ------------------------------------------------------------------------------------------------ weight gradient
// A chunk of an expert's rows and a tile of its matrix per CTA; the partial sums [chunk][N * K | N] are added by a second kernel in order.
constexpr int CHUNK_ROWS = 512;

template <typename T>
__global__ void __launch_bounds__(THREADS) product_wgrad_kernel(Groups groups, const T* X, const T* G, const T* slope, int K, int N, T* partial) {
  __shared__ __align__(16) T sg[BK][PITCH], sx[BK][PITCH];
  wait_for_previous_kernel();
  long long m0;
  int m_rows;
  tile_of<CHUNK_ROWS>(groups, groups.experts, blockIdx.x, &m0, &m_rows);
  if (m_rows == 0) return;
  const int tiles_k = max(1, (K + TILE - 1) / TILE), n0 = ((int)blockIdx.y / tiles_k) * TILE, k0 = ((int)blockIdx.y % tiles_k) * TILE;
  const int t = threadIdx.x, tn = (t / 16) * 4, tk = (t % 16) * 4;
  T sum[4][4] = {}, column = T(0);
  for (int r0 = 0; r0 < m_rows; r0 += BK) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = t % 64, r = t / 64 + 4 * i;
      const bool there = r0 + r < m_rows;
      const long long row = m0 + r0 + r;
      T g = T(0);
      if (there && n0 + c < N) {
        const long long at = row * N + n0 + c;
        g = slope ? G[at] * slope[at] : G[at];
      }
      sg[r][c] = g;
      sx[r][c] = there && k0 + c < K ? X[row * K + k0 + c] : T(0);
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
  T* dst = partial + (size_t)blockIdx.x * ((size_t)N * K + N);
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j)
      if (n0 + tn + i < N && k0 + tk + j < K) dst[(size_t)(n0 + tn + i) * K + k0 + tk + j] = sum[i][j];
  if (k0 == 0 && t < TILE && n0 + t < N) dst[(size_t)N * K + n0 + t] = column;
}

// 32 values of an expert to a CTA, eight threads to each, which take every eighth chunk and are added in order
template <typename T>
__global__ void __launch_bounds__(256) product_reduce_kernel(Groups groups, const T* partial, int K, int N, T* gw, T* gb) {
  __shared__ T part[8][33];
  wait_for_previous_kernel();
  const int e = blockIdx.y;
  const size_t nk = (size_t)N * K, all = nk + N, i = (size_t)blockIdx.x * 32 + threadIdx.x;
  const long long begin = groups.first(e), end = groups.first(e + 1), c0 = begin / CHUNK_ROWS + e, n = (end - begin + CHUNK_ROWS - 1) / CHUNK_ROWS;
  T s = T(0);
  if (i < all) {
#pragma unroll 4
    for (long long c = threadIdx.y; c < n; c += 8) s += partial[(size_t)(c0 + c) * all + i];
  }
  part[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && i < all) {
#pragma unroll
    for (int j = 1; j < 8; ++j) s += part[j][threadIdx.x];
    if (i < nk) gw[(size_t)e * nk + i] = s;
    else if (gb) gb[(size_t)e * N + (i - nk)] = s;
  }
}

// ------------------------------------------------------------------------------------------------ entries
int check(const fasteq_product_problem* p, const int32_t* offsets) {
  if (!p || (p->dtype != FASTEQ_F32 && p->dtype != FASTEQ_F64) || p->k < 0 || p->n < 0 || p->rows < 0 || p->experts < 1 || p->inner < 1 ||
      p->act < 0 || p->act > 4 || (!offsets && p->experts != 1))
    return FASTEQ_INVALID;
  if (p->experts > FASTEQ_MAX_EXPERTS || p->rows / p->inner > 0x7fff0000LL || p->rows / TILE > 0x7fff0000LL || p->n > TILE * 65535LL || p->k > TILE * 65535LL)
    return FASTEQ_UNSUPPORTED;
  return FASTEQ_OK;
}
Groups groups_of(const fasteq_product_problem* p, const int32_t* offsets) { return Groups{offsets, p->experts, p->inner, (long long)p->rows}; }

template <typename T>
int forward(const fasteq_product_problem* p, const void* x, const void* w, const void* bias, const void* residual, const int32_t* offsets, void* y,
            void* slope, cudaStream_t s) {
  const dim3 grid((unsigned)tile_numbers<TILE>(p->rows, p->experts + 1), (unsigned)((p->n + TILE - 1) / TILE));
  const cudaError_t e = launch_dependent(product_kernel<T, true>, grid, THREADS, 0, s, groups_of(p, offsets), (const T*)x, (const T*)nullptr, (const T*)w,
                                         (const T*)bias, (const T*)residual, p->k, p->n, p->act, (T*)y, (T*)slope);
  return e == cudaSuccess ? FASTEQ_OK : cuda_fail(e);
}
template <typename T>
int dgrad(const fasteq_product_problem* p, const void* g, const void* slope, const void* w, const int32_t* offsets, void* gx, cudaStream_t s) {
  const dim3 grid((unsigned)tile_numbers<TILE>(p->rows, p->experts + 1), (unsigned)((p->k + TILE - 1) / TILE));
  const cudaError_t e = launch_dependent(product_kernel<T, false>, grid, THREADS, 0, s, groups_of(p, offsets), (const T*)g, (const T*)slope, (const T*)w,
                                         (const T*)nullptr, (const T*)nullptr, p->n, p->k, 0, (T*)gx, (T*)nullptr);
  return e == cudaSuccess ? FASTEQ_OK : cuda_fail(e);
}
template <typename T>
int wgrad(const fasteq_product_problem* p, const void* x, const void* g, const void* slope, const int32_t* offsets, void* gw, void* gb, void* scratch,
          cudaStream_t s) {
  const Groups groups = groups_of(p, offsets);
  const int tiles = ((p->n + TILE - 1) / TILE) * std::max(1, (p->k + TILE - 1) / TILE);
  cudaError_t e = cudaSuccess;
  if (p->rows == 0) {
    if (p->k > 0) e = cudaMemsetAsync(gw, 0, (size_t)p->experts * p->n * p->k * sizeof(T), s);
    if (e == cudaSuccess && gb) e = cudaMemsetAsync(gb, 0, (size_t)p->experts * p->n * sizeof(T), s);
    return e == cudaSuccess ? FASTEQ_OK : cuda_fail(e);
  }
  e = launch_dependent(product_wgrad_kernel<T>, dim3((unsigned)tile_numbers<CHUNK_ROWS>(p->rows, p->experts), (unsigned)tiles), THREADS, 0, s, groups, (const T*)x,
                       (const T*)g, (const T*)slope, p->k, p->n, (T*)scratch);
  if (e == cudaSuccess)
    e = launch_dependent(product_reduce_kernel<T>, dim3((unsigned)(((size_t)p->n * p->k + p->n + 31) / 32), (unsigned)p->experts), dim3(32, 8), 0, s, groups,
                         (const T*)scratch, p->k, p->n, (T*)gw, (T*)gb);
  return e == cudaSuccess ? FASTEQ_OK : cuda_fail(e);
}

}  // namespace

namespace {

bool wide(int extent, std::initializer_list<const void*> pointers) {
  uintptr_t all = 0;
  for (const void* q : pointers) all |= reinterpret_cast<uintptr_t>(q);
  return extent % 4 == 0 && (all & 15u) == 0;
}

// Units of the tensor-core kernel (at most), which counts them, and a CTA's blocks, in 32 bits.
long long most_units(const fasteq_product_problem* p, int K, int N) {
  const long long units = (p->rows / ptc::BM + p->experts) * ((N + ptc::BN - 1) / ptc::BN);
  return units > 0x7fffffffLL || (units / 64 + 1) * ((K + ptc::KB - 1) / ptc::KB) > 0x3fffffffLL ? -1 : units;
}

// bytes of the weights split beforehand: none where a CTA keeps them
int64_t split_bytes(const fasteq_product_problem* p, bool forward) {
  const int K = forward ? p->k : p->n, N = forward ? p->n : p->k, n_kb = (K + ptc::KB - 1) / ptc::KB;
  if (p->dtype != FASTEQ_F32 || K == 0 || N == 0 || p->rows == 0 || most_units(p, K, N) < 0) return 0;
  const int slots = forward ? ptc::Cfg<false>::slots(p->experts) : ptc::Cfg<true>::slots(p->experts);
  return n_kb <= std::min(slots, ptc::Cfg<false>::slots(p->experts)) ? 0 : (int64_t)p->experts * ((N + ptc::BN - 1) / ptc::BN) * n_kb * ptc::B_BYTES;
}

template <bool FORWARD, bool SLOPE, int ACT>
int launch_tc(const fasteq_product_problem* p, ptc::Args& a, int sms, const CUtensorMap (&tm)[4], cudaStream_t s) {
  a.slots = ptc::Cfg<SLOPE>::slots(p->experts);
  const int smem = ptc::Cfg<SLOPE>::smem(a.slots, p->experts);
  cudaError_t e = cudaFuncSetAttribute(ptc::product_tc_kernel<FORWARD, SLOPE, ACT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess)
    e = launch_dependent(ptc::product_tc_kernel<FORWARD, SLOPE, ACT>, (unsigned)std::min<long long>(sms, most_units(p, a.K, a.N)), ptc::NT, smem, s, a, tm[0], tm[1], tm[2], tm[3]);
  return e == cudaSuccess ? FASTEQ_OK : cuda_fail(e);
}

// K and N as the kernel sees them (grad_x: exchanged)
template <bool FORWARD>
int run_tc(const fasteq_product_problem* p, const void* A, const void* slope, const void* W, const void* bias, const void* residual,
           const int32_t* offsets, void* C, void* slope_out, void* scratch, cudaStream_t s) {
  ptc::Args a{};
  a.groups = groups_of(p, offsets);
  a.A = (const float*)A; a.slope = (const float*)slope; a.W = (const float*)W; a.bias = (const float*)bias; a.residual = (const float*)residual;
  a.C = (float*)C; a.slope_out = (float*)slope_out;
  a.K = FORWARD ? p->k : p->n; a.N = FORWARD ? p->n : p->k;
  a.a_wide = wide(a.K, {A, slope}) && p->rows <= 0x7fffffffLL; a.w_wide = wide(p->k, {W}); a.c_wide = wide(a.N, {C, slope_out, bias, residual}) && p->rows <= 0x7fffffffLL;
  int sms = 0, dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e == cudaSuccess) e = tc::status_word(&a.status);
  if (e != cudaSuccess) return cuda_fail(e);
  if (split_bytes(p, FORWARD) > 0) {
    const int n_tiles = (a.N + ptc::BN - 1) / ptc::BN, n_kb = (a.K + ptc::KB - 1) / ptc::KB;
    e = launch_dependent(ptc::split_weights_kernel<FORWARD>, (unsigned)((int64_t)p->experts * n_tiles * n_kb), 256, 0, s, a.W, (unsigned char*)scratch, a.N, a.K,
                         n_tiles, n_kb, a.w_wide);
    if (e != cudaSuccess) return cuda_fail(e);
    a.split = (const unsigned char*)scratch;
  }
  CUtensorMap tm[4] = {};               // A, its slope; C, its slope
  int rc = FASTEQ_OK;
  auto map = [&](int i, const float* base, int columns, uint32_t box_rows) {
    if (rc == FASTEQ_OK && base) rc = tc::make_map(&tm[i], base, (uint64_t)columns, 1, (uint64_t)p->rows, (uint64_t)columns, (uint64_t)columns, 32, 1, box_rows);
  };
  if (a.a_wide) { map(0, a.A, a.K, ptc::BM); map(1, a.slope, a.K, ptc::BM); }
  if (a.c_wide) { map(2, a.C, a.N, 32); map(3, a.slope_out, a.N, 32); }
  if (rc != FASTEQ_OK) return rc;
  if (!FORWARD) return slope ? launch_tc<false, true, kIdentity>(p, a, sms, tm, s) : launch_tc<false, false, kIdentity>(p, a, sms, tm, s);
  switch (p->act) {
    case kSilu: return launch_tc<true, false, kSilu>(p, a, sms, tm, s);
    case kTanh: return launch_tc<true, false, kTanh>(p, a, sms, tm, s);
    case kSigmoid: return launch_tc<true, false, kSigmoid>(p, a, sms, tm, s);
    case kAbs: return launch_tc<true, false, kAbs>(p, a, sms, tm, s);
    default: return launch_tc<true, false, kIdentity>(p, a, sms, tm, s);
  }
}

}  // namespace

extern "C" int fasteq_product_scratch(const fasteq_product_problem* p, int32_t grad_x, int64_t* bytes) {
  static const int32_t some = 0;
  if (!bytes) return FASTEQ_INVALID;
  if (const int rc = check(p, &some)) return rc;
  *bytes = split_bytes(p, !grad_x);
  return FASTEQ_OK;
}

extern "C" int fasteq_product_forward(const fasteq_product_problem* p, const void* x, const void* w, const void* bias, const void* residual,
                                      const int32_t* offsets, void* y, void* slope, void* scratch, int64_t scratch_bytes, fasteq_stream_t stream) {
  if (const int rc = check(p, offsets)) return rc;
  if (p->rows == 0 || p->n == 0) return FASTEQ_OK;
  const int64_t need = split_bytes(p, true);
  if (!y || (p->k > 0 && (!x || !w)) || (need > 0 && (!scratch || scratch_bytes < need))) return FASTEQ_INVALID;
  if (p->dtype == FASTEQ_F32 && p->k > 0 && most_units(p, p->k, p->n) > 0)
    return run_tc<true>(p, x, nullptr, w, bias, residual, offsets, y, slope, scratch, (cudaStream_t)stream);
  return p->dtype == FASTEQ_F32 ? forward<float>(p, x, w, bias, residual, offsets, y, slope, (cudaStream_t)stream)
                                : forward<double>(p, x, w, bias, residual, offsets, y, slope, (cudaStream_t)stream);
}

extern "C" int fasteq_product_dgrad(const fasteq_product_problem* p, const void* grad_y, const void* slope, const void* w, const int32_t* offsets,
                                    void* grad_x, void* scratch, int64_t scratch_bytes, fasteq_stream_t stream) {
  if (const int rc = check(p, offsets)) return rc;
  if (p->rows == 0 || p->k == 0) return FASTEQ_OK;
  const int64_t need = split_bytes(p, false);
  if (!grad_x || (p->n > 0 && (!grad_y || !w)) || (need > 0 && (!scratch || scratch_bytes < need))) return FASTEQ_INVALID;
  if (p->dtype == FASTEQ_F32 && p->n > 0 && most_units(p, p->n, p->k) > 0)
    return run_tc<false>(p, grad_y, slope, w, nullptr, nullptr, offsets, grad_x, nullptr, scratch, (cudaStream_t)stream);
  return p->dtype == FASTEQ_F32 ? dgrad<float>(p, grad_y, slope, w, offsets, grad_x, (cudaStream_t)stream)
                                : dgrad<double>(p, grad_y, slope, w, offsets, grad_x, (cudaStream_t)stream);
}

extern "C" int fasteq_product_wgrad_scratch(const fasteq_product_problem* p, int64_t* bytes) {
  static const int32_t some = 0;
  if (!bytes) return FASTEQ_INVALID;
  if (const int rc = check(p, &some)) return rc;
  *bytes = tile_numbers<CHUNK_ROWS>(p->rows, p->experts) * ((int64_t)p->n * p->k + p->n) * (p->dtype == FASTEQ_F32 ? 4 : 8);
  return FASTEQ_OK;
}

extern "C" int fasteq_product_wgrad(const fasteq_product_problem* p, const void* x, const void* grad_y, const void* slope, const int32_t* offsets,
                                    void* grad_w, void* grad_bias, void* scratch, int64_t scratch_bytes, fasteq_stream_t stream) {
  if (const int rc = check(p, offsets)) return rc;
  int64_t need = 0;
  if (const int rc = fasteq_product_wgrad_scratch(p, &need)) return rc;
  if (p->n == 0) return FASTEQ_OK;
  if ((p->k > 0 && !grad_w) || (need > 0 && (!scratch || scratch_bytes < need)) || (p->rows > 0 && (!grad_y || (p->k > 0 && !x)))) return FASTEQ_INVALID;
  return p->dtype == FASTEQ_F32 ? wgrad<float>(p, x, grad_y, slope, offsets, grad_w, grad_bias, scratch, (cudaStream_t)stream)
                                : wgrad<double>(p, x, grad_y, slope, offsets, grad_w, grad_bias, scratch, (cudaStream_t)stream);
}
