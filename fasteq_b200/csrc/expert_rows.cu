// Rows in the order of the experts their entries are given to, and back.
//
// An entry is a (token, slot) pair i = t * slots + s with expert e_i; a negative expert means none.  With key(i) = e_i, or X for none,
//   position[i] = #{j : key(j) < key(i)} + #{j < i : key(j) = key(i)}         (a stable counting sort)
//   offsets[x]  = #{j : key(j) < x},  x = 0 .. X                              (rows from offsets[X] on belong to no expert)
//   gather   rows[position[i]] = x[t]                  (0 for no expert)      gradient: grad_x[t] = sum_s grad_rows[position[t, s]]
//   combine  y[t] = sum_s w[t, s] rows[position[t, s]]                        gradients: grad_rows[position] = w grad_y[t],
//                                                                             grad_w[t, s] = <rows[position], grad_y[t]>
// The permutation is known from both sides, so every sum is a walk over a token's slots in their order: no atomics, the same bits every time.
// Bound: memory, each row tensor once; a token's row is read once for all its slots.  Rows are loaded and stored past the caches' order of use
// (__ldcs, __stcs): 301,746 rows of 512 FP32 values take 142 us to gather (927 MB, 6.5 TB/s, the rate of a copy), 151 us to combine, 243 us for the
// gradients of the combination; with ordinary accesses the gather's own gradient took 177 us instead of 151 us, behind a kernel that left the L2 full.
#include <cstdint>
#include <cuda_runtime.h>
#include "fasteq_b200.h"
#include "core_common.h"
#include "fasteq_device.cuh"
#include "launch.cuh"

using namespace fasteq;

namespace {

__device__ int g_expert_status;

constexpr int PLAN_THREADS = 1024, PLAN_WARPS = PLAN_THREADS / 32;
// Entries of a CTA: GROUPS of 32 a warp, held in registers.  One group keeps a CTA's chain short (1,000 entries of 8 experts 3.9 us, with four groups 5.0 us;
// 20,000 in 3.1 + 4.8 us to count and to place, 4.6 + 6.9 us; 300,000 of 89 experts 5.9 + 14.4 us, 7.9 + 14.5 us).  Four where they leave one CTA, which
// needs no counts before it (4,000 entries of 8 experts 6.2 us, with one group 3.1 + 4.8 us), and where there would be so many CTAs that
// adding up all their counts in each takes over.
constexpr int MOST_GROUPS = 4, MANY = 512 * 1024;
int groups_for(long long n) { return n <= PLAN_THREADS || (n > MOST_GROUPS * PLAN_THREADS && n <= MANY) ? 1 : MOST_GROUPS; }

// 64-bit expert numbers as torch's top-k gives them, or 32-bit ones; experts that are not there count as none and are reported
template <typename I> __device__ __forceinline__ int key_of(const I* expert, long long i, int X) {
  const I e = *reinterpret_cast<const volatile I*>(expert + i);
  if (e < 0) return X;
  if (e >= (I)X) { atomicExch(&g_expert_status, (int)kDevBadIndex); return X; }
  return (int)e;
}

// This warp's entries (first + 32 g + lane), their keys in registers, -1 beyond the end.
template <typename I, int GROUPS> __device__ __forceinline__ void load_keys(const I* expert, long long first, long long n, int X, int (&keys)[GROUPS]) {
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) {
    const long long i = first + g * 32 + (threadIdx.x & 31);
    keys[g] = i < n ? key_of(expert, i, X) : -1;
  }
}
// Entries of equal key in a group find each other; the first of them counts for all.  counts: this warp's [X + 1].
template <int GROUPS> __device__ __forceinline__ void count_entries(const int (&keys)[GROUPS], int* counts) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) {
    const unsigned same = __match_any_sync(0xffffffffu, keys[g]);
    if (keys[g] >= 0 && lane == __ffs(same) - 1) counts[keys[g]] += __popc(same);
    __syncwarp();
  }
}
template <int GROUPS> __device__ __forceinline__ void place_entries(const int (&keys)[GROUPS], long long first, int* next, int* position) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) {
    const unsigned same = __match_any_sync(0xffffffffu, keys[g]);
    if (keys[g] >= 0) position[first + g * 32 + lane] = next[keys[g]] + __popc(same & ((1u << lane) - 1u));
    __syncwarp();
    if (keys[g] >= 0 && lane == __ffs(same) - 1) next[keys[g]] += __popc(same);
    __syncwarp();
  }
}

// exclusive prefix sums of v[0 .. n) in shared memory (all threads); n <= PLAN_THREADS + 1
__device__ __forceinline__ void scan_keys(int* v, int n, int* warp_sums) {
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int mine = t < n ? v[t] : 0;
  int sum = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += u;
  }
  if (lane == 31) warp_sums[warp] = sum;
  __syncthreads();
  if (warp == 0) {
    int w = warp_sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += u;
    }
    warp_sums[lane] = w;
  }
  __syncthreads();
  const int before = sum - mine + (warp ? warp_sums[warp - 1] : 0);
  if (t < n) v[t] = before;
  if (n > PLAN_THREADS && t == PLAN_THREADS - 1) v[PLAN_THREADS] = before + mine;
  __syncthreads();
}

// counts of the warps [warp][K] -> counts of the warps before; their sums to total (may be null).  A warp to a key.
__device__ __forceinline__ void scan_warps(int* counts, int K, int* total) {
  const int lane = threadIdx.x & 31;
  for (int k = threadIdx.x >> 5; k < K; k += PLAN_WARPS) {
    const int mine = counts[lane * K + k];
    int sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += u;
    }
    counts[lane * K + k] = sum - mine;
    if (total && lane == 31) total[k] = sum;
  }
}

template <typename I, int GROUPS> __global__ void __launch_bounds__(PLAN_THREADS) expert_count_kernel(const I* expert, long long n, int X, int* counts) {
  extern __shared__ int sm[];                       // [PLAN_WARPS][X + 1] | [X + 1]
  const int K = X + 1;
  for (int j = threadIdx.x; j < PLAN_WARPS * K; j += PLAN_THREADS) sm[j] = 0;
  wait_for_previous_kernel();
  int keys[GROUPS];
  load_keys<I, GROUPS>(expert, ((long long)blockIdx.x * PLAN_WARPS + (threadIdx.x >> 5)) * 32 * GROUPS, n, X, keys);
  __syncthreads();
  count_entries<GROUPS>(keys, sm + (threadIdx.x >> 5) * K);
  __syncthreads();
  scan_warps(sm, K, sm + PLAN_WARPS * K);
  __syncthreads();
  for (int k = threadIdx.x; k < K; k += PLAN_THREADS) counts[(long long)blockIdx.x * K + k] = sm[PLAN_WARPS * K + k];
}

// One CTA (`counts` null), or several, their counts known.
template <typename I, int GROUPS>
__global__ void __launch_bounds__(PLAN_THREADS) expert_place_kernel(const I* expert, long long n, int X, const int* counts, int* position, int* offsets) {
  extern __shared__ int sm[];                       // [PLAN_WARPS][X + 1] | [X + 1] totals | [X + 1] of earlier CTAs | [32]
  const int K = X + 1;
  int *total = sm + PLAN_WARPS * K, *earlier = total + K, *warp_sums = earlier + K;
  for (int j = threadIdx.x; j < PLAN_WARPS * K; j += PLAN_THREADS) sm[j] = 0;
  for (int k = threadIdx.x; k < K; k += PLAN_THREADS) total[k] = earlier[k] = 0;
  wait_for_previous_kernel();
  const long long first = ((long long)blockIdx.x * PLAN_WARPS + (threadIdx.x >> 5)) * 32 * GROUPS;
  int keys[GROUPS];
  load_keys<I, GROUPS>(expert, first, n, X, keys);
  __syncthreads();
  if (counts) {
    // all CTAs' counts, a key and a share of the CTAs to each thread; whole numbers, so that the order of the additions does not matter
    const int parts = max(1, PLAN_THREADS / K), n_ctas = (int)gridDim.x;
    for (int j = threadIdx.x; j < parts * K; j += PLAN_THREADS) {
      const int k = j % K, p = j / K;
      int s = 0, b = 0;
#pragma unroll 8
      for (int c = p; c < n_ctas; c += parts) {
        const int v = counts[(long long)c * K + k];
        s += v;
        if (c < (int)blockIdx.x) b += v;
      }
      atomicAdd(&total[k], s);
      atomicAdd(&earlier[k], b);
    }
  }
  count_entries<GROUPS>(keys, sm + (threadIdx.x >> 5) * K);
  __syncthreads();
  scan_warps(sm, K, counts ? nullptr : total);
  __syncthreads();
  scan_keys(total, K, warp_sums);
  if (blockIdx.x == 0)
    for (int k = threadIdx.x; k < K; k += PLAN_THREADS) offsets[k] = total[k];
  for (int j = threadIdx.x; j < PLAN_WARPS * K; j += PLAN_THREADS) {
    const int k = j % K;
    sm[j] += total[k] + earlier[k];
  }
  __syncthreads();
  place_entries<GROUPS>(keys, first, sm + (threadIdx.x >> 5) * K, position);
}

constexpr size_t count_smem(int K) { return (size_t)(PLAN_WARPS + 1) * K * 4; }
constexpr size_t place_smem(int K) { return ((size_t)(PLAN_WARPS + 2) * K + 32) * 4; }
int plan_ctas(long long n) { return (int)((n + groups_for(n) * PLAN_THREADS - 1) / (groups_for(n) * PLAN_THREADS)); }

template <typename I, int GROUPS>
int launch_plan(const void* expert, long long n, int X, int* position, int* offsets, void* scratch, cudaStream_t s) {
  const int K = X + 1, ctas = plan_ctas(n);
  cudaError_t e = cudaSuccess;
  if (place_smem(K) > 48 * 1024) {       // the same limit in every call: another thread may be between this and its launch
    constexpr int MOST = FASTEQ_MAX_EXPERTS + 1;
    e = cudaFuncSetAttribute(expert_count_kernel<I, GROUPS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)count_smem(MOST));
    if (e == cudaSuccess) e = cudaFuncSetAttribute(expert_place_kernel<I, GROUPS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)place_smem(MOST));
    if (e != cudaSuccess) return cuda_fail(e);
  }
  const int* counts = nullptr;
  if (ctas > 1) {
    e = launch_dependent(expert_count_kernel<I, GROUPS>, (unsigned)ctas, PLAN_THREADS, count_smem(K), s, (const I*)expert, n, X, (int*)scratch);
    if (e != cudaSuccess) return cuda_fail(e);
    counts = (const int*)scratch;
  }
  e = launch_dependent(expert_place_kernel<I, GROUPS>, (unsigned)(ctas > 1 ? ctas : 1), PLAN_THREADS, place_smem(K), s, (const I*)expert, n, X, counts, position, offsets);
  return e == cudaSuccess ? FASTEQ_OK : cuda_fail(e);
}
template <typename I> int launch_plan(const void* expert, long long n, int X, int* position, int* offsets, void* scratch, cudaStream_t s) {
  return groups_for(n) == 1 ? launch_plan<I, 1>(expert, n, X, position, offsets, scratch, s) : launch_plan<I, MOST_GROUPS>(expert, n, X, position, offsets, scratch, s);
}

// ------------------------------------------------------------------------------------------------ rows
// blockDim = (tx, ty): tx threads (a power of two) walk a row's packs of V values, ty tokens to a CTA
template <typename T, int V> struct alignas(sizeof(T) * V) Pack { T v[V]; };
template <typename T, int V> __device__ __forceinline__ Pack<T, V> read_once(const T* p, long long i) {
  Pack<T, V> r;
  if constexpr (sizeof(r) == 16) {
    *reinterpret_cast<float4*>(&r) = __ldcs(reinterpret_cast<const float4*>(p) + i);
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) r.v[k] = __ldcs(p + i * V + k);
  }
  return r;
}
template <typename T, int V> __device__ __forceinline__ void write_once(T* p, long long i, const Pack<T, V>& r) {
  if constexpr (sizeof(r) == 16) {
    __stcs(reinterpret_cast<float4*>(p) + i, *reinterpret_cast<const float4*>(&r));
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) __stcs(p + i * V + k, r.v[k]);
  }
}

// An entry's row.  Positions are the caller's memory: one that is not among the rows is reported and becomes -1, which no kernel reads or writes at.
__device__ __forceinline__ int row_of(const int* position, long long entry, long long entries) {
  const int p = position[entry];
  if (p >= 0 && p < entries) return p;
  atomicExch(&g_expert_status, (int)kDevBadIndex);
  return -1;
}

template <typename T, int V>
__global__ void __launch_bounds__(256) expert_gather_kernel(const T* x, const int* position, const int* offsets, int X, long long tokens, int slots,
                                                            int packs, T* rows) {
  using P = Pack<T, V>;
  wait_for_previous_kernel();
  const int routed = offsets[X];
  const long long entries = tokens * slots;
  for (long long t = (long long)blockIdx.x * blockDim.y + threadIdx.y; t < tokens; t += (long long)gridDim.x * blockDim.y) {
    for (int c = threadIdx.x; c < packs; c += blockDim.x) {
      const P v = read_once<T, V>(x, t * packs + c);
      for (int s = 0; s < slots; ++s) {
        const int p = row_of(position, t * slots + s, entries);
        if (p >= 0) write_once<T, V>(rows, (long long)p * packs + c, p < routed ? v : P{});
      }
    }
  }
}

template <typename T, int V, bool WEIGHTED>
__global__ void __launch_bounds__(256) expert_combine_kernel(const T* rows, const T* weight, const int* position, const int* offsets, int X,
                                                             long long tokens, int slots, int packs, T* y) {
  using P = Pack<T, V>;
  wait_for_previous_kernel();
  const int routed = offsets[X];
  const long long entries = tokens * slots;
  for (long long t = (long long)blockIdx.x * blockDim.y + threadIdx.y; t < tokens; t += (long long)gridDim.x * blockDim.y) {
    for (int c = threadIdx.x; c < packs; c += blockDim.x) {
      P sum{};
      for (int s = 0; s < slots; ++s) {
        const int p = row_of(position, t * slots + s, entries);
        if (p < 0 || p >= routed) continue;
        const P v = read_once<T, V>(rows, (long long)p * packs + c);
        const T w = WEIGHTED ? weight[t * slots + s] : T(1);
#pragma unroll
        for (int k = 0; k < V; ++k) sum.v[k] = WEIGHTED ? vfma(w, v.v[k], sum.v[k]) : sum.v[k] + v.v[k];
      }
      write_once<T, V>(y, t * packs + c, sum);
    }
  }
}

// grad_rows and grad_w (either may be null).  tx <= 32: a token's threads are lanes of one warp.
template <typename T, int V>
__global__ void __launch_bounds__(256) expert_combine_backward_kernel(const T* rows, const T* weight, const T* g, const int* position,
                                                                      const int* offsets, int X, long long tokens, int slots, int packs, T* grows,
                                                                      T* gweight) {
  using P = Pack<T, V>;
  wait_for_previous_kernel();
  const int routed = offsets[X];
  const long long entries = tokens * slots;
  const long long step = (long long)gridDim.x * blockDim.y;
  // whole warps run the loop together, for the sums over their lanes
  const long long rounds = (tokens + step - 1) / step;
  for (long long r = 0; r < rounds; ++r) {
    const long long t = r * step + (long long)blockIdx.x * blockDim.y + threadIdx.y;
    const bool there = t < tokens;
    for (int s = 0; s < slots; ++s) {
      const int p = there ? row_of(position, t * slots + s, entries) : -1;
      const bool live = p >= 0 && p < routed;
      const T w = live && grows ? weight[t * slots + s] : T(0);
      T dot = T(0);
      if (there) {
#pragma unroll 4
        for (int c = threadIdx.x; c < packs; c += blockDim.x) {
          P o{};
          if (live) {
            const P gv = reinterpret_cast<const P*>(g)[t * packs + c];
            if (gweight) {
              const P v = read_once<T, V>(rows, (long long)p * packs + c);
#pragma unroll
              for (int k = 0; k < V; ++k) dot = vfma(v.v[k], gv.v[k], dot);
            }
#pragma unroll
            for (int k = 0; k < V; ++k) o.v[k] = w * gv.v[k];
          }
          if (grows && p >= 0) write_once<T, V>(grows, (long long)p * packs + c, o);
        }
      }
      if (gweight) {
        for (int o = blockDim.x >> 1; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
        if (there && threadIdx.x == 0) gweight[t * slots + s] = dot;
      }
    }
  }
}

struct Shape {
  dim3 grid, block;
  int packs;
};
template <typename T, int V> Shape shape_of(long long tokens, int width, int most_x) {
  Shape r;
  r.packs = width / V;
  int tx = 1;
  while (tx < r.packs && tx < most_x) tx *= 2;
  r.block = dim3((unsigned)tx, (unsigned)(256 / tx));
  const long long blocks = (tokens + r.block.y - 1) / r.block.y;
  r.grid = dim3((unsigned)(blocks < 148 * 64 ? blocks : 148 * 64));
  return r;
}
bool aligned16(const void* a, const void* b, const void* c = nullptr) {
  return ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(c)) & 15u) == 0;
}

template <typename T, int V>
int gather(const void* x, const int* position, const int* offsets, int X, long long tokens, int slots, int width, void* rows, cudaStream_t s) {
  const Shape h = shape_of<T, V>(tokens, width, 256);
  const cudaError_t e = launch_dependent(expert_gather_kernel<T, V>, h.grid, h.block, 0, s, (const T*)x, position, offsets, X, tokens, slots, h.packs, (T*)rows);
  return e == cudaSuccess ? FASTEQ_OK : cuda_fail(e);
}
template <typename T, int V>
int combine(const void* rows, const void* weight, const int* position, const int* offsets, int X, long long tokens, int slots, int width, void* y,
            cudaStream_t s) {
  const Shape h = shape_of<T, V>(tokens, width, 256);
  const cudaError_t e = weight ? launch_dependent(expert_combine_kernel<T, V, true>, h.grid, h.block, 0, s, (const T*)rows, (const T*)weight, position, offsets, X, tokens, slots, h.packs, (T*)y)
                               : launch_dependent(expert_combine_kernel<T, V, false>, h.grid, h.block, 0, s, (const T*)rows, (const T*)weight, position, offsets, X, tokens, slots, h.packs, (T*)y);
  return e == cudaSuccess ? FASTEQ_OK : cuda_fail(e);
}
template <typename T, int V>
int combine_backward(const void* rows, const void* weight, const void* g, const int* position, const int* offsets, int X, long long tokens, int slots,
                     int width, void* grows, void* gweight, cudaStream_t s) {
  const Shape h = shape_of<T, V>(tokens, width, 32);
  const cudaError_t e = launch_dependent(expert_combine_backward_kernel<T, V>, h.grid, h.block, 0, s, (const T*)rows, (const T*)weight, (const T*)g, position, offsets, X,
                                         tokens, slots, h.packs, (T*)grows, (T*)gweight);
  return e == cudaSuccess ? FASTEQ_OK : cuda_fail(e);
}

bool sizes_ok(int32_t dtype, int64_t tokens, int32_t slots, int32_t experts, int32_t width) {
  return (dtype == FASTEQ_F32 || dtype == FASTEQ_F64) && tokens >= 0 && slots >= 1 && experts >= 1 && width >= 0;
}

}  // namespace

extern "C" int fasteq_expert_plan_scratch(int64_t entries, int32_t experts, int64_t* bytes) {
  if (!bytes || entries < 0 || experts < 1) return FASTEQ_INVALID;
  if (experts > FASTEQ_MAX_EXPERTS || entries > 0x7fff0000LL) return FASTEQ_UNSUPPORTED;
  const int64_t ctas = plan_ctas(entries);
  *bytes = ctas > 1 ? ctas * (experts + 1) * 4 : 0;
  return FASTEQ_OK;
}

extern "C" int fasteq_expert_plan(const void* expert, int32_t index_bytes, int64_t entries, int32_t experts, int32_t* position, int32_t* offsets,
                                  void* scratch, fasteq_stream_t stream) {
  int64_t need = 0;
  if (!offsets || (entries > 0 && (!expert || !position)) || (index_bytes != 4 && index_bytes != 8)) return FASTEQ_INVALID;
  if (const int rc = fasteq_expert_plan_scratch(entries, experts, &need)) return rc;
  if (need > 0 && !scratch) return FASTEQ_INVALID;
  return index_bytes == 4 ? launch_plan<int>(expert, entries, experts, position, offsets, scratch, (cudaStream_t)stream)
                          : launch_plan<long long>(expert, entries, experts, position, offsets, scratch, (cudaStream_t)stream);
}

extern "C" int fasteq_expert_gather(int32_t dtype, const void* x, const int32_t* position, const int32_t* offsets, int32_t experts, int64_t tokens,
                                    int32_t slots, int32_t width, void* rows, fasteq_stream_t stream) {
  if (!sizes_ok(dtype, tokens, slots, experts, width)) return FASTEQ_INVALID;
  if (tokens == 0 || width == 0) return FASTEQ_OK;
  if (!x || !position || !offsets || !rows) return FASTEQ_INVALID;
  cudaStream_t s = (cudaStream_t)stream;
  const bool wide = aligned16(x, rows);
  if (dtype == FASTEQ_F32) return wide && width % 4 == 0 ? gather<float, 4>(x, position, offsets, experts, tokens, slots, width, rows, s)
                                                         : gather<float, 1>(x, position, offsets, experts, tokens, slots, width, rows, s);
  return wide && width % 2 == 0 ? gather<double, 2>(x, position, offsets, experts, tokens, slots, width, rows, s)
                                : gather<double, 1>(x, position, offsets, experts, tokens, slots, width, rows, s);
}

extern "C" int fasteq_expert_combine(int32_t dtype, const void* rows, const void* weight, const int32_t* position, const int32_t* offsets,
                                     int32_t experts, int64_t tokens, int32_t slots, int32_t width, void* y, fasteq_stream_t stream) {
  if (!sizes_ok(dtype, tokens, slots, experts, width)) return FASTEQ_INVALID;
  if (tokens == 0 || width == 0) return FASTEQ_OK;
  if (!rows || !position || !offsets || !y) return FASTEQ_INVALID;
  cudaStream_t s = (cudaStream_t)stream;
  const bool wide = aligned16(rows, y);
  if (dtype == FASTEQ_F32) return wide && width % 4 == 0 ? combine<float, 4>(rows, weight, position, offsets, experts, tokens, slots, width, y, s)
                                                         : combine<float, 1>(rows, weight, position, offsets, experts, tokens, slots, width, y, s);
  return wide && width % 2 == 0 ? combine<double, 2>(rows, weight, position, offsets, experts, tokens, slots, width, y, s)
                                : combine<double, 1>(rows, weight, position, offsets, experts, tokens, slots, width, y, s);
}

extern "C" int fasteq_expert_combine_backward(int32_t dtype, const void* rows, const void* weight, const void* grad_y, const int32_t* position,
                                              const int32_t* offsets, int32_t experts, int64_t tokens, int32_t slots, int32_t width, void* grad_rows,
                                              void* grad_weight, fasteq_stream_t stream) {
  if (!sizes_ok(dtype, tokens, slots, experts, width)) return FASTEQ_INVALID;
  if (tokens == 0 || (!grad_rows && !grad_weight)) return FASTEQ_OK;
  if ((grad_rows && !weight) || !position || !offsets || (width > 0 && (!rows || !grad_y))) return FASTEQ_INVALID;
  cudaStream_t s = (cudaStream_t)stream;
  const bool wide = aligned16(rows, grad_y, grad_rows);
  if (dtype == FASTEQ_F32)
    return wide && width % 4 == 0 ? combine_backward<float, 4>(rows, weight, grad_y, position, offsets, experts, tokens, slots, width, grad_rows, grad_weight, s)
                                  : combine_backward<float, 1>(rows, weight, grad_y, position, offsets, experts, tokens, slots, width, grad_rows, grad_weight, s);
  return wide && width % 2 == 0 ? combine_backward<double, 2>(rows, weight, grad_y, position, offsets, experts, tokens, slots, width, grad_rows, grad_weight, s)
                                : combine_backward<double, 1>(rows, weight, grad_y, position, offsets, experts, tokens, slots, width, grad_rows, grad_weight, s);
}

extern "C" int fasteq_expert_device_status(int32_t* code) {
  if (!code) return FASTEQ_INVALID;
  int v = 0;
  const int zero = 0;
  cudaError_t e = cudaDeviceSynchronize();      // the copy would not wait for streams that do not wait for the default one
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&v, g_expert_status, sizeof(int));
  if (e == cudaSuccess && v != 0) e = cudaMemcpyToSymbol(g_expert_status, &zero, sizeof(int));
  if (e != cudaSuccess) return cuda_fail(e);
  *code = v;
  return FASTEQ_OK;
}
