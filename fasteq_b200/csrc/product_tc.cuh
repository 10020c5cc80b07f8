// FP32 product of a dense layer on the tensor cores, one matrix for all rows or one per expert:
//   C[r, n] = epilogue(sum_k A[r, k] (slope[r, k]) B[e(r)][k, n]),   B = W^T (forward) or W (grad_x)
//
// Each FP32 operand v is three bf16 parts v = v1 + v2 + v3 (exact: 8 + 8 + 8 significand bits, see wgrad_bf16x6.cuh for the range), and
// v1 w1 + (v1 w2 + v2 w1) + (v1 w3 + v2 w2 + v3 w1) leaves out terms of 2^-27 v w.  The weights' parts of a 32-wide k-block lie stacked in
// shared memory, [w1; w2; w3] = 192 rows of 64 columns' tiles, so that a K = 16 step is three MMAs, v1 x 192, v2 x 128, v3 x 64, which leave
// the three magnitudes in accumulators of their own: only the first is as large as the result, and the tensor core's truncating
// additions cost it one rounding toward zero per 16 products.
//
// A persistent CTA per SM walks a share of the units (expert, 64 columns, 128 rows), rows innermost: the split weights stay in shared memory
// as long as expert and columns do (k up to 32 x SLOTS).  Beyond that a kernel before this one splits the weights, and their blocks go through
// the slots as a ring, a bulk copy each.
//   warp 0       brings A's raw k-blocks to shared memory: TMA where K and the address allow it, else copies of four bytes (cp.async)
//   warp 1       issues the MMAs
//   warps 2-3    load, split and store the weights' k-blocks, or bring the split ones
//   warps 4-11   split raw blocks into tensor memory (thread = row = TMEM lane), four warps the even and four the odd ones
//   warps 12-19  split the first weights, then add the three accumulators, turn the tile in shared memory, and write it with bias, activation and
//                residual
// Every 256 of k the accumulators are emptied (into C, for the sum to go on from there): see GAIN.
// All waits are bounded; sums that are not finite (operands that are not, or beyond the split's range) are formed again in FP32.
#pragma once
#include "product.cuh"
#include "tcgen05_util.cuh"
#include "wgrad_bf16x6.cuh"

namespace fasteq {
namespace ptc {

using namespace tc;
using product::Groups;

constexpr int BM = 128, BN = 64, KB = 32, NT = 640;
constexpr int SEG = 256 / KB;              // k-blocks of an accumulation
constexpr int A_BYTES = BM * KB * 4, B_PART = BN * KB * 2, B_BYTES = 3 * B_PART;
constexpr uint32_t ACC_COLS = 3 * BN, A_COL0 = 2 * ACC_COLS, A_COLS = 3 * KB / 2;
// What a K = 16 step's truncation costs on average, of the sum: measured 0.18 to 0.21 x 2^-24 with operands of both signs, 0.27 to 0.40 with those of
// one.  Given back with the small parts.  Errors (2-norm, 1e-8; torch's FP32 products, this without the gain, this) at k = 64, 128, 256: both signs
// 14.5, 7.1, 5.1; 20.3, 12.1, 7.9; 28.8, 22.9, 14.4; one sign 12.2, 9.1, 5.0; 17.5, 17.9, 8.6; 24.7, 38.8, 15.3.
constexpr float GAIN = 0.27f / 16777216.f;

template <bool SLOPE> struct Cfg {
  static constexpr int STAGES = SLOPE ? 3 : 4, STAGE_BYTES = SLOPE ? 2 * A_BYTES : A_BYTES;
  static constexpr int SLOTS = SLOPE ? 7 : 10, SLABS = 8 * 4096;
  static constexpr int BARRIERS = 2 * STAGES + 2 * 2 + 2 * SLOTS + 2 * 2;
  static constexpr int FIXED = 1024 + SLOTS * B_BYTES + STAGES * STAGE_BYTES + SLABS + BARRIERS * 8 + 16;
  static constexpr int smem(int experts) { return FIXED + (experts + 1) * 4; }
  static_assert(FIXED + 1025 * 4 <= 227 * 1024, "shared memory of one CTA");
};

__device__ __forceinline__ void cp_async_4(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(there ? 4 : 0) : "memory");
}
// one arrival on the barrier once the thread's copies so far have landed
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void mbar_arrive_n(uint64_t* bar, uint32_t n) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// A CTA's walk over its units.  tiles: exclusive prefix sums of the experts' row tiles, [experts + 1].
struct Walk {
  const int* tiles;
  int experts, n_tiles;
  int e, n, m, mt;
  __device__ __forceinline__ Walk(const int* t, int x, int nt, int unit) : tiles(t), experts(x), n_tiles(nt) {
    int lo = 0, hi = x - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (tiles[mid + 1] * n_tiles > unit) hi = mid; else lo = mid + 1;
    }
    e = lo;
    mt = tiles[e + 1] - tiles[e];
    const int rest = unit - tiles[e] * n_tiles;
    n = mt ? rest / mt : 0;
    m = rest - n * mt;
  }
  __device__ __forceinline__ void next() {
    if (++m < mt) return;
    m = 0;
    if (++n < n_tiles) return;
    n = 0;
    do ++e; while (e < experts && tiles[e + 1] == tiles[e]);
    mt = e < experts ? tiles[e + 1] - tiles[e] : 0;
  }
  __device__ __forceinline__ bool run_begins(bool first) const { return first || m == 0; }
  __device__ __forceinline__ bool run_ends(bool last) const { return last || m + 1 == mt; }
};

__device__ __forceinline__ void tmem_ld_16_begin(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
// waits for the loads begun before; names their registers, so that no use of them moves ahead of it
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]),
                 "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])::"memory");
}

// Values of a 64-column k-block of the weights for THREADS threads: forward, rows n = t / 8 + (THREADS / 8) i of W, four k from 4 (t % 8);
// grad_x, column n = t % 64 of W, PER k from PER (t / 64)
template <bool FORWARD, int THREADS>
__device__ __forceinline__ void load_weights(const float* W, int n0, int N, int K, int kb, int t, bool wide, float (&v)[2048 / THREADS]) {
  if (FORWARD) {
    const int k = kb * KB + (t & 7) * 4;
#pragma unroll
    for (int i = 0; i < 512 / THREADS; ++i) {
      const int n = n0 + (t >> 3) + (THREADS / 8) * i;
      const float* src = W + (size_t)n * K + k;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (n < N) {
        if (wide) { if (k < K) x = *reinterpret_cast<const float4*>(src); }
        else {
          if (k < K) x.x = src[0];
          if (k + 1 < K) x.y = src[1];
          if (k + 2 < K) x.z = src[2];
          if (k + 3 < K) x.w = src[3];
        }
      }
      v[4 * i] = x.x; v[4 * i + 1] = x.y; v[4 * i + 2] = x.z; v[4 * i + 3] = x.w;
    }
  } else {
    constexpr int PER = 2048 / THREADS;
    const int n = n0 + (t & 63), k = kb * KB + (t >> 6) * PER;
#pragma unroll
    for (int i = 0; i < PER; ++i) v[i] = n < N && k + i < K ? W[(size_t)(k + i) * N + n] : 0.f;
  }
}
// their parts at `st`: row n of a part 64 bytes, 16-byte chunk j at chunk position j ^ ((n >> 1) & 3)
template <bool FORWARD, int THREADS> __device__ __forceinline__ void store_weights(unsigned char* st, int t, const float (&v)[2048 / THREADS]) {
  if (FORWARD) {
#pragma unroll
    for (int i = 0; i < 512 / THREADS; ++i) {
      const int n = (t >> 3) + (THREADS / 8) * i, at = n * 64 + ((((t & 7) >> 1) ^ ((n >> 1) & 3)) << 4) + (t & 1) * 8;
      uint2 q[3];
      wg::split_pair(make_float2(v[4 * i], v[4 * i + 1]), q[0].x, q[1].x, q[2].x);
      wg::split_pair(make_float2(v[4 * i + 2], v[4 * i + 3]), q[0].y, q[1].y, q[2].y);
#pragma unroll
      for (int e = 0; e < 3; ++e) *reinterpret_cast<uint2*>(st + e * B_PART + at) = q[e];
    }
  } else {
    constexpr int CHUNKS = 256 / THREADS;
    const int n = t & 63;
#pragma unroll
    for (int h = 0; h < CHUNKS; ++h) {
      uint32_t q[3][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) wg::split_pair(make_float2(v[8 * h + 2 * j], v[8 * h + 2 * j + 1]), q[0][j], q[1][j], q[2][j]);
      const int at = n * 64 + ((((t >> 6) * CHUNKS + h) ^ ((n >> 1) & 3)) << 4);
#pragma unroll
      for (int e = 0; e < 3; ++e) *reinterpret_cast<uint4*>(st + e * B_PART + at) = make_uint4(q[e][0], q[e][1], q[e][2], q[e][3]);
    }
  }
}

// All weights split beforehand, [expert][64 columns][k-block] as they lie in shared memory: a block of 256 threads each
template <bool FORWARD> __global__ void __launch_bounds__(256) split_weights_kernel(const float* W, unsigned char* out, int N, int K, int n_tiles, int n_kb, bool wide) {
  wait_for_previous_kernel();
  const int kb = blockIdx.x % n_kb, rest = blockIdx.x / n_kb, n = rest % n_tiles, e = rest / n_tiles;
  float v[8];
  load_weights<FORWARD, 256>(W + (size_t)e * N * K, n * BN, N, K, kb, threadIdx.x, wide, v);
  store_weights<FORWARD, 256>(out + (size_t)blockIdx.x * B_BYTES, threadIdx.x, v);
}

// sum_k a[k] (d[k]) b[k * stride] with FP32's own products
__device__ __noinline__ float sum_fp32(const float* a, const float* d, const float* b, int K, int stride) {
  float v = 0.f;
#pragma unroll 1
  for (int k = 0; k < K; ++k) v = fmaf(d ? a[k] * d[k] : a[k], b[(size_t)k * stride], v);
  return v;
}

template <int ACT> __device__ __noinline__ void wild(float4& v, float4& d) {
  v.x = product::activate<ACT>(v.x, d.x); v.y = product::activate<ACT>(v.y, d.y);
  v.z = product::activate<ACT>(v.z, d.z); v.w = product::activate<ACT>(v.w, d.w);
}

struct Args {
  Groups groups;
  const float *A, *slope, *W, *bias, *residual;
  const unsigned char* split;         // the weights' blocks where they do not stay in shared memory
  float *C, *slope_out;
  int K, N;
  bool a_wide, w_wide, c_wide;        // 16-byte accesses of A (and slope), of W, of everything shaped like C (and bias)
  int* status;
};

template <bool FORWARD, bool SLOPE, int ACT>
__global__ void __launch_bounds__(NT, 1) product_tc_kernel(const __grid_constant__ Args p, const __grid_constant__ CUtensorMap tmA,
                                                           const __grid_constant__ CUtensorMap tmSlope) {
  using C_ = Cfg<SLOPE>;
  constexpr int STAGES = C_::STAGES, SLOTS = C_::SLOTS;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* a_raw = smem + SLOTS * B_BYTES;
  unsigned char* slabs = a_raw + STAGES * C_::STAGE_BYTES;
  uint64_t* a_full = reinterpret_cast<uint64_t*>(slabs + C_::SLABS);     // [STAGES] a raw k-block has landed
  uint64_t* a_empty = a_full + STAGES;                                   // [STAGES] it has been split
  uint64_t* s_full = a_empty + STAGES;                                   // [2] its parts are in tensor memory
  uint64_t* s_empty = s_full + 2;                                        // [2] the MMAs have read them
  uint64_t* b_full = s_empty + 2;                                        // [SLOTS]
  uint64_t* b_empty = b_full + SLOTS;                                    // [SLOTS]
  uint64_t* acc_full = b_empty + SLOTS;                                  // [2]
  uint64_t* acc_empty = acc_full + 2;                                    // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  int* tiles = reinterpret_cast<int*>(tmem_slot + 4);                    // [experts + 1]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, K = p.K, N = p.N, X = p.groups.experts;
  int* status = p.status;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(&a_full[s], p.a_wide ? 1 : 32); mbar_init(&a_empty[s], 4); }
    for (int s = 0; s < SLOTS; ++s) { mbar_init(&b_full[s], p.split ? 1 : 8); mbar_init(&b_empty[s], 1); }
    for (int s = 0; s < 2; ++s) { mbar_init(&s_full[s], 4); mbar_init(&s_empty[s], 1); mbar_init(&acc_full[s], 1); mbar_init(&acc_empty[s], 8); }
    mbar_fence_init();
  }
  if (warp == 1) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  wait_for_previous_kernel();
  for (int e = threadIdx.x; e < X; e += NT) tiles[e] = (int)((p.groups.first(e + 1) - p.groups.first(e) + BM - 1) / BM);
  __syncthreads();
  if (warp == 0) {
    int total = 0;
    for (int e0 = 0; e0 < X; e0 += 32) {
      const int v = e0 + lane < X ? tiles[e0 + lane] : 0;
      int sum = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += u;
      }
      if (e0 + lane < X) tiles[e0 + lane] = total + sum - v;
      total += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (lane == 0) tiles[X] = total;
  }
  __syncthreads();
  const uint32_t tmem = *tmem_slot;
  const int n_tiles = (N + BN - 1) / BN, n_kb = (K + KB - 1) / KB;
  const bool resident = p.split == nullptr;        // n_kb <= SLOTS then
  const long long units = (long long)tiles[X] * n_tiles;
  const int u0 = (int)(units * blockIdx.x / gridDim.x), u1 = (int)(units * (blockIdx.x + 1) / gridDim.x);

  if (u0 < u1) {
    Walk w(tiles, X, n_tiles, u0);
    if (warp == 0) {
      // ------------------------------------------------------------------ raw k-blocks of A
      // row r of a block: 128 bytes, 16-byte chunk j at chunk position j ^ (r & 7).  TMA brings the rows behind the expert's last too: their
      // results are not written
      int it = 0;
      for (int u = u0; u < u1; ++u, w.next()) {
        const long long begin = p.groups.first(w.e), left = p.groups.first(w.e + 1) - begin - (long long)w.m * BM;
        const long long row0 = begin + (long long)w.m * BM;
        for (int kb = 0; kb < n_kb; ++kb, ++it) {
          const int s = it % STAGES;
          unsigned char* st = a_raw + (size_t)s * C_::STAGE_BYTES;
          mbar_wait(&a_empty[s], ((it / STAGES) & 1u) ^ 1u, status);
          if (p.a_wide) {
            if (lane == 0) {
              mbar_arrive_expect_tx(&a_full[s], (uint32_t)C_::STAGE_BYTES);
              tma_load_3d(st, &tmA, kb * KB, 0, (int)row0, &a_full[s]);
              if (SLOPE) tma_load_3d(st + A_BYTES, &tmSlope, kb * KB, 0, (int)row0, &a_full[s]);
            }
            __syncwarp();
          } else {
            const int rows = left < BM ? (int)left : BM, k = kb * KB + lane;
#pragma unroll
            for (int side = 0; side < (SLOPE ? 2 : 1); ++side) {
              const float* src = side ? p.slope : p.A;
              const float* a = src + (size_t)row0 * K + k;
              const uint32_t d = smem_u32(st) + side * A_BYTES + (lane & 3) * 4;
#pragma unroll 8
              for (int r = 0; r < BM; ++r) {
                const bool there = r < rows && k < K;
                cp_async_4(d + r * 128 + (((lane >> 2) ^ (r & 7)) << 4), there ? a + (size_t)r * K : src, there);
              }
            }
            cp_async_arrive(&a_full[s]);
          }
        }
      }
      cp_async_wait_all();
    } else if (warp == 1) {
      // ------------------------------------------------------------------ MMAs (whole warp, one elected lane)
      const uint32_t idesc1 = wg::idesc_bf16_m128(3 * BN), idesc2 = wg::idesc_bf16_m128(2 * BN), idesc3 = wg::idesc_bf16_m128(BN);
      const uint32_t tm = uniform(tmem);
      const uint64_t desc0 = wg::desc_sw64(uniform(smem_u32(smem)));
      int it = 0, lt = 0, run = 0;         // lt: accumulations, run: number of the run's first block
      for (int u = u0; u < u1; ++u) {
        const bool ends = !resident || uniform((uint32_t)w.run_ends(u + 1 == u1));
        for (int k0 = 0; k0 < n_kb; k0 += SEG, ++lt) {
          const int buf = lt & 1, k1 = min(n_kb, k0 + SEG);
          mbar_wait(&acc_empty[buf], ((lt >> 1) & 1u) ^ 1u, status);
          const uint32_t d = tm + (uint32_t)buf * ACC_COLS;
          for (int kb = k0; kb < k1; ++kb, ++it) {
            const int fill = run + kb, bs = fill % SLOTS, slot = it & 1;
            mbar_wait(&b_full[bs], (fill / SLOTS) & 1u, status);
            mbar_wait(&s_full[slot], (it >> 1) & 1u, status);
            __syncwarp();
            tc_fence_after();
            const uint32_t a = tm + A_COL0 + (uint32_t)(slot * A_COLS);
            const uint64_t b = desc_at(desc0, (uint32_t)(bs * B_BYTES));
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
              const uint64_t bk = desc_at(b, (uint32_t)(ks * 32));
              warp_mma_bf16_a_tmem(d, a + (uint32_t)(ks * 8), bk, idesc1, kb > k0 || ks ? 1u : 0u);
              warp_mma_bf16_a_tmem(d + BN, a + (uint32_t)(KB / 2 + ks * 8), bk, idesc2, 1u);
              warp_mma_bf16_a_tmem(d + 2 * BN, a + (uint32_t)(KB + ks * 8), bk, idesc3, 1u);
            }
            warp_mma_commit(&s_empty[slot]);
            if (ends) warp_mma_commit(&b_empty[bs]);
          }
          warp_mma_commit(&acc_full[buf]);
        }
        if (ends) run += n_kb;
        w.next();
      }
    } else if (warp < 4) {
      // ------------------------------------------------------------------ the weights' parts
      const int t = threadIdx.x - 64;
      int fill = 0;
      for (int u = u0; u < u1; ++u, w.next()) {
        if (!resident) {
          if (t == 0) {
            const unsigned char* src = p.split + ((size_t)w.e * n_tiles + w.n) * n_kb * B_BYTES;
            for (int kb = 0; kb < n_kb; ++kb, ++fill) {
              const int slot = fill % SLOTS;
              mbar_wait(&b_empty[slot], ((fill / SLOTS) & 1u) ^ 1u, status);
              mbar_arrive_expect_tx(&b_full[slot], (uint32_t)B_BYTES);
              bulk_g2s(smem + (size_t)slot * B_BYTES, src + (size_t)kb * B_BYTES, (uint32_t)B_BYTES, &b_full[slot]);
            }
          }
          continue;
        }
        if (u == u0) fill += n_kb;                 // the first ones are split by the epilogue's warps
        if (u == u0 || !w.run_begins(false)) continue;
        const float* W = p.W + (size_t)w.e * N * K;
        float v[32], ahead[32];
        load_weights<FORWARD, 64>(W, w.n * BN, N, K, 0, t, p.w_wide, v);
        for (int kb = 0; kb < n_kb; ++kb, ++fill) {
          if (kb + 1 < n_kb) load_weights<FORWARD, 64>(W, w.n * BN, N, K, kb + 1, t, p.w_wide, ahead);
          const int slot = fill % SLOTS;
          mbar_wait(&b_empty[slot], ((fill / SLOTS) & 1u) ^ 1u, status);
          store_weights<FORWARD, 64>(smem + (size_t)slot * B_BYTES, t, v);
          fence_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive_n(&b_full[slot], 4);
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = ahead[i];
        }
      }
    } else if (warp < 12) {
      // ------------------------------------------------------------------ split A into tensor memory
      const int row = (warp & 3) * 32 + lane, slot = (warp - 4) >> 2;
      const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16) + A_COL0 + (uint32_t)(slot * A_COLS);
      const int total = (u1 - u0) * n_kb;
      for (int it = slot; it < total; it += 2) {
        const int s = it % STAGES;
        // The slot first: with block it - 2 multiplied, the other warps have passed the stage's last phase (it - STAGES), and its parity
        // cannot be taken for this block's.
        mbar_wait(&s_empty[slot], ((it >> 1) & 1u) ^ 1u, status);
        mbar_wait(&a_full[s], (it / STAGES) & 1u, status);
        __syncwarp();
        tc_fence_after();
        const unsigned char* st = a_raw + (size_t)s * C_::STAGE_BYTES + row * 128;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          uint32_t q[3][8];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int at = ((ks * 4 + j) ^ (row & 7)) << 4;
            float4 v = *reinterpret_cast<const float4*>(st + at);
            if (SLOPE) {
              const float4 d = *reinterpret_cast<const float4*>(st + A_BYTES + at);
              v.x *= d.x; v.y *= d.y; v.z *= d.z; v.w *= d.w;
            }
            wg::split_pair(make_float2(v.x, v.y), q[0][2 * j], q[1][2 * j], q[2][2 * j]);
            wg::split_pair(make_float2(v.z, v.w), q[0][2 * j + 1], q[1][2 * j + 1], q[2][2 * j + 1]);
          }
#pragma unroll
          for (int e = 0; e < 3; ++e) wg::tmem_st_8(lanes + (uint32_t)(e * (KB / 2) + ks * 8), q[e]);
        }
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        tc_fence_before();
        fence_async_smem();                 // the reads precede the TMA write that refills the stage
        __syncwarp();
        if (lane == 0) { mbar_arrive(&s_full[slot]); mbar_arrive(&a_empty[s]); }
      }
    } else {
      // ------------------------------------------------------------------ epilogue: 32 rows and 32 columns to a warp
      if (resident) {
        const int t = threadIdx.x - 384;
        const float* W = p.W + (size_t)w.e * N * K;
        for (int k0 = 0; k0 < n_kb; k0 += 4) {
          float v[4][8];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (k0 + i < n_kb) load_weights<FORWARD, 256>(W, w.n * BN, N, K, k0 + i, t, p.w_wide, v[i]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (k0 + i >= n_kb) break;
            store_weights<FORWARD, 256>(smem + (size_t)(k0 + i) * B_BYTES, t, v[i]);
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&b_full[k0 + i]);
          }
        }
      }
      const int quarter = warp & 3, half = (warp - 12) >> 2;
      unsigned char* slab = slabs + (size_t)(warp - 12) * 4096;      // 16-byte chunk j of row r at j ^ (r & 7)
      const uint32_t cols = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(half * 32);
      int lt = 0;
      for (int u = u0; u < u1; ++u, w.next()) {
        const int nh = w.n * BN + half * 32;
        const long long begin = p.groups.first(w.e), left = p.groups.first(w.e + 1) - begin - (long long)w.m * BM;
        const int rows = (int)(left < BM ? left : BM) - quarter * 32;      // of this warp
        const size_t row0 = (size_t)(begin + (long long)w.m * BM + quarter * 32);
        // wide: four columns, eight rows a thread; else one column, all rows
        const int c = p.c_wide ? (lane & 7) * 4 : lane, n = nh + c;
        const bool column = n < N;
        float4 bias = make_float4(0.f, 0.f, 0.f, 0.f);
        if (FORWARD && p.bias && column) {
          const float* b = p.bias + (size_t)w.e * N + n;
          if (p.c_wide) bias = *reinterpret_cast<const float4*>(b); else bias.x = *b;
        }
        for (int k0 = 0; k0 < n_kb; k0 += SEG, ++lt) {
          const int buf = lt & 1;
          const bool last = k0 + SEG >= n_kb;
          const float gain = GAIN * (float)((min(K, (k0 + SEG) * KB) - k0 * KB + 15) / 16);
          mbar_wait(&acc_full[buf], (lt >> 1) & 1u, status);
          __syncwarp();
          tc_fence_after();
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t x[16], y[16], z[16];
            const uint32_t at = cols + (uint32_t)buf * ACC_COLS + (uint32_t)(h * 16);
            tmem_ld_16_begin(at, x);
            tmem_ld_16_begin(at + BN, y);
            tmem_ld_16_begin(at + 2 * BN, z);
            tmem_ld_wait(x);
            tmem_ld_wait(y);
            tmem_ld_wait(z);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              float2 o[2];
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const int q = 4 * j + 2 * i;
                auto two = [&](const uint32_t (&r)[16]) { return make_float2(__uint_as_float(r[q]), __uint_as_float(r[q + 1])); };
                o[i] = vmul(vadd(two(x), vfma(two(x), make_float2(gain, gain), vadd(two(y), two(z)))), make_float2(wg::UNSCALE, wg::UNSCALE));
              }
              *reinterpret_cast<float4*>(slab + lane * 128 + (((h * 4 + j) ^ (lane & 7)) << 4)) = make_float4(o[0].x, o[0].y, o[1].x, o[1].y);
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&acc_empty[buf]);
          // a sum that is not finite, again in FP32
          auto again = [&](float v, int r, int m) {
            if (fabsf(v) <= 3.402823466e38f) return v;
            return sum_fp32(p.A + (row0 + r) * K, SLOPE ? p.slope + (row0 + r) * K : nullptr,
                            p.W + (size_t)w.e * N * K + (FORWARD ? (size_t)m * K : (size_t)m), K, FORWARD ? 1 : N);
          };
          if (column && p.c_wide) {
            const float* from = reinterpret_cast<const float*>(slab + (lane >> 3) * 128);
#pragma unroll 4
            for (int i = 0; i < 8; ++i) {
              const int r = (lane >> 3) + i * 4;
              if (r >= rows) break;
              const size_t o = (row0 + r) * N + n;
              float4 v = *reinterpret_cast<const float4*>(from + i * 128 + (((lane & 7) ^ (r & 7)) << 2));
              if (k0 > 0) {
                const float4 before = *reinterpret_cast<const float4*>(p.C + o);
                v.x += before.x; v.y += before.y; v.z += before.z; v.w += before.w;
              }
              if (last) {
                const float2 z0 = make_float2(v.x + bias.x, v.y + bias.y), z1 = make_float2(v.z + bias.z, v.w + bias.w);
                float4 d;
                // larger than kTame, infinite or not a number: in magnitude bits
                auto bits = [](float x) { return __float_as_uint(x) & 0x7fffffffu; };
                constexpr float most = ACT == product::kIdentity || ACT == product::kAbs ? 3.402823466e38f : product::kTame;
                if (max(max(bits(z0.x), bits(z0.y)), max(bits(z1.x), bits(z1.y))) <= __float_as_uint(most)) {
                  float2 d0, d1;
                  const float2 y0 = FORWARD ? product::activate_tame<ACT>(z0, p.slope_out != nullptr, d0) : z0;
                  const float2 y1 = FORWARD ? product::activate_tame<ACT>(z1, p.slope_out != nullptr, d1) : z1;
                  v = make_float4(y0.x, y0.y, y1.x, y1.y);
                  d = make_float4(d0.x, d0.y, d1.x, d1.y);
                } else {
                  v.x = again(v.x, r, n) + bias.x; v.y = again(v.y, r, n + 1) + bias.y; v.z = again(v.z, r, n + 2) + bias.z; v.w = again(v.w, r, n + 3) + bias.w;
                  if (FORWARD) wild<ACT>(v, d);
                }
                if (FORWARD && p.residual) {
                  const float4 res = *reinterpret_cast<const float4*>(p.residual + o);
                  v.x += res.x; v.y += res.y; v.z += res.z; v.w += res.w;
                }
                if (FORWARD && p.slope_out) *reinterpret_cast<float4*>(p.slope_out + o) = d;
              }
              *reinterpret_cast<float4*>(p.C + o) = v;
            }
          } else if (column) {
#pragma unroll 4
            for (int r = 0; r < 32; ++r) {
              if (r >= rows) break;
              const size_t o = (row0 + r) * N + n;
              float d, v = *reinterpret_cast<const float*>(slab + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4);
              if (k0 > 0) v += p.C[o];
              if (last) {
                const float res = FORWARD && p.residual ? p.residual[o] : 0.f;
                v = again(v, r, n);
                if (FORWARD) {
                  v = product::activate<ACT>(v + bias.x, d) + res;
                  if (p.slope_out) p.slope_out[o] = d;
                }
              }
              p.C[o] = v;
            }
          }
          __syncwarp();
        }
      }
    }
  }
  // rows of no expert
  if (p.groups.offsets) {
    const size_t first = (size_t)p.groups.first(X) * N, end = (size_t)p.groups.rows * N;
    for (size_t i = first + (size_t)blockIdx.x * NT + threadIdx.x; i < end; i += (size_t)gridDim.x * NT) {
      p.C[i] = 0.f;
      if (FORWARD && p.slope_out) p.slope_out[i] = 0.f;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) { tc_fence_after(); tmem_dealloc(tmem, 512); }
}

}  // namespace ptc
}  // namespace fasteq
