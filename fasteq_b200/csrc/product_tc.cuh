// FP32 product of a dense layer on the tensor cores, one matrix for all rows or one per expert:
//   C[r, n] = epilogue(sum_k A[r, k] (slope[r, k]) B[e(r)][k, n]),   B = W^T (forward) or W (grad_x)
//
// Each FP32 operand v is three bf16 parts v = v1 + v2 + v3 (exact: 8 + 8 + 8 significand bits, see wgrad_bf16x6.cuh for the range), and
// v1 w1 + (v1 w2 + v2 w1 + v1 w3 + v2 w2 + v3 w1) leaves out terms of 2^-27 v w.  The weights' parts of a 32-wide k-block lie stacked in
// shared memory, [w1; w2; w3], so that a K = 16 step is five MMAs, v1 x [w1; w2] and four of 64 columns.  The first product has an
// accumulator of its own and the small ones another: only the first is as large as the result, and the tensor core's truncating additions
// cost it one rounding toward zero per 16 products.
//
// A persistent CTA per SM takes 64 columns and walks a share of the row tiles (128 rows of an expert): the split weights stay in shared memory
// as long as the expert does (k up to 32 x slots).  Beyond that a kernel before this one splits the weights, and their blocks go through
// the slots as a ring, a bulk copy each.
//   warp 0       brings A's raw k-blocks to shared memory (TMA; rows that are not 16-byte aligned a kernel before this one copies apart)
//   warp 1       issues the MMAs
//   warps 2-3    load, split and store the weights' k-blocks, or bring the split ones
//   warps 4-11   split raw blocks into tensor memory (thread = row = TMEM lane), four warps the even and four the odd ones
//   warps 12-19  split the first weights, then add the two accumulators, bias, activation and residual, and store tiles of 32 x 32 by TMA
// Every 256 of k the accumulators are emptied (into the slabs, for the sum to go on from there), which bounds what the truncations add up to.  Nothing is given
// back for them: that would move sums that lose nothing (one-hot rows, whole numbers), which come out exact so.  Errors against 64 bits (2-norm, 1e-8;
// torch's FP32 products, this) at k = 64, 256, 1,664: operands of both signs 14.4, 7.0; 28.6, 23.1; 73.2, 23.1; of one sign, where truncations do not cancel,
// 12.2, 9.0; 24.7, 38.7; 56.1, 36.5.
// All waits are bounded; sums that are not finite (operands that are not, or beyond the split's range) are formed again in FP32, the 32 columns of
// such a row that a warp holds.
//
// Why so: 2 x 128 columns of accumulators and 4 x 48 of A's parts fill 448 of the 512 columns of tensor memory, eight blocks of the weights (k = 256), four
// raw ones of A and the slabs 227 KB of shared memory.  The six products' rate is the bf16 one / 6 (271 TFLOP/s of 1627), a K = 16 step takes 25 + 0.44
// columns clocks an MMA, 294 for the five.  Measured: 100,000 rows of 256 to 256 channels 99 us (132 TFLOP/s of FP32-accurate products; the ten MMAs
// are 588 of a block's 1,050 clocks, a wait of their warp 240 while some are queued), 24,576 of 128 to 256 21 us, 644,000 of 64 to 64 with SiLU 78 us (330 MB,
// 4.2 TB/s: the epilogue warps' latency, 4,300 clocks a tile, while the split warps idle), 192 of 128 to 128 8 us (one tile's chain).  Two tiles side by side with an issuing warp each instead: 90, 21.6,
// 77 and 8.4 us, taken back; 16 warps of the epilogue spill at 72 registers.
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
constexpr uint32_t ACC_COLS = 2 * BN, A_COL0 = 2 * ACC_COLS, A_COLS = 3 * KB / 2;
constexpr int A_SLOTS = 4;                 // of tensor memory: 2 x 128 columns of accumulators, 4 x 48 of A's parts
template <bool SLOPE> struct Cfg {
  // Even: a stage then always belongs to the same set of split warps, which sees each of its phases (a set that saw every other one could take
  // the parity of a phase long past for its own).
  static constexpr int STAGES = SLOPE ? 2 : 4, STAGE_BYTES = SLOPE ? 2 * A_BYTES : A_BYTES;
  static constexpr int SLABS = SLOPE ? 8 * 4096 : 8 * 8192;       // forward: values and slopes
  static constexpr int MOST_SLOTS = 16;
  static constexpr int BARRIERS = 2 * STAGES + 2 * A_SLOTS + 2 * MOST_SLOTS + 2 * 2;
  static constexpr int smem(int slots, int experts) { return 1024 + slots * B_BYTES + STAGES * STAGE_BYTES + SLABS + BARRIERS * 8 + 8 * 128 + 16 + (experts + 1) * 4; }
  // as many of the weights' blocks as an SM holds: 8 forward, 10 for grad_x, one less with more than about 150 experts
  static constexpr int slots(int experts) { return (227 * 1024 - smem(0, experts)) / B_BYTES < MOST_SLOTS ? (227 * 1024 - smem(0, experts)) / B_BYTES : MOST_SLOTS; }
};

__device__ __forceinline__ void mbar_arrive_n(uint64_t* bar, uint32_t n) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(n) : "memory");
}

// A CTA's walk over its units: the row tiles [first, first + count) of all experts' for its columns n, and again for those n_step further on.
// tiles: exclusive prefix sums of the experts' row tiles, [experts + 1].
struct Walk {
  const int* tiles;
  int experts, first, count, n_step;
  int e, n, m, mt, left;
  __device__ __forceinline__ Walk(const int* t, int x, int f, int c, int n0, int step) : tiles(t), experts(x), first(f), count(c), n_step(step), n(n0) { start(); }
  __device__ __forceinline__ void start() {
    int lo = 0, hi = experts - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (tiles[mid + 1] > first) hi = mid; else lo = mid + 1;
    }
    e = lo;
    mt = tiles[e + 1] - tiles[e];
    m = first - tiles[e];
    left = count;
  }
  __device__ __forceinline__ void next() {
    if (--left == 0) {
      n += n_step;
      start();
    } else if (++m == mt) {
      m = 0;
      do ++e; while (tiles[e + 1] == tiles[e]);          // ends at a later one of the CTA's tiles
      mt = tiles[e + 1] - tiles[e];
    }
  }
  __device__ __forceinline__ bool run_begins() const { return left == count || m == 0; }
  __device__ __forceinline__ bool run_ends() const { return left == 1 || m + 1 == mt; }
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

__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, int column, int row, const void* src) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(map), "r"(column), "r"(0), "r"(row), "r"(smem_u32(src))
               : "memory");
}

// a map on its way to the cache before its first copy needs it
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }

struct Args {
  Groups groups;
  const float *A, *slope, *W, *bias, *residual;
  const unsigned char* split;         // the weights' blocks where they do not stay in shared memory
  float *C, *slope_out;
  int K, N, lda, ldd, slots;          // columns between A's rows and between slope's, slots of the weights' blocks
  bool w_wide, c_wide;                // 16-byte accesses of W, of C and the residual
  int* status;
};

// 16-byte chunk j of row r in a slab of 32 rows and 32 columns (what a TMA store with 128-byte swizzle takes)
__device__ __forceinline__ int slab_at(int r, int j) { return r * 128 + ((j ^ (r & 7)) << 4); }

// A residual of 16-byte aligned rows is brought into the slab while the sums are formed (80,533 rows of 36 to 100 channels with SiLU: 34 us, 41 us where it
// is read as the slab is stored); with several accumulations the sums so far are there, and it is added as the slab is stored.  So it is where rows are
// not aligned (33 to 99 channels: 51 us either way).
__device__ __forceinline__ bool early_residual(const Args& p) { return p.residual && p.c_wide && p.K <= SEG * KB; }
__device__ __noinline__ void fetch_slab(const float* from, size_t row0, int rows, int n0, int N, unsigned char* slab) {
  const int lane = threadIdx.x & 31, n = n0 + (lane & 7) * 4;
  if (n >= N) return;
#pragma unroll 4
  for (int r = lane >> 3; r < rows; r += 4)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(slab + slab_at(r, lane & 7))), "l"(from + (row0 + r) * N + n) : "memory");
}

// 32 columns of this thread's row again with FP32's own products, where a sum is not finite.  Apart from the kernel and with nothing handed back: values
// whose addresses a call takes would live in memory for good.
template <bool FORWARD, bool SLOPE, int ACT>
__device__ __noinline__ void wild_row(const Args& p, int e, size_t row, int n, unsigned char* slab, unsigned char* slopes) {
  const int lane = threadIdx.x & 31;
  const float *a = p.A + row * p.lda, *g = SLOPE ? p.slope + row * p.ldd : nullptr, *b = p.W + (size_t)e * p.N * p.K + (FORWARD ? (size_t)n * p.K : (size_t)n);
#pragma unroll 1
  for (int j = 0; j < 32 && n + j < p.N; ++j) {
    const int at = slab_at(lane, j >> 2) + (j & 3) * 4;
    float d = 1.f, v = 0.f;
#pragma unroll 1
    for (int k = 0; k < p.K; ++k) v = fmaf(SLOPE ? a[k] * g[k] : a[k], b[FORWARD ? (size_t)j * p.K + k : (size_t)k * p.N + j], v);
    if (FORWARD) {
      v = product::activate<ACT>(p.bias ? v + p.bias[(size_t)e * p.N + n + j] : v, d);
      if (early_residual(p)) v += p.residual[row * p.N + n + j];
      if (ACT != product::kIdentity && p.slope_out) *reinterpret_cast<float*>(slopes + at) = d;
    }
    *reinterpret_cast<float*>(slab + at) = v;
  }
}

// Activations of 16 columns of this thread's row with a |z| beyond kNear: z lies where the slopes go.  Apart from the kernel, as it hardly ever happens.
template <int ACT> __device__ __noinline__ void far_row(unsigned char* slab, unsigned char* slopes, int chunk, bool residual) {
  const int lane = threadIdx.x & 31;
#pragma unroll 1
  for (int i = 0; i < 16; ++i) {
    const int at = slab_at(lane, chunk + (i >> 2)) + (i & 3) * 4;
    float d;
    const float y = product::activate<ACT>(*reinterpret_cast<const float*>(slopes + at), d);
    *reinterpret_cast<float*>(slopes + at) = d;
    *reinterpret_cast<float*>(slab + at) = residual ? y + *reinterpret_cast<const float*>(slab + at) : y;
  }
}

// the largest magnitude of three, NaN if one is
__device__ __forceinline__ float largest(float a, float b, float c) {
  float m;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
  return m;
}

// 16 values to `dst`, of which `count` are there
__device__ __forceinline__ void store_16(float* dst, int count, bool wide, const float2 (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (wide) { if (4 * i < count) *reinterpret_cast<float4*>(dst + 4 * i) = make_float4(v[2 * i].x, v[2 * i].y, v[2 * i + 1].x, v[2 * i + 1].y); }
    else {
      if (4 * i < count) dst[4 * i] = v[2 * i].x;
      if (4 * i + 1 < count) dst[4 * i + 1] = v[2 * i].y;
      if (4 * i + 2 < count) dst[4 * i + 2] = v[2 * i + 1].x;
      if (4 * i + 3 < count) dst[4 * i + 3] = v[2 * i + 1].y;
    }
  }
}

// A slab's rows without TMA: plus a residual, where the tile ends inside the tensor (another expert's rows follow), or where rows are not 16-byte aligned.
__device__ __noinline__ void store_slab(float* C, const float* residual, size_t row0, int rows, int n0, int N, int pitch, bool wide, const unsigned char* slab) {
  const int lane = threadIdx.x & 31;
  if (wide) {
    const int n = n0 + (lane & 7) * 4;
    if (n >= N) return;
    for (int r0 = lane >> 3; r0 < rows; r0 += 16) {
      float4 more[4] = {};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (residual && r0 + 4 * i < rows) more[i] = *reinterpret_cast<const float4*>(residual + (row0 + r0 + 4 * i) * pitch + n);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (r0 + 4 * i >= rows) break;
        float4 v = *reinterpret_cast<const float4*>(slab + slab_at(r0 + 4 * i, lane & 7));
        v.x += more[i].x; v.y += more[i].y; v.z += more[i].z; v.w += more[i].w;
        *reinterpret_cast<float4*>(C + (row0 + r0 + 4 * i) * pitch + n) = v;
      }
    }
  } else {
    const int n = n0 + lane, columns = N - n0;
    if (columns < 32) {                    // a few columns of many rows, side by side in the lanes
#pragma unroll 4
      for (int i = lane; i < rows * columns; i += 32) {
        const int r = i / columns, c = i - r * columns;
        const size_t at = (row0 + r) * pitch + n0 + c;
        const float v = *reinterpret_cast<const float*>(slab + slab_at(r, c >> 2) + (c & 3) * 4);
        C[at] = residual ? v + residual[at] : v;
      }
      return;
    }
    float* to = C + row0 * pitch + n;
    const float* from = residual ? residual + row0 * pitch + n : nullptr;
#pragma unroll 1
    for (int r0 = 0; r0 < rows; r0 += 8, to += 8 * (size_t)pitch) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = from && r0 + i < rows ? from[(size_t)(r0 + i) * pitch] : 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] += *reinterpret_cast<const float*>(slab + slab_at(r0 + i, lane >> 2) + (lane & 3) * 4);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (r0 + i < rows) to[(size_t)i * pitch] = v[i];
    }
  }
}

template <bool FORWARD, bool SLOPE, int ACT>
__global__ void __launch_bounds__(NT, 1) product_tc_kernel(const __grid_constant__ Args p, const __grid_constant__ CUtensorMap tmA,
                                                           const __grid_constant__ CUtensorMap tmSlope, const __grid_constant__ CUtensorMap tmC,
                                                           const __grid_constant__ CUtensorMap tmD) {
  using C_ = Cfg<SLOPE>;
  constexpr int STAGES = C_::STAGES;
  const int slots = p.slots;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* a_raw = smem + (size_t)slots * B_BYTES;
  unsigned char* slabs = a_raw + STAGES * C_::STAGE_BYTES;
  uint64_t* a_full = reinterpret_cast<uint64_t*>(slabs + C_::SLABS);     // [STAGES] a raw k-block has landed
  uint64_t* a_empty = a_full + STAGES;                                   // [STAGES] it has been split
  uint64_t* s_full = a_empty + STAGES;                                   // [A_SLOTS] its parts are in tensor memory
  uint64_t* s_empty = s_full + A_SLOTS;                                  // [A_SLOTS] the MMAs have read them
  uint64_t* b_full = s_empty + A_SLOTS;                                        // [slots]
  uint64_t* b_empty = b_full + C_::MOST_SLOTS;                           // [slots]
  uint64_t* acc_full = b_empty + C_::MOST_SLOTS;                                  // [2]
  uint64_t* acc_empty = acc_full + 2;                                    // [2]
  float* biases = reinterpret_cast<float*>(acc_empty + 2);               // [8][32] of the epilogue's warps
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(biases + 8 * 32);
  int* tiles = reinterpret_cast<int*>(tmem_slot + 4);                    // [experts + 1]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, K = p.K, N = p.N, X = p.groups.experts;
  int* status = p.status;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(&a_full[s], 1); mbar_init(&a_empty[s], 4); }
    for (int s = 0; s < slots; ++s) { mbar_init(&b_full[s], p.split ? 1 : 8); mbar_init(&b_empty[s], 1); }
    for (int s = 0; s < A_SLOTS; ++s) { mbar_init(&s_full[s], 4); mbar_init(&s_empty[s], 1); }
    for (int s = 0; s < 2; ++s) { mbar_init(&acc_full[s], 1); mbar_init(&acc_empty[s], 8); }
    mbar_fence_init();
    tiles[0] = 0;                                  // of one matrix; experts' follow
    tiles[1] = (int)((p.groups.rows + BM - 1) / BM);
  }
  if (warp == 1) tmem_alloc(tmem_slot, 512);
  if (threadIdx.x == 64) {
    prefetch_map(&tmA);
    if (SLOPE) prefetch_map(&tmSlope);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  wait_for_previous_kernel();
  if (p.groups.offsets) {
    for (int e = threadIdx.x; e < X; e += NT) tiles[e] = (int)max((p.groups.first(e + 1) - p.groups.first(e) + BM - 1) / BM, 0LL);
    __syncthreads();
    if (warp == 0) {
      const int most = (int)(p.groups.rows / BM) + X;       // of offsets that ascend
      int total = 0;
      for (int e0 = 0; e0 < X; e0 += 32) {
        const int v = e0 + lane < X ? tiles[e0 + lane] : 0;
        int sum = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int u = __shfl_up_sync(0xffffffffu, sum, o);
          if (lane >= o) sum += u;
        }
        if (e0 + lane < X) tiles[e0 + lane] = min(total + sum - v, most);
        total = min(total + __shfl_sync(0xffffffffu, sum, 31), most);
      }
      if (lane == 0) tiles[X] = total;
    }
    __syncthreads();
  }
  const uint32_t tmem = *tmem_slot;
  const int n_tiles = (N + BN - 1) / BN, n_kb = (K + KB - 1) / KB;
  const bool resident = p.split == nullptr;        // n_kb <= slots then
  // CTAs with neighbouring columns of the same rows lie side by side and walk together, so that A comes from memory once
  const int beside = min(n_tiles, (int)gridDim.x), sets = (int)gridDim.x / beside, set_no = (int)blockIdx.x / beside, n_first = (int)blockIdx.x % beside;
  const int first = (int)((long long)tiles[X] * set_no / sets), count = set_no < sets ? (int)((long long)tiles[X] * (set_no + 1) / sets) - first : 0;
  const int units = count * ((n_tiles - n_first + beside - 1) / beside);

  if (units > 0) {
    Walk w(tiles, X, first, count, n_first, beside);
    if (warp == 0) {
      // ------------------------------------------------------------------ raw k-blocks of A
      // row r of a block: 128 bytes, 16-byte chunk j at chunk position j ^ (r & 7).  TMA brings the rows behind the expert's last too: their
      // results are not written
      int it = 0;
      for (int u = 0; u < units; ++u, w.next()) {
        const long long row0 = p.groups.first(w.e) + (long long)w.m * BM;
        for (int kb = 0; kb < n_kb; ++kb, ++it) {
          const int s = it % STAGES;
          unsigned char* st = a_raw + (size_t)s * C_::STAGE_BYTES;
          mbar_wait(&a_empty[s], ((it / STAGES) & 1u) ^ 1u, status);
          if (lane == 0) {
            mbar_arrive_expect_tx(&a_full[s], (uint32_t)C_::STAGE_BYTES);
            tma_load_3d(st, &tmA, kb * KB, 0, (int)row0, &a_full[s]);
            if (SLOPE) tma_load_3d(st + A_BYTES, &tmSlope, kb * KB, 0, (int)row0, &a_full[s]);
          }
          __syncwarp();
        }
      }
    } else if (warp == 1) {
      // ------------------------------------------------------------------ MMAs (whole warp, one elected lane)
      // A few MMAs are queued at most, and a wait takes as long as three of 64 columns: the next block is waited for in the middle of this one
      // (at its end the tensor cores idled 450 of 830 clocks a block).
      const uint32_t idesc2 = wg::idesc_bf16_m128(2 * BN), idesc1 = wg::idesc_bf16_m128(BN);
      const uint32_t tm = uniform(tmem);
      const uint64_t desc0 = wg::desc_sw64(uniform(smem_u32(smem)));
      const int total = units * n_kb;
      int it = 0, lt = 0, run = 0, run_phase = 0;         // lt: accumulations; run, run_phase: slot of the run's first block and its parity
      for (int u = 0; u < units; ++u) {
        const bool ends = !resident || uniform((uint32_t)w.run_ends()), begins = !resident || uniform((uint32_t)w.run_begins());
        int bs = run;
        uint32_t bp = run_phase;
        for (int k0 = 0; k0 < n_kb; k0 += SEG, ++lt) {
          const int buf = lt & 1, k1 = min(n_kb, k0 + SEG);
          mbar_wait(&acc_empty[buf], ((lt >> 1) & 1u) ^ 1u, status);
          const uint32_t d = tm + (uint32_t)buf * ACC_COLS;
          for (int kb = k0; kb < k1; ++kb, ++it) {
            const int slot = it % A_SLOTS;
            if (begins) mbar_wait(&b_full[bs], bp, status);
            if (it == 0) mbar_wait(&s_full[0], 0, status);
            __syncwarp();
            tc_fence_after();
            const uint32_t a = tm + A_COL0 + (uint32_t)(slot * A_COLS);
            const uint64_t b = desc_at(desc0, (uint32_t)(bs * B_BYTES));
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
              if (ks == 1) {
                if (it + 1 < total) mbar_wait(&s_full[(it + 1) % A_SLOTS], ((it + 1) / A_SLOTS) & 1u, status);
                __syncwarp();
              }
              const uint64_t w1 = desc_at(b, (uint32_t)(ks * 32)), w2 = desc_at(w1, B_PART), w3 = desc_at(w1, 2 * B_PART);
              const uint32_t v1 = a + (uint32_t)(ks * 8), v2 = v1 + KB / 2, v3 = v1 + KB;
              warp_mma_bf16_a_tmem(d, v1, w1, idesc2, kb > k0 || ks ? 1u : 0u);
              warp_mma_bf16_a_tmem(d + BN, v1, w3, idesc1, 1u);
              warp_mma_bf16_a_tmem(d + BN, v2, w1, idesc1, 1u);
              warp_mma_bf16_a_tmem(d + BN, v2, w2, idesc1, 1u);
              warp_mma_bf16_a_tmem(d + BN, v3, w1, idesc1, 1u);
            }
            warp_mma_commit(&s_empty[slot]);
            if (ends) warp_mma_commit(&b_empty[bs]);
            if (++bs == slots) { bs = 0; bp ^= 1u; }
          }
          warp_mma_commit(&acc_full[buf]);
        }
        if (ends) { run = bs; run_phase = bp; }
        w.next();
      }
    } else if (warp < 4) {
      // ------------------------------------------------------------------ the weights' parts
      const int t = threadIdx.x - 64;
      int slot = resident ? n_kb % slots : 0;        // the first ones are split by the epilogue's warps
      uint32_t phase = resident && n_kb == slots ? 1u : 0u;
      auto next = [&] { if (++slot == slots) { slot = 0; phase ^= 1u; } };
      for (int u = 0; u < units; ++u, w.next()) {
        if (!resident) {
          if (t == 0) {
            const unsigned char* src = p.split + ((size_t)w.e * n_tiles + w.n) * n_kb * B_BYTES;
            for (int kb = 0; kb < n_kb; ++kb, next()) {
              mbar_wait(&b_empty[slot], phase ^ 1u, status);
              mbar_arrive_expect_tx(&b_full[slot], (uint32_t)B_BYTES);
              bulk_g2s(smem + (size_t)slot * B_BYTES, src + (size_t)kb * B_BYTES, (uint32_t)B_BYTES, &b_full[slot]);
            }
          }
          continue;
        }
        if (u == 0 || !w.run_begins()) continue;
        const float* W = p.W + (size_t)w.e * N * K;
        float v[32], ahead[32];
        load_weights<FORWARD, 64>(W, w.n * BN, N, K, 0, t, p.w_wide, v);
        for (int kb = 0; kb < n_kb; ++kb, next()) {
          if (kb + 1 < n_kb) load_weights<FORWARD, 64>(W, w.n * BN, N, K, kb + 1, t, p.w_wide, ahead);
          mbar_wait(&b_empty[slot], phase ^ 1u, status);
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
      const int row = (warp & 3) * 32 + lane, set = (warp - 4) >> 2;
      const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16) + A_COL0;
      const int total = units * n_kb;
      for (int it = set; it < total; it += 2) {
        const int s = it % STAGES, slot = it % A_SLOTS;
        mbar_wait(&a_full[s], (it / STAGES) & 1u, status);
        mbar_wait(&s_empty[slot], ((it / A_SLOTS) & 1u) ^ 1u, status);
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
          for (int e = 0; e < 3; ++e) wg::tmem_st_8(lanes + (uint32_t)(slot * A_COLS + e * (KB / 2) + ks * 8), q[e]);
        }
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        tc_fence_before();
        fence_async_smem();                 // the reads precede the TMA write that refills the stage
        __syncwarp();
        if (lane == 0) { mbar_arrive(&s_full[slot]); mbar_arrive(&a_empty[s]); }
      }
    } else {
      // ------------------------------------------------------------------ epilogue: thread = row = TMEM lane, 16 columns at a time, 32 to a slab
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
      unsigned char* slab = slabs + (size_t)(warp - 12) * (SLOPE ? 4096 : 8192);
      unsigned char* slopes = slab + 4096;
      const bool keep = FORWARD && ACT != product::kIdentity && p.slope_out, early = FORWARD && early_residual(p), late = FORWARD && p.residual && !early;
      float* bias = biases + (warp - 12) * 32;
      const uint32_t cols = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(half * 32);
      int lt = 0;
      for (int u = 0; u < units; ++u, w.next()) {
        const long long begin = p.groups.first(w.e), left = p.groups.first(w.e + 1) - begin - (long long)w.m * BM;
        const int rows = min((int)(left < BM ? left : BM) - quarter * 32, 32), n0 = w.n * BN + half * 32;      // of this warp, 0 or fewer: none
        const size_t row0 = (size_t)(begin + (long long)w.m * BM + quarter * 32);
        const bool mine = lane < rows;
        if (FORWARD && w.run_begins()) bias[lane] = p.bias && n0 + lane < N ? p.bias[(size_t)w.e * N + n0 + lane] : 0.f;
        for (int k0 = 0; k0 < n_kb; k0 += SEG, ++lt) {
          const int buf = lt & 1;
          if (lane == 0 && k0 == 0) bulk_wait_read<0>();      // the slabs' last stores have read them
          if (early) {
            __syncwarp();
            fetch_slab(p.residual, row0, rows, n0, N, slab);
          }
          mbar_wait(&acc_full[buf], (lt >> 1) & 1u, status);
          if (early) asm volatile("cp.async.wait_all;" ::: "memory");
          // One copy of this code for both halves, with what is rare apart, and the warp together all through it: it is bound by the instructions
          // of two warps to a scheduler, which wait for their code where it is long.
          const bool whole = k0 + SEG >= n_kb;
          float check = 0.f;
#pragma unroll 1
          for (int h = 0; h < 2; ++h) {
            __syncwarp();
            tc_fence_after();
            uint32_t x[16], y[16];
            const uint32_t at = cols + (uint32_t)buf * ACC_COLS + (uint32_t)(h * 16);
            tmem_ld_16_begin(at, x);
            tmem_ld_16_begin(at + BN, y);
            tmem_ld_wait(x);
            tmem_ld_wait(y);
            if (h == 1) {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&acc_empty[buf]);
            }
            float v[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(x[i]) + __uint_as_float(y[i]);
            if (k0 > 0) {                            // and the sums so far
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const float4 before = *reinterpret_cast<const float4*>(slab + slab_at(lane, h * 4 + j));
                v[4 * j] += before.x; v[4 * j + 1] += before.y; v[4 * j + 2] += before.z; v[4 * j + 3] += before.w;
              }
            }
            if (whole) {
              if (FORWARD) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  const float4 b = *reinterpret_cast<const float4*>(bias + h * 16 + 4 * j);
                  v[4 * j] = fmaf(v[4 * j], wg::UNSCALE, b.x); v[4 * j + 1] = fmaf(v[4 * j + 1], wg::UNSCALE, b.y);
                  v[4 * j + 2] = fmaf(v[4 * j + 2], wg::UNSCALE, b.z); v[4 * j + 3] = fmaf(v[4 * j + 3], wg::UNSCALE, b.w);
                }
              } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] *= wg::UNSCALE;
              }
              float reach = 0.f;
#pragma unroll
              for (int i = 0; i < 16; i += 2) reach = largest(reach, v[i], v[i + 1]);
              check = largest(check, reach, 0.f);
              if ((ACT == product::kSilu || ACT == product::kSigmoid) && !(reach <= product::kNear)) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                  *reinterpret_cast<float4*>(slopes + slab_at(lane, h * 4 + j)) = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
                far_row<ACT>(slab, slopes, h * 4, early);
                continue;
              }
              if (FORWARD && ACT != product::kIdentity) {
                if (keep) {
#pragma unroll
                  for (int j = 0; j < 4; ++j) {
                    float2 d[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                      const float2 r = product::activate_near<ACT>(make_float2(v[4 * j + 2 * i], v[4 * j + 2 * i + 1]), d[i]);
                      v[4 * j + 2 * i] = r.x; v[4 * j + 2 * i + 1] = r.y;
                    }
                    *reinterpret_cast<float4*>(slopes + slab_at(lane, h * 4 + j)) = make_float4(d[0].x, d[0].y, d[1].x, d[1].y);
                  }
                } else {
#pragma unroll
                  for (int i = 0; i < 8; ++i) {
                    float2 d;
                    const float2 r = product::activate_near<ACT>(make_float2(v[2 * i], v[2 * i + 1]), d);
                    v[2 * i] = r.x; v[2 * i + 1] = r.y;
                  }
                }
              }
              if (early) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  const float4 more = *reinterpret_cast<const float4*>(slab + slab_at(lane, h * 4 + j));
                  v[4 * j] += more.x; v[4 * j + 1] += more.y; v[4 * j + 2] += more.z; v[4 * j + 3] += more.w;
                }
              }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
              *reinterpret_cast<float4*>(slab + slab_at(lane, h * 4 + j)) = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
          }
          if (!whole) continue;
          if (mine && !(check <= 3.402823466e38f)) wild_row<FORWARD, SLOPE, ACT>(p, w.e, row0 + lane, n0, slab, slopes);
          fence_async_smem();
          __syncwarp();
          if (n0 < N && rows > 0) {
            if (p.c_wide && !late && (rows == 32 || row0 + rows == (size_t)p.groups.rows)) {
              if (lane == 0) tma_store_3d(&tmC, n0, (int)row0, slab);
            } else {
              store_slab(p.C, late ? p.residual : nullptr, row0, rows, n0, N, N, p.c_wide, slab);
            }
            if (keep) {
              if (rows == 32 || row0 + rows == (size_t)p.groups.rows) {
                if (lane == 0) tma_store_3d(&tmD, n0, (int)row0, slopes);
              } else {
                store_slab(p.slope_out, nullptr, row0, rows, n0, N, p.ldd, true, slopes);
              }
            }
            if (lane == 0) bulk_commit();
          }
          __syncwarp();
        }
      }
      if (lane == 0) bulk_wait_all<0>();
    }
  }
  // rows of no expert
  if (p.groups.offsets) {
    const size_t first = (size_t)p.groups.first(X) * N, end = (size_t)p.groups.rows * N;
    for (size_t i = first + (size_t)blockIdx.x * NT + threadIdx.x; i < end; i += (size_t)gridDim.x * NT) p.C[i] = 0.f;
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) { tc_fence_after(); tmem_dealloc(tmem, 512); }
}

}  // namespace ptc
}  // namespace fasteq
