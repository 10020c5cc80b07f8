// FP32 weight gradient of the dense layers on the tensor cores:  gw[e][n, k] = sum over e's rows r of (g[r, n] slope[r, n]) x[r, k],
// gb[e][n] = sum_r g[r, n] slope[r, n].
//
// The arithmetic of product_tc.cuh (three bf16 parts per operand, six products, an accumulator for the first and one for the small ones) with the
// rows as contraction index: both operands are split column by column as they come, thread = channel, pairs of rows packed, so nothing is turned.
// A CTA takes a chunk of an expert's rows and a tile of 128 x 64 of its matrix:
//   warp 0       brings blocks of 32 rows of g (and slope) and x (TMA)
//   warps 1, 2   issue the MMAs, of the even blocks and of the odd ones: each has accumulators of its own, and its waits pass under the other's MMAs
//   warps 4-11   split g into tensor memory, four warps the even and four the odd blocks, and add its columns for gb
//   warps 12-15  split x into shared memory
//   warps 16-23  every 256 rows of either add the accumulators to their registers; in the end write the tile's sums
// Chunks are long enough to give each SM one tile, at least 64 rows, or 256 where experts have no more than that on average (chunk_rows); an expert of several chunks leaves partial sums, which a second kernel adds
// in order.  Sums that are not finite are formed again in FP32, the whole tile.  Errors against 64 bits (2-norm, 1e-8; torch's FP32 products, this) at 60, 1,000,
// 12,288 and 100,003 rows of 128 x 128: 14.0, 5.4; 25.8, 8.3; 63.1, 12.6; 112, 23.6; operands of one sign 11.9, 5.7; 9.8, 6.5; 17.2, 12.0; 19.9, 34.2.
// Bound: the warps' instructions between the waits (the tensor cores are busy for 31 %, issue slots for 53 % of the time).  Measured, g without a slope:
// 12,288 rows of 128 x 256 12.9 us, 24,576 18.8 us, 100,000 of 128 x 128 32.0 us (103 TFLOP/s of FP32-accurate products; one issuing warp: 34.3).
#pragma once
#include "product_tc.cuh"

namespace fasteq {
namespace pwg {

using namespace ptc;
using product::Chunk;

constexpr int TM = 128, TN = 64, ROWS = 32, NTW = 768, STAGES_W = 4, SLOTS_W = 4, SEG_W = 256 / ROWS;
constexpr int G_BYTES = ROWS * TM * 4, X_BYTES = ROWS * TN * 4;
template <bool SLOPE> struct CfgW {
  static constexpr int STAGE = G_BYTES * (SLOPE ? 2 : 1) + X_BYTES;
  static constexpr int SMEM = 1024 + SLOTS_W * B_BYTES + STAGES_W * STAGE + (2 * STAGES_W + 2 * A_SLOTS + 2 * SLOTS_W + 4) * 8 + 2 * TM * 4 + 32;
  static_assert(SMEM <= 227 * 1024, "shared memory of one CTA");
};

struct ArgsW {
  Groups groups;
  const float *x, *g, *slope;
  float *gw, *gb, *partial;           // gb may be null
  int K, N, ldx, ldg, ldd;            // columns, and columns between the rows of x, g and slope
  int size, tiles_k, tiles;           // size: rows of a chunk
  bool wide;                          // 16-byte accesses of the results
  int* status;
};

// The tile again with FP32's own products: 64 columns of it to 64 threads, every 12th row each.
template <bool SLOPE>
__device__ __noinline__ void tile_fp32(const ArgsW& p, const Chunk& c, int n0, int k0, float* dst) {
  const int k = k0 + (threadIdx.x & 63);
  for (int n = n0 + (threadIdx.x >> 6); n < min(p.N, n0 + TM); n += NTW / 64) {
    if (k >= p.K) return;
    float total = 0.f;
#pragma unroll 1
    for (int r0 = 0; r0 < c.rows; r0 += ROWS) {
      float s = 0.f;
#pragma unroll 4
      for (int r = r0; r < min(c.rows, r0 + ROWS); ++r) {
        const size_t row = (size_t)(c.m0 + r);
        s = fmaf(SLOPE ? p.g[row * p.ldg + n] * p.slope[row * p.ldd + n] : p.g[row * p.ldg + n], p.x[row * p.ldx + k], s);
      }
      total += s;
    }
    dst[(size_t)n * p.K + k] = total;
  }
}

template <bool SLOPE>
__global__ void __launch_bounds__(NTW, 1) product_wgrad_tc_kernel(const __grid_constant__ ArgsW p, const __grid_constant__ CUtensorMap tmG,
                                                                  const __grid_constant__ CUtensorMap tmD, const __grid_constant__ CUtensorMap tmX) {
  using C_ = CfgW<SLOPE>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* raw = smem + SLOTS_W * B_BYTES;               // [stage]: g [32][128] | slope | x [32][64]
  uint64_t* a_full = reinterpret_cast<uint64_t*>(raw + STAGES_W * C_::STAGE);
  uint64_t* a_empty = a_full + STAGES_W;
  uint64_t* s_full = a_empty + STAGES_W;
  uint64_t* s_empty = s_full + A_SLOTS;
  uint64_t* b_full = s_empty + A_SLOTS;
  uint64_t* b_empty = b_full + SLOTS_W;
  uint64_t* acc_full = b_empty + SLOTS_W;
  uint64_t* acc_empty = acc_full + 2;
  float* columns = reinterpret_cast<float*>(acc_empty + 2);    // [2][128] column sums of g
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(columns + 2 * TM);
  int* redo = reinterpret_cast<int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int* status = p.status;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES_W; ++s) { mbar_init(&a_full[s], 1); mbar_init(&a_empty[s], 8); }
    for (int s = 0; s < A_SLOTS; ++s) { mbar_init(&s_full[s], 4); mbar_init(&s_empty[s], 1); }
    for (int s = 0; s < SLOTS_W; ++s) { mbar_init(&b_full[s], 4); mbar_init(&b_empty[s], 1); }
    for (int s = 0; s < 2; ++s) { mbar_init(&acc_full[s], 1); mbar_init(&acc_empty[s], 8); }
    mbar_fence_init();
    *redo = 0;
  }
  if (warp == 1) tmem_alloc(tmem_slot, 512);
  if (threadIdx.x == 64) {
    prefetch_map(&tmG);
    prefetch_map(&tmX);
    if (SLOPE) prefetch_map(&tmD);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  wait_for_previous_kernel();
  const uint32_t tmem = *tmem_slot;
  const Chunk c = product::chunk_of(p.groups, p.groups.experts, p.size, blockIdx.x / p.tiles);
  const int tile = blockIdx.x % p.tiles, n0 = tile / p.tiles_k * TM, k0 = tile % p.tiles_k * TN, N = p.N, K = p.K;
  const int n_blocks = (c.rows + ROWS - 1) / ROWS;
  float* dst = nullptr;
  if (n_blocks > 0) {
    dst = c.count == 1 ? p.gw + (size_t)c.e * N * K : p.partial + (size_t)product::partial_slot(c, p.size) * ((size_t)N * K + N);
    if (warp == 0) {
      // ------------------------------------------------------------------ blocks of 32 rows
      for (int i = 0; i < n_blocks; ++i) {
        const int s = i % STAGES_W;
        unsigned char* st = raw + (size_t)s * C_::STAGE;
        const long long row = c.m0 + (long long)i * ROWS;
        mbar_wait(&a_empty[s], ((i / STAGES_W) & 1u) ^ 1u, status);
        if (lane == 0) {
          mbar_arrive_expect_tx(&a_full[s], (uint32_t)C_::STAGE);
          tma_load_3d(st, &tmG, n0, 0, (int)row, &a_full[s]);
          if (SLOPE) tma_load_3d(st + G_BYTES, &tmD, n0, 0, (int)row, &a_full[s]);
          tma_load_3d(st + C_::STAGE - X_BYTES, &tmX, k0, 0, (int)row, &a_full[s]);
        }
        __syncwarp();
      }
    } else if (warp == 1 || warp == 2) {
      // ------------------------------------------------------------------ MMAs
      const int pipe = warp - 1;
      const uint32_t idesc2 = wg::idesc_bf16_m128(2 * BN), idesc1 = wg::idesc_bf16_m128(BN), tm = uniform(tmem);
      const uint64_t desc0 = wg::desc_sw64(uniform(smem_u32(smem)));
      const uint32_t d = tm + (uint32_t)pipe * ACC_COLS;
      for (int i = pipe, j = 0; i < n_blocks; i += 2, ++j) {
        const int slot = i % A_SLOTS, bs = i % SLOTS_W;
        if (j % SEG_W == 0) mbar_wait(&acc_empty[pipe], ((j / SEG_W) & 1u) ^ 1u, status);
        mbar_wait(&b_full[bs], (i / SLOTS_W) & 1u, status);
        mbar_wait(&s_full[slot], (i / A_SLOTS) & 1u, status);
        __syncwarp();
        tc_fence_after();
        const uint32_t a = tm + A_COL0 + (uint32_t)(slot * A_COLS);
        const uint64_t b = desc_at(desc0, (uint32_t)(bs * B_BYTES));
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          const uint64_t w1 = desc_at(b, (uint32_t)(ks * 32)), w2 = desc_at(w1, B_PART), w3 = desc_at(w1, 2 * B_PART);
          const uint32_t v1 = a + (uint32_t)(ks * 8), v2 = v1 + KB / 2, v3 = v1 + KB;
          warp_mma_bf16_a_tmem(d, v1, w1, idesc2, j % SEG_W || ks ? 1u : 0u);
          warp_mma_bf16_a_tmem(d + BN, v1, w3, idesc1, 1u);
          warp_mma_bf16_a_tmem(d + BN, v2, w1, idesc1, 1u);
          warp_mma_bf16_a_tmem(d + BN, v2, w2, idesc1, 1u);
          warp_mma_bf16_a_tmem(d + BN, v3, w1, idesc1, 1u);
        }
        warp_mma_commit(&s_empty[slot]);
        warp_mma_commit(&b_empty[bs]);
        if ((j + 1) % SEG_W == 0 || i + 2 >= n_blocks) warp_mma_commit(&acc_full[pipe]);
      }
    } else if (warp >= 4 && warp < 12) {
      // ------------------------------------------------------------------ g: thread = channel = TMEM lane
      const int ch = (warp & 3) * 32 + lane, set = (warp - 4) >> 2;
      const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16) + A_COL0;
      float column = 0.f;
      for (int i = set; i < n_blocks; i += 2) {
        const int s = i % STAGES_W, slot = i % A_SLOTS, rows = c.rows - i * ROWS;
        mbar_wait(&a_full[s], (i / STAGES_W) & 1u, status);
        mbar_wait(&s_empty[slot], ((i / A_SLOTS) & 1u) ^ 1u, status);
        __syncwarp();
        tc_fence_after();
        const float* st = reinterpret_cast<const float*>(raw + (size_t)s * C_::STAGE) + ch;
        float2 sum = make_float2(0.f, 0.f);
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          uint32_t q[3][8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int r = ks * 16 + 2 * j;
            float2 v = make_float2(st[r * TM], st[(r + 1) * TM]);
            if (SLOPE) v = vmul(v, make_float2(st[G_BYTES / 4 + r * TM], st[G_BYTES / 4 + (r + 1) * TM]));
            if (rows < ROWS) {                     // TMA brought the rows behind the expert's last as well
              if (r >= rows) v.x = 0.f;
              if (r + 1 >= rows) v.y = 0.f;
            }
            sum = vadd(sum, v);
            wg::split_pair(v, q[0][j], q[1][j], q[2][j]);
          }
#pragma unroll
          for (int e = 0; e < 3; ++e) wg::tmem_st_8(lanes + (uint32_t)(slot * A_COLS + e * (KB / 2) + ks * 8), q[e]);
        }
        column += sum.x + sum.y;
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        tc_fence_before();
        fence_async_smem();
        __syncwarp();
        if (lane == 0) { mbar_arrive(&s_full[slot]); mbar_arrive(&a_empty[s]); }
      }
      columns[set * TM + ch] = column;
    } else if (warp >= 12 && warp < 16) {
      // ------------------------------------------------------------------ x: thread = channel and 16 of the 32 rows
      const int t = threadIdx.x - 384, ch = t & 63, r0 = (t >> 6) * 16;
      for (int i = 0; i < n_blocks; ++i) {
        const int s = i % STAGES_W, bs = i % SLOTS_W, rows = c.rows - i * ROWS;
        mbar_wait(&a_full[s], (i / STAGES_W) & 1u, status);
        mbar_wait(&b_empty[bs], ((i / SLOTS_W) & 1u) ^ 1u, status);
        const float* st = reinterpret_cast<const float*>(raw + (size_t)(s + 1) * C_::STAGE - X_BYTES) + r0 * TN + ch;
        float v[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = st[j * TN];
        if (rows < ROWS) {
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (r0 + j >= rows) v[j] = 0.f;
        }
        store_weights<false, 128>(smem + (size_t)bs * B_BYTES, t, v);
        fence_async_smem();
        __syncwarp();
        if (lane == 0) { mbar_arrive(&b_full[bs]); mbar_arrive(&a_empty[s]); }
      }
    } else if (warp >= 16) {
      // ------------------------------------------------------------------ sums: thread = row n of the tile, 32 columns
      const int quarter = warp & 3, half = (warp - 16) >> 2;
      const uint32_t cols = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(half * 32);
      float2 sum[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) sum[j] = make_float2(0.f, 0.f);
      // accumulations of the two pipes in turn: 0 and 1 their first, 2 and 3 their second, ...
      const int n_acc = (n_blocks + 2 * SEG_W - 1) / (2 * SEG_W) * 2;
      for (int seg = 0; seg < n_acc; ++seg) {
        const int buf = seg & 1, first = (seg >> 1) * 2 * SEG_W + buf, blocks = min(SEG_W, (n_blocks - first + 1) / 2);
        if (blocks <= 0) continue;
        mbar_wait(&acc_full[buf], (seg >> 1) & 1u, status);
        __syncwarp();
        tc_fence_after();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t x[16], y[16];
          const uint32_t at = cols + (uint32_t)buf * ACC_COLS + (uint32_t)(h * 16);
          tmem_ld_16_begin(at, x);
          tmem_ld_16_begin(at + BN, y);
          tmem_ld_wait(x);
          tmem_ld_wait(y);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float2 large = make_float2(__uint_as_float(x[2 * j]), __uint_as_float(x[2 * j + 1]));
            const float2 small = make_float2(__uint_as_float(y[2 * j]), __uint_as_float(y[2 * j + 1]));
            sum[h * 8 + j] = vadd(sum[h * 8 + j], vadd(large, small));
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_empty[buf]);
      }
      const int n = n0 + quarter * 32 + lane, k = k0 + half * 32;
      if (n < N) {
        float2 all = make_float2(0.f, 0.f);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          all = vadd(all, sum[j]);
          sum[j] = vmul(sum[j], make_float2(wg::UNSCALE, wg::UNSCALE));
        }
        if (!(fabsf(all.x + all.y) <= 3.402823466e38f)) *reinterpret_cast<volatile int*>(redo) = 1;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float2 v[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = sum[h * 8 + j];
          store_16(dst + (size_t)n * K + k + h * 16, K - k - h * 16, p.wide, v);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) { tc_fence_after(); tmem_dealloc(tmem, 512); }
  if (n_blocks == 0) return;
  if (p.gb && k0 == 0 && threadIdx.x < TM && n0 + (int)threadIdx.x < N) {
    const float v = columns[threadIdx.x] + columns[TM + threadIdx.x];
    if (c.count == 1) p.gb[(size_t)c.e * N + n0 + threadIdx.x] = v; else dst[(size_t)N * K + n0 + threadIdx.x] = v;
  }
  if (*redo) tile_fp32<SLOPE>(p, c, n0, k0, dst);
}

}  // namespace pwg
}  // namespace fasteq
