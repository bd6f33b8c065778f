// Matrix product with 4-bit weights on the 5th-generation tensor cores (see gemm_w4.cu for the weights' form):
//   y[M, N] = x[M, K] * W[N, K]^T,   W[n, k] = (code[n, k] - 8) * scale[n, k / G].
//
// 128 rows of W are the rows of the tensor core's tile, T tokens its columns.  The codes become bfloat16 whole numbers on
// their way into tensor memory, where the product takes its left operand from: the weights never exist in 16 bits outside the
// SM.  A group's columns are summed from zero in a tile of their own, which is read back, multiplied by the group's scales
// (a thread holds one row) and added up in registers: nothing but the result is rounded, and folding the scales into 16-bit
// weights would cost as many instructions (four multiplications for eight weights, against T / 2 for 64 of a thread's).
//
//   two load warps: TMA of codes (128 rows x 256 columns, 16 KB) and of x (T rows x 128) into rings
//   8 worker warps: a row's 64 codes -> 32 words of bfloat16 pairs -> tensor memory; the sums of the chunk before -> registers
//   MMA warp:       eight tcgen05.mma a chunk of 128 columns
// Where the tiles are too few for the chip a cluster of 2, 4 or 8 blocks shares one: each sums a stretch of K, and they add up
// over distributed shared memory in the order of the stretches.
//
// What bounds it: the workers, who unpack the codes (11 instructions for eight weights) and scale the sums in turn: 28,672 x
// 4,096 takes 25 us with 16 tokens, 30 with 64 (reading the codes 9.3, the products with 64 tokens 9.0), 57 with 128.
#include <type_traits>

#include "gemm_w4.cuh"
#include "tc5_primitives.cuh"
#include "tensor_map.cuh"

namespace {
using namespace fg_tc5;
using namespace fg_w4;

constexpr int ROWS4 = 128;   // rows of W a tile
constexpr int KC = 128;      // columns of a chunk
constexpr int W_COLS = 256;  // columns of a stage of codes: two chunks
constexpr int W_STAGE = ROWS4 * W_COLS / 2;
constexpr int WORKERS = 256, THREADS4 = WORKERS + 96, LOAD_W_WARP = 8, LOAD_X_WARP = 9, MMA_WARP_ID = 10;
constexpr int A_COLS = KC / 2;  // tensor-memory columns of a chunk of weights

// T tokens a tile, G columns a group
template <int T_, int G_>
struct Shape4 {
  static constexpr int T = T_, TC = T / 2, G = G_, PARTS = KC / G;
  static constexpr int X_UNIT = T * KC * 2, X_HALF = T * 128;  // a chunk of x: two halves of 64 columns, rows of 128 bytes
  static constexpr int COL_A = 0, COL_D = 2 * A_COLS;
  static constexpr int D_COLS = PARTS * T;
  static constexpr int D_BUFS = COL_D + 2 * D_COLS <= 256 || (COL_D + D_COLS > 256 && COL_D + 2 * D_COLS <= 512) ? 2 : 1;
  static constexpr int TMEM = COL_D + D_BUFS * D_COLS <= 256 ? 256 : 512;
  static constexpr int BLOCKS = TMEM == 256 && T <= 64 ? 2 : 1;  // an SM
  static constexpr int W_STAGES = T <= 32 ? 4 : BLOCKS == 2 ? 3 : 4;
  static constexpr int X_UNITS = T == 64 ? 3 : 4;
  static constexpr int RINGS = W_STAGES * W_STAGE + X_UNITS * X_UNIT;
  // The blocks of a cluster wait for one another, so none of them may wait for tensor memory that a block of another
  // cluster keeps meanwhile: shared memory is asked for such that an SM holds no more blocks, of any of these
  // shapes, than its tensor memory serves.  (And no block takes tensor memory before the kernel ahead of this one is over.)
  static constexpr size_t LEAST = (TMEM == 256 ? 77 : 152) * 1024;
  static constexpr size_t SMEM = 1024 + RINGS > LEAST ? 1024 + RINGS : LEAST;
  static_assert(COL_D + D_BUFS * D_COLS <= TMEM && SMEM <= 227 * 1024 && BLOCKS * SMEM <= 227 * 1024, "");
  static_assert(T * ROWS4 * 4 <= RINGS, "the exchange of a cluster reuses the rings");
};

__device__ __forceinline__ void tma_2d(void* dst, const CUtensorMap* map, int c0, int c1, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(c0), "r"(c1), "r"(smem_u32(bar))
      : "memory");
}
// 8 consecutive columns of this thread's lane; several may be in flight before tmem_ld_wait
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }

__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
  return r;
}
// one element of the result from its sum; called by whole warps, a lane a row of W (32 neighbouring ones)
template <typename TO>
__device__ __forceinline__ void store_sum(float v, int m, int n, bool ok, int N, TO* y, int ldy, const Epilogue4& epi, float bias) {
  using namespace fg_skinny;
  if (epi.gated) {
    const float up = __shfl_down_sync(0xffffffffu, v, 8);
    if (ok && n < N && (n & 8) == 0) {
      // both are rounded to bfloat16 first, as a separate gate kernel would see them
      const float gr = __bfloat162float(__float2bfloat16_rn(v)), ur = __bfloat162float(__float2bfloat16_rn(up));
      y[(size_t)m * ldy + (n >> 4) * 8 + (n & 7)] = from_f32<TO>((epi.act ? fmaxf(gr, 0.f) : gr / (1.f + expf(-gr))) * ur);
    }
    return;
  }
  if (!ok || n >= N) return;
  v += bias;
  // the product is rounded to bfloat16 before the activation, as a separate kernel would see it
  if (epi.act != ACT_NONE) v = activate(__bfloat162float(__float2bfloat16_rn(v)), epi.act);
  y[(size_t)m * ldy + n] = from_f32<TO>(v);
}

template <typename S, typename TO>
__global__ void __launch_bounds__(THREADS4, S::BLOCKS)
gemm_w4_tc5_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map,
                   const __nv_bfloat16* __restrict__ scales, TO* y, int ldy, int M, int N, int K, int share, int m_tiles,
                   Epilogue4 epi, int* status) {
  constexpr int T = S::T, TC = S::TC, PARTS = S::PARTS;
  extern __shared__ unsigned char smem_unaligned[];
  unsigned char* const ws = reinterpret_cast<unsigned char*>(((uintptr_t)smem_unaligned + 1023) & ~(uintptr_t)1023);
  unsigned char* const xs = ws + S::W_STAGES * W_STAGE;
  __shared__ __align__(8) uint64_t w_full[S::W_STAGES], w_empty[S::W_STAGES], x_full[S::X_UNITS], x_empty[S::X_UNITS], op_full[2],
      d_full[2], d_empty[2], drained;
  __shared__ uint32_t tmem_base;
  __shared__ int gave_up;
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);

  pdl_trigger();
  if (tid == 0) {
    gave_up = 0;
    for (int i = 0; i < S::W_STAGES; ++i) {
      mbar_init(&w_full[i], 1);
      mbar_init(&w_empty[i], WORKERS / 32);
    }
    for (int i = 0; i < S::X_UNITS; ++i) {
      mbar_init(&x_full[i], 1);
      mbar_init(&x_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&op_full[i], WORKERS / 32);
      mbar_init(&d_full[i], 1);
      mbar_init(&d_empty[i], WORKERS / 32);
    }
    mbar_init(&drained, 1);
    mbar_fence_init();
  }
  __syncthreads();

  const int rank = share > 1 ? (int)cluster_rank() : 0;
  const int tile = blockIdx.x / share, n0 = tile / m_tiles * ROWS4, m0 = tile % m_tiles * T;
  // the block's stretch of K, in stages of W_COLS columns
  const int stages = (K + W_COLS - 1) / W_COLS, per_block = (stages + share - 1) / share;
  const int stage0 = min(stages, rank * per_block), n_stages = min(per_block, stages - stage0);
  const int k_begin = stage0 * W_COLS;
  // (chunks wholly behind K, in the last stage, are left out)
  const int total = n_stages > 0 ? (min(K, (stage0 + n_stages) * W_COLS) - k_begin + KC - 1) / KC : 0;

  // the tensor memory's address, from the MMA warp to the workers (the load warps do without)
  auto share_tmem = [&]() { asm volatile("bar.sync 1, %0;\n" ::"n"(WORKERS + 32) : "memory"); };

  if (warp == LOAD_W_WARP) {
    if (elect_one()) {
      // the codes depend on nothing that is computed in the step: no wait for the kernel ahead
      for (int i = 0; i < n_stages; ++i) {
        const int slot = i % S::W_STAGES, use = i / S::W_STAGES;
        if (use > 0) mbar_wait(&w_empty[slot], (use - 1) & 1, status, &gave_up);
        mbar_arrive_expect(&w_full[slot], W_STAGE);
        tma_2d(ws + slot * W_STAGE, &w_map, (stage0 + i) * (W_COLS / 2), n0, &w_full[slot]);
      }
      if (*reinterpret_cast<volatile int*>(&gave_up) != 0)
        // a wait ran out: the copies in flight land before the block leaves
        for (int i = 0; i < min(S::W_STAGES, n_stages); ++i) mbar_wait(&w_full[i], (n_stages - 1 - i) / S::W_STAGES & 1, status);
    }
    __syncwarp();
  } else if (warp == LOAD_X_WARP) {
    if (elect_one()) {
      pdl_wait();
      for (int j = 0; j < total; ++j) {
        const int slot = j % S::X_UNITS, use = j / S::X_UNITS;
        if (use > 0) mbar_wait(&x_empty[slot], (use - 1) & 1, status, &gave_up);
        mbar_arrive_expect(&x_full[slot], S::X_UNIT);
        tma_2d(xs + slot * S::X_UNIT, &x_map, k_begin + j * KC, m0, &x_full[slot]);
        tma_2d(xs + slot * S::X_UNIT + S::X_HALF, &x_map, k_begin + j * KC + 64, m0, &x_full[slot]);
      }
      if (*reinterpret_cast<volatile int*>(&gave_up) != 0)
        for (int i = 0; i < min(S::X_UNITS, total); ++i) mbar_wait(&x_full[i], (total - 1 - i) / S::X_UNITS & 1, status);
    }
    __syncwarp();
  } else if (warp == MMA_WARP_ID) {
    pdl_wait();
    tmem_alloc(&tmem_base, S::TMEM);
    tmem_relinquish();
    tc_fence_before();
    share_tmem();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_base, 0);
    if (elect_one()) {
      constexpr uint32_t IDESC = instr_desc(T, false);
      const uint64_t x_desc = smem_desc(xs, 16);
      int slot = 0, use = 0;
      for (int j = 0; j < total; ++j) {
        const int buf = j & 1, db = S::D_BUFS == 2 ? buf : 0, d_use = S::D_BUFS == 2 ? j >> 1 : j;
        mbar_wait(&op_full[buf], (j >> 1) & 1, status, &gave_up);
        mbar_wait(&x_full[slot], use & 1, status, &gave_up);
        if (d_use > 0) mbar_wait(&d_empty[db], (d_use - 1) & 1, status, &gave_up);
        tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < KC / 16; ++kk) {
          const uint64_t bd = x_desc + (uint64_t)((slot * S::X_UNIT + (kk >> 2) * S::X_HALF + (kk & 3) * 32) >> 4);
          umma_f16_ts(tmem + S::COL_D + db * S::D_COLS + kk * 16 / S::G * T, tmem + S::COL_A + buf * A_COLS + kk * 8, bd, IDESC,
                      kk * 16 % S::G ? 1u : 0u);
        }
        umma_commit(&x_empty[slot]);
        umma_commit(&d_full[db]);
        if (++slot == S::X_UNITS) {
          slot = 0;
          ++use;
        }
      }
      if (*reinterpret_cast<volatile int*>(&gave_up) != 0) {
        umma_commit(&drained);
        mbar_wait(&drained, 0, status);
      }
    }
    __syncwarp();
  } else {
    // ================================ workers ================================
    const int half = warp >> 2, row = (warp & 3) * 32 + lane, n = n0 + row;
    const uint32_t my_lane = (uint32_t)((warp & 3) * 32) << 16;
    const int groups = K / S::G;
    const __nv_bfloat16* my_scales = scales + (size_t)min(n, N - 1) * groups;
    float acc[TC];
#pragma unroll
    for (int i = 0; i < TC; ++i) acc[i] = 0.f;
    share_tmem();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_base, 0);
    const __nv_bfloat16* next_scale = my_scales + k_begin / S::G;
    __nv_bfloat16 sc_next[PARTS];
    float sc[PARTS];
    // pieces of 16 bytes (32 codes) of this thread's row in a stage, swizzled: chunk c's two for this half of the columns
    const unsigned char* my_row = ws + row * 128;
    int piece_at[2][2];
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int i = 0; i < 2; ++i) piece_at[c][i] = ((c * 4 + half * 2 + i) ^ (row & 7)) << 4;
    const uint32_t op0 = tmem + my_lane + S::COL_A + half * 32, d0 = tmem + my_lane + S::COL_D + half * TC;

    // a chunk's codes (the stage's chunk PARITY) -> tensor memory; the sums of the chunk before it -> acc
    auto expand = [&](auto parity_tag, int j, int slot) {
      constexpr int PARITY = decltype(parity_tag)::value;
#pragma unroll
      for (int p = 0; p < PARTS; ++p) {
        sc[p] = __bfloat162float(sc_next[p]);
        // (groups of 128: every chunk is whole)
        sc_next[p] = S::G == KC || k_begin + j * KC + p * S::G < K ? next_scale[p] : __float2bfloat16_rn(0.f);
      }
      next_scale += PARTS;
      uint4 codes[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) codes[i] = *reinterpret_cast<const uint4*>(my_row + slot * W_STAGE + piece_at[PARITY][i]);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t w[4] = {codes[i].x, codes[i].y, codes[i].z, codes[i].w};
        uint32_t v[16];
#pragma unroll
        for (int c = 0; c < 16; ++c) v[c] = weights_of(w[c >> 2], c & 3);
        tmem_st16(op0 + PARITY * A_COLS + i * 16, v);
      }
      if (PARITY == 1) warp_arrive(&w_empty[slot]);
      tmem_st_wait();
      tc_fence_before();
      warp_arrive(&op_full[PARITY]);
    };
    auto add_sums = [&](int j) {  // of chunk j
      const int db = S::D_BUFS == 2 ? j & 1 : 0, d_use = S::D_BUFS == 2 ? j >> 1 : j;
      mbar_wait(&d_full[db], d_use & 1, status, &gave_up);
      tc_fence_after();
#pragma unroll
      for (int p = 0; p < PARTS; ++p) {
        const uint32_t d = d0 + db * S::D_COLS + p * T;
        constexpr int FLIGHT = TC < 32 ? TC : 32;  // columns in flight
#pragma unroll
        for (int c = 0; c < TC; c += FLIGHT) {
          uint32_t v[FLIGHT];
#pragma unroll
          for (int i = 0; i < FLIGHT; i += 8) tmem_ld8(d + c + i, v + i);
          tmem_ld_wait();
          if (p + 1 == PARTS && c + FLIGHT >= TC) {
            tc_fence_before();
            warp_arrive(&d_empty[db]);
          }
#pragma unroll
          for (int i = 0; i < FLIGHT; ++i) acc[c + i] = fmaf(__uint_as_float(v[i]), sc[p], acc[c + i]);
        }
      }
    };
    int slot = 0, use = 0;
#pragma unroll
    for (int p = 0; p < PARTS; ++p) sc_next[p] = __float2bfloat16_rn(0.f);
    for (int j = 0; j < total; j += 2) {
      mbar_wait(&w_full[slot], use & 1, status, &gave_up);
      expand(std::integral_constant<int, 0>(), j, slot);
      if (j > 0) add_sums(j - 1);
      if (j + 1 < total) {
        expand(std::integral_constant<int, 1>(), j + 1, slot);
        add_sums(j);
      }
      if (++slot == S::W_STAGES) {
        slot = 0;
        ++use;
      }
    }
    if (total > 0) {
#pragma unroll
      for (int p = 0; p < PARTS; ++p) sc[p] = __bfloat162float(sc_next[p]);
      add_sums(total - 1);
    }
    // the sums to shared memory: every chunk of this block has been read out of the rings by now
    float* part = reinterpret_cast<float*>(ws);
#pragma unroll
    for (int i = 0; i < TC; ++i) part[(half * TC + i) * ROWS4 + row] = acc[i];
    if (share == 1) asm volatile("bar.sync 2, %0;\n" ::"n"(WORKERS) : "memory");
  }
  if (share > 1) cluster_sync();
  if (tid < WORKERS) {
    // a warp 32 rows of W of one token, the cluster's warps in turn (one loop for all of them: the activations' code once)
    const int tokens = min(T, M - m0);
#pragma unroll 1
    for (int u = warp * share + rank; u < tokens * 4; u += 8 * share) {
      const int i = u >> 2, r = (u & 3) * 32 + lane, n = n0 + r;
      float v;
      if (share == 1) {
        v = reinterpret_cast<const float*>(ws)[i * ROWS4 + r];
      } else {
        const uint32_t at = smem_u32(ws) + (i * ROWS4 + r) * 4;
        float p[8];
#pragma unroll
        for (int s = 0; s < 8; ++s) p[s] = s < share ? ld_cluster(at, s) : 0.f;
        v = p[0];
#pragma unroll
        for (int s = 1; s < 8; ++s) v += p[s];
      }
      const float bias = epi.bias != nullptr && n < N ? __bfloat162float(epi.bias[n]) : 0.f;
      store_sum<TO>(v, m0 + i, n, true, N, y, ldy, epi, bias);
    }
  }
  if (share > 1) {
    __syncwarp();
    cluster_sync();  // nobody leaves while its sums are being read
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == MMA_WARP_ID) tmem_dealloc(__shfl_sync(0xffffffffu, tmem_base, 0), S::TMEM);
}

template <typename S, typename TO>
int launch(const void* x, int ldx, const void* w, const void* scales, void* y, int ldy, int M, int N, int K, int share,
           const Epilogue4& epi, int* status, cudaStream_t stream) {
  alignas(64) CUtensorMap w_map, x_map;
  const cuuint64_t wd[2] = {(cuuint64_t)K / 2, (cuuint64_t)N}, wst[1] = {(cuuint64_t)K / 2};
  const cuuint32_t wbox[2] = {W_COLS / 2, ROWS4};
  int rc = fg_encode_tensor_map(&w_map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, w, wd, wst, wbox);
  if (rc) return rc;
  const cuuint64_t xd[2] = {(cuuint64_t)K, (cuuint64_t)M}, xst[1] = {(cuuint64_t)ldx * 2};
  const cuuint32_t xbox[2] = {64, (cuuint32_t)S::T};
  rc = fg_encode_tensor_map(&x_map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, x, xd, xst, xbox);
  if (rc) return rc;
  auto kern = gemm_w4_tc5_kernel<S, TO>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::SMEM);
  FG_CHECK_ARG(e == cudaSuccess, "fg_gemm_w4_tc5: shared memory: %s", cudaGetErrorString(e));
  const int m_tiles = (M + S::T - 1) / S::T;
  const long tiles = (long)m_tiles * ((N + ROWS4 - 1) / ROWS4);
  FG_CHECK_ARG(tiles * share <= (1l << 30), "fg_gemm_w4_tc5: M=%d N=%d too large", M, N);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * share));
  cfg.blockDim = dim3(THREADS4);
  cfg.dynamicSmemBytes = S::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = fg_pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = share;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = share > 1 ? 2 : 1;
  const cudaError_t le = cudaLaunchKernelEx(&cfg, kern, w_map, x_map, (const __nv_bfloat16*)scales, (TO*)y, ldy, M, N, K, share,
                                            m_tiles, epi, status);
  FG_CHECK_ARG(le == cudaSuccess, "fg_gemm_w4_tc5: launch failed: %s", cudaGetErrorString(le));
  return 0;
}

// How many blocks share a tile: as many as give every SM one, each with a stage of codes or more; a second block an SM only
// where they keep four stages each.  (us by blocks a tile, 16 tokens: 4,096 x 4,096 2 / 4 / 8: 10.6 / 6.8 / 8.1; 4,096 x 14,336
// 28.3 / 16.0 / 15.4; 6,144 x 4,096 10.7 / 9.8 / 11.3; 28,672 x 4,096 1 / 2: 25.3 / 30.7.)
template <typename S>
int share_of(int M, int N, int K) {
  const long tiles = (long)((M + S::T - 1) / S::T) * ((N + ROWS4 - 1) / ROWS4);
  const int stages = (K + W_COLS - 1) / W_COLS, sms = fg_sm_count();
  int share = 1;
  while (share < 8 && ((tiles * share * 2 <= sms && stages >= share * 2) ||
                       (tiles * share * 2 <= (long)S::BLOCKS * sms && stages >= share * 8)))
    share *= 2;
  return share;
}

template <int G, typename TO>
int choose(const void* x, int ldx, const void* w, const void* scales, void* y, int ldy, int M, int N, int K,
           const Epilogue4& epi, int* status, cudaStream_t stream) {
#define FG_W4(T)                                                                                                       \
  return launch<Shape4<T, G>, TO>(x, ldx, w, scales, y, ldy, M, N, K, share_of<Shape4<T, G>>(M, N, K), epi, status, stream)
  if (M <= 16) FG_W4(16);
  if (M <= 32) FG_W4(32);
  if (M <= 64 || G == 32) FG_W4(64);
  if constexpr (G > 32) FG_W4(128);
#undef FG_W4
  return -1;
}

template <typename TO>
int by_group(int group, const void* x, int ldx, const void* w, const void* scales, void* y, int ldy, int M, int N, int K,
             const Epilogue4& epi, int* status, cudaStream_t stream) {
  if (group == 128) return choose<128, TO>(x, ldx, w, scales, y, ldy, M, N, K, epi, status, stream);
  if (group == 64) return choose<64, TO>(x, ldx, w, scales, y, ldy, M, N, K, epi, status, stream);
  return choose<32, TO>(x, ldx, w, scales, y, ldy, M, N, K, epi, status, stream);
}

}  // namespace

// Arguments as of fg_gemm_w4, any M.
extern "C" int fg_gemm_w4_tc5(const void* x, int ldx, const void* w, const void* scales, int group, void* y, int ldy,
                              int out_dtype, int M, int N, int K, const void* bias, int act, int gated, int* status,
                              cudaStream_t stream) {
  if (M == 0 || N == 0) return 0;
  FG_CHECK_ARG(group == 32 || group == 64 || group == 128, "fg_gemm_w4_tc5: groups of %d columns are not supported (32, 64, 128)",
               group);
  FG_CHECK_ARG(M > 0 && K > 0 && K % group == 0, "fg_gemm_w4_tc5: M=%d, K=%d with groups of %d", M, K, group);
  FG_CHECK_ARG(ldx % 8 == 0 && ldx >= K && ldy >= (gated ? N / 2 : N), "fg_gemm_w4_tc5: row strides %d and %d", ldx, ldy);
  FG_CHECK_ARG((((uintptr_t)x | (uintptr_t)w) & 15) == 0, "fg_gemm_w4_tc5: x and the codes must be 16-byte aligned");
  FG_CHECK_ARG(!gated || (N % 16 == 0 && bias == nullptr && out_dtype == FG_BF16), "fg_gemm_w4_tc5: a gated product of %d rows", N);
  FG_CHECK_ARG(act >= fg_skinny::ACT_NONE && act <= fg_skinny::ACT_RELU2, "fg_gemm_w4_tc5: unknown activation %d", act);
  const Epilogue4 epi{(const __nv_bfloat16*)bias, act, gated != 0};
  int rc;
  if (out_dtype == FG_BF16)
    rc = by_group<__nv_bfloat16>(group, x, ldx, w, scales, y, ldy, M, N, K, epi, status, stream);
  else if (out_dtype == FG_F32)
    rc = by_group<float>(group, x, ldx, w, scales, y, ldy, M, N, K, epi, status, stream);
  else
    FG_CHECK_ARG(false, "fg_gemm_w4_tc5: bad output dtype %d", out_dtype);
  if (rc) return rc;
  FG_CHECK_LAUNCH("fg_gemm_w4_tc5");
  return 0;
}
