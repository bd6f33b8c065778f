// Matrix product of a few tokens with 4-bit weights:
//   y[M, N] = x[M, K] * W[N, K]^T,   W[n, k] = (code[n, k] - 8) * scale[n, k / G],   G = 32, 64 or 128,
// x bfloat16, float32 accumulation, M <= 8.  (gemm_w4_tc5.cu has more tokens.)
//
// Bound by reading the codes once, half a byte a weight.  As in gemm_skinny.cu, 16 rows of W are the "M" side of
// mma.sync m16n8k16 and 8 tokens its "N" side, a thread streams its own pieces through a ring of cp.async stages that only it
// reads back, and the eight warps of a block, or of each block of a cluster, split K in chunks of 128 that are summed in a fixed order.
//  * A 32-bit word holds eight columns of a row, the even columns in its low half's nibbles and the odd ones in its
//    high half's: the nibbles at bit 4 i of both halves are columns 2 i and 2 i + 1, so that one `and-or` with 0x4300 (128 in
//    bfloat16, whose last bit is then 1) makes the pair 128 + code of an operand register and one subtraction code - 8: 11
//    instructions for eight weights, all of them exact.
//  * The weights enter the product as the whole numbers they are; a group's sums are multiplied by the group's scale in
//    float32 on their way into the accumulators.  Nothing is rounded to 16 bits but the result.
//  * What it spends (28,672 x 4,096, one token, 19 us): the copies alone take 11.4, the products and scales add the rest; two
//    blocks an SM do not hide all of one another's waits.
//  * In a chunk a lane takes 32 neighbouring columns (one 16-byte piece a row).  Groups of 32 and 64 columns must not meet in
//    one instruction: there the four lanes of a row take a word each of the same 32 columns, four pieces of four bytes.
//    (28,672 x 4,096, one token: groups of 128 20 us, 64 41, 32 55; weights in 16 bits 37.)
#include "gemm_w4.cuh"

namespace {

using namespace fg_skinny;
using namespace fg_w4;

constexpr int KCHUNK = 128;  // columns a warp takes at a time
constexpr int TOKENS = 8;
constexpr int MAX_SHARE = 4;  // blocks of a cluster that split K

__device__ __forceinline__ void cp_async_4(void* dst, const void* src, bool pred) {
  const int bytes = pred ? 4 : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes) : "memory");
}

// RT tiles of 16 rows a block; G columns a group
template <int RT_, int G_>
struct Plan4 {
  static constexpr int RT = RT_, G = G_;
  static constexpr int PIECES = 2 * RT + 4;  // 16-byte pieces a thread copies per chunk: codes, x
  static constexpr int STAGES = PIECES <= 6 ? 4 : PIECES <= 8 ? 3 : 2;
  static constexpr size_t RING = (size_t)STAGES * PIECES * THREADS * 16;
  static constexpr size_t SUMS = (size_t)WARPS * RT * ROWS * TOKENS * 4;
  static constexpr size_t SMEM = RING + SUMS;
  static constexpr int BLOCKS = SMEM <= 75 * 1024 ? 3 : 2;  // an SM
};

template <typename P, typename TO>
__global__ void __launch_bounds__(THREADS, P::BLOCKS)
gemm_w4_kernel(const __nv_bfloat16* x, int ldx, const uint32_t* __restrict__ w, int ldw, const __nv_bfloat16* __restrict__ scales,
               int lds, TO* __restrict__ y, int ldy, int M, int N, int K, int share, Epilogue4 epi) {
  constexpr int RT = P::RT, PARTS = KCHUNK / P::G;  // groups of a chunk
  // Rows beyond N and tokens beyond M are read as the last ones and left out of the result; K is whole chunks where the
  // groups are (WHOLE), else columns beyond K are zeros.
  constexpr bool WHOLE = P::G == KCHUNK;
  extern __shared__ __align__(16) unsigned char ring_raw[];
  uint4* const ring = reinterpret_cast<uint4*>(ring_raw) + threadIdx.x;  // [STAGES][PIECES][THREADS]
  typedef float Sums[RT * ROWS][TOKENS];
  Sums* const red = reinterpret_cast<Sums*>(ring_raw + P::RING);  // [WARPS]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int rank = blockIdx.x % share, n0 = blockIdx.x / share * RT * ROWS;
  // chunk c is the cluster's warp c mod (8 share)'s: `mine` of them from `first` on, `step` apart
  const int n_chunks = (K + KCHUNK - 1) / KCHUNK, first = rank * WARPS + warp, step = share * WARPS;
  const int mine = first < n_chunks ? (n_chunks - first + step - 1) / step : 0;
  pdl_trigger();

  uint32_t w_row[2 * RT];
#pragma unroll
  for (int r = 0; r < 2 * RT; ++r)
    w_row[r] = (uint32_t)min(n0 + r * 8 + g, N - 1) * ldw + first * (KCHUNK / 8) + (WHOLE ? 4 * t : t);
  const uint32_t x_row = (uint32_t)min(g, M - 1) * ldx + first * KCHUNK + (WHOLE ? 32 * t : 8 * t);
  auto issue_w = [&](int i, uint4* slot) {
#pragma unroll
    for (int r = 0; r < 2 * RT; ++r) {
      if (WHOLE) {
        cp_async_16<false>(slot + r * THREADS, w + (w_row[r] + i * (step * (KCHUNK / 8))), true);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bool ok = (first + i * step) * KCHUNK + 32 * j + 8 * t < K;
          cp_async_4(reinterpret_cast<uint32_t*>(slot + r * THREADS) + j, w + (ok ? w_row[r] + i * (step * (KCHUNK / 8)) + 4 * j : 0u), ok);
        }
      }
    }
  };
  auto issue_x = [&](int i, uint4* slot) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool ok = WHOLE || (first + i * step) * KCHUNK + 32 * j + 8 * t < K;
      cp_async_16<true>(slot + (2 * RT + j) * THREADS, x + (ok ? x_row + i * (step * KCHUNK) + (WHOLE ? 8 * j : 32 * j) : 0u), ok);
    }
  };
  // the scales of a chunk: rows g + 8 r of the tiles, its groups
  auto fetch_scales = [&](int i, __nv_bfloat16 (&s)[2 * RT][PARTS]) {
#pragma unroll
    for (int r = 0; r < 2 * RT; ++r)
#pragma unroll
      for (int p = 0; p < PARTS; ++p) {
        const bool ok = i < mine && (WHOLE || (first + i * step) * KCHUNK + p * P::G < K);
        const uint32_t at = (uint32_t)min(n0 + r * 8 + g, N - 1) * lds + (first + i * step) * PARTS + p;
        s[r][p] = ok ? scales[at] : __float2bfloat16_rn(0.f);
      }
  };

  // codes and scales depend on nothing that is computed in the step: on their way before the wait
#pragma unroll
  for (int s = 0; s < P::STAGES - 1; ++s)
    if (s < mine) issue_w(s, ring + s * P::PIECES * THREADS);
  __nv_bfloat16 sc[2 * RT][PARTS];
  fetch_scales(0, sc);
  pdl_wait();
#pragma unroll
  for (int s = 0; s < P::STAGES - 1; ++s) {
    if (s < mine) issue_x(s, ring + s * P::PIECES * THREADS);
    cp_async_commit();
  }

  float acc[RT][4];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[rt][e] = 0.f;
  int stage = 0, free = P::STAGES - 1;
  for (int i = 0; i < mine; ++i) {
    if (i + P::STAGES - 1 < mine) {
      issue_w(i + P::STAGES - 1, ring + free * P::PIECES * THREADS);
      issue_x(i + P::STAGES - 1, ring + free * P::PIECES * THREADS);
    }
    cp_async_commit();
    free = free + 1 == P::STAGES ? 0 : free + 1;
    __nv_bfloat16 next[2 * RT][PARTS];
    fetch_scales(i + 1, next);
    cp_async_wait<P::STAGES - 1>();  // this thread's copies of the chunk have landed; only it reads them
    const uint4* slot = ring + stage * P::PIECES * THREADS;
    stage = stage + 1 == P::STAGES ? 0 : stage + 1;
    uint4 b[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) b[j] = slot[(2 * RT + j) * THREADS];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const uint4 lo = slot[(2 * rt) * THREADS], hi = slot[(2 * rt + 1) * THREADS];
      const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
      for (int p = 0; p < PARTS; ++p) {
        float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = p * 4 / PARTS; j < (p + 1) * 4 / PARTS; ++j) {
          mma(part, weights_of(wl[j], 0), weights_of(wh[j], 0), weights_of(wl[j], 1), weights_of(wh[j], 1), b[j].x, b[j].y);
          mma(part, weights_of(wl[j], 2), weights_of(wh[j], 2), weights_of(wl[j], 3), weights_of(wh[j], 3), b[j].z, b[j].w);
        }
        const float s_lo = __bfloat162float(sc[2 * rt][p]), s_hi = __bfloat162float(sc[2 * rt + 1][p]);
        acc[rt][0] = fmaf(part[0], s_lo, acc[rt][0]);
        acc[rt][1] = fmaf(part[1], s_lo, acc[rt][1]);
        acc[rt][2] = fmaf(part[2], s_hi, acc[rt][2]);
        acc[rt][3] = fmaf(part[3], s_hi, acc[rt][3]);
      }
    }
#pragma unroll
    for (int r = 0; r < 2 * RT; ++r)
#pragma unroll
      for (int p = 0; p < PARTS; ++p) sc[r][p] = next[r][p];
  }
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    float* at = &red[warp][rt * ROWS + g][2 * t];
    *reinterpret_cast<float2*>(at) = make_float2(acc[rt][0], acc[rt][1]);
    *reinterpret_cast<float2*>(at + 8 * TOKENS) = make_float2(acc[rt][2], acc[rt][3]);
  }
  __syncthreads();
  // the block's warps in turn; then, over distributed shared memory, the cluster's blocks
  float* const part = reinterpret_cast<float*>(ring_raw);  // [RT * ROWS * TOKENS]: every warp has read its copies by now
  if (share > 1) {
    for (int i = tid; i < RT * ROWS * TOKENS; i += THREADS) {
      float v = 0.f;
#pragma unroll
      for (int wi = 0; wi < WARPS; ++wi) v += (&red[wi][0][0])[i];
      part[i] = v;
    }
    cluster_sync();
  }
  auto sum = [&](int row, int tok) {
    float v = 0.f;
    if (share == 1) {
#pragma unroll
      for (int wi = 0; wi < WARPS; ++wi) v += red[wi][row][tok];
    } else {
      const uint32_t at = smem_u32(part + row * TOKENS + tok);
      float p[MAX_SHARE];
#pragma unroll
      for (int b = 0; b < MAX_SHARE; ++b) p[b] = b < share ? ld_cluster(at, b) : 0.f;
#pragma unroll
      for (int b = 0; b < MAX_SHARE; ++b) v += p[b];
    }
    return v;
  };
  if (epi.gated) {
    for (int i = rank * THREADS + tid; i < RT * 8 * TOKENS; i += share * THREADS) {
      const int tok = i / (RT * 8), f = i - tok * (RT * 8), row = f / 8 * 16 + f % 8;
      if (tok < M && n0 + row + 8 < N) {
        // both are rounded to bfloat16 first, as a separate gate kernel would see them
        const float gr = __bfloat162float(__float2bfloat16_rn(sum(row, tok)));
        const float ur = __bfloat162float(__float2bfloat16_rn(sum(row + 8, tok)));
        y[(size_t)tok * ldy + n0 / 2 + f] = from_f32<TO>((epi.act ? fmaxf(gr, 0.f) : gr / (1.f + expf(-gr))) * ur);
      }
    }
  } else {
    for (int i = rank * THREADS + tid; i < RT * ROWS * TOKENS; i += share * THREADS) {
      const int tok = i / (RT * ROWS), row = i - tok * (RT * ROWS);  // consecutive threads write consecutive columns of y
      if (tok < M && n0 + row < N) {
        float v = sum(row, tok);
        if (epi.bias != nullptr) v += __bfloat162float(epi.bias[n0 + row]);
        // the product is rounded to bfloat16 before the activation, as a separate kernel would see it
        if (epi.act != ACT_NONE) v = activate(__bfloat162float(__float2bfloat16_rn(v)), epi.act);
        y[(size_t)tok * ldy + n0 + row] = from_f32<TO>(v);
      }
    }
  }
  if (share > 1) cluster_sync();  // nobody leaves while its sums are being read
}

template <typename P, typename TO>
int launch(const void* x, int ldx, const void* w, const void* scales, void* y, int ldy, int M, int N, int K, int share,
           const Epilogue4& epi, cudaStream_t stream) {
  auto kern = gemm_w4_kernel<P, TO>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)P::SMEM);
  FG_CHECK_ARG(e == cudaSuccess, "fg_gemm_w4: shared memory: %s", cudaGetErrorString(e));
  const int units = (N + P::RT * ROWS - 1) / (P::RT * ROWS);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(units * share));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = P::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = fg_pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = share;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = share > 1 ? 2 : 1;
  const cudaError_t le = cudaLaunchKernelEx(&cfg, kern, (const __nv_bfloat16*)x, ldx, (const uint32_t*)w, K / 8,
                                            (const __nv_bfloat16*)scales, K / P::G, (TO*)y, ldy, M, N, K, share, epi);
  FG_CHECK_ARG(le == cudaSuccess, "fg_gemm_w4: launch failed: %s", cudaGetErrorString(le));
  return 0;
}

// Blocks cost more than rows do: a call wants between one and two of them an SM, all resident at once, each with as many rows
// as that leaves, since the rows of a block share its copies of x.  Long rows are split over the blocks of a cluster, as long
// as each warp keeps two chunks.  us for 8 tokens, by row tiles a block / blocks a cluster (192 to 256 blocks in the first
// two of a line):
//   4,096 x 4,096: 2/2 5.8, 1/1 6.4, 4/1 9.9;  4,096 x 14,336: 4/4 14.0, 1/1 18.3, 4/1 28.7;  8,192 x 8,192: 4/2 13.1, 2/1 15.6,
//   4/1 20.7;  6,144 x 4,096: 4/2 8.6, 2/1 8.6, 1/1 10.0, 4/4 11.9;  14,336 x 4,096: 4/1 12.6, 2/1 16.5, 1/1 20.9.
template <int G, typename TO>
int choose(const void* x, int ldx, const void* w, const void* scales, void* y, int ldy, int M, int N, int K, const Epilogue4& epi,
           cudaStream_t stream) {
  const int tiles = (N + ROWS - 1) / ROWS, chunks = (K + KCHUNK - 1) / KCHUNK, sms = fg_sm_count();
  int rt = 4, share;
  for (;; rt /= 2) {
    const int units = (tiles + rt - 1) / rt;
    share = 1;
    while (share < MAX_SHARE && units * share * 2 <= 2 * sms && chunks >= 2 * WARPS * share * 2) share *= 2;
    if (rt == 1 || units * share >= sms) break;
  }
  if (rt == 4) return launch<Plan4<4, G>, TO>(x, ldx, w, scales, y, ldy, M, N, K, share, epi, stream);
  if (rt == 2) return launch<Plan4<2, G>, TO>(x, ldx, w, scales, y, ldy, M, N, K, share, epi, stream);
  return launch<Plan4<1, G>, TO>(x, ldx, w, scales, y, ldy, M, N, K, share, epi, stream);
}

template <typename TO>
int by_group(int group, const void* x, int ldx, const void* w, const void* scales, void* y, int ldy, int M, int N, int K,
             const Epilogue4& epi, cudaStream_t stream) {
  if (group == 128) return choose<128, TO>(x, ldx, w, scales, y, ldy, M, N, K, epi, stream);
  if (group == 64) return choose<64, TO>(x, ldx, w, scales, y, ldy, M, N, K, epi, stream);
  return choose<32, TO>(x, ldx, w, scales, y, ldy, M, N, K, epi, stream);
}

// The matrix in bfloat16, for products of many tokens: a thread eight columns.  Bound by its bytes: half of one read and two
// written a weight.
__global__ void __launch_bounds__(256)
dense_kernel(const uint32_t* __restrict__ w, const __nv_bfloat16* __restrict__ scales, int group_words, uint4* out, size_t words) {
  pdl_trigger();
  pdl_wait();  // the memory written may still be read by the kernels before
  const size_t step = (size_t)gridDim.x * blockDim.x;
  for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < words; i += step) {
    const uint32_t c = w[i];
    const __nv_bfloat162 s = __bfloat162bfloat162(scales[i / group_words]);
    uint32_t v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t x = weights_of(c, j);
      const __nv_bfloat162 y = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&x), s);
      v[j] = *reinterpret_cast<const uint32_t*>(&y);
    }
    out[i] = make_uint4(v[0], v[1], v[2], v[3]);
  }
}

}  // namespace

// out: bf16 [N, K], each weight rounded once
extern "C" int fg_w4_dense(const void* w, const void* scales, int group, void* out, int N, int K, cudaStream_t stream) {
  FG_CHECK_ARG((group == 32 || group == 64 || group == 128) && N > 0 && K > 0 && K % group == 0, "fg_w4_dense: N=%d, K=%d in groups of %d",
               N, K, group);
  FG_CHECK_ARG(((uintptr_t)out & 15) == 0 && ((uintptr_t)w & 3) == 0, "fg_w4_dense: unaligned");
  const size_t words = (size_t)N * (K / 8);
  const size_t blocks = (words + 255) / 256, most = (size_t)16 * fg_sm_count();
  fg_launch_pdl(dense_kernel, dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, stream, (const uint32_t*)w,
                (const __nv_bfloat16*)scales, group / 8, (uint4*)out, words);
  FG_CHECK_LAUNCH("fg_w4_dense");
  return 0;
}

// x: [M, K] bf16 (row stride ldx); w: codes [N, K / 8] words (see above); scales: bf16 [N, K / group]; y: [M, N] bf16 or float32,
// or with `gated` [M, N / 2] bf16: silu (relu with act 1) of the gate rows times the up rows, which lie in blocks of 8 in
// turn.  bias: bf16 [N] or null, added to the sums; act: ACT_* applied after it.
extern "C" int fg_gemm_w4(const void* x, int ldx, const void* w, const void* scales, int group, void* y, int ldy, int out_dtype,
                          int M, int N, int K, const void* bias, int act, int gated, cudaStream_t stream) {
  if (M == 0 || N == 0) return 0;
  FG_CHECK_ARG(M <= TOKENS, "fg_gemm_w4: M=%d exceeds %d", M, TOKENS);
  FG_CHECK_ARG(group == 32 || group == 64 || group == 128, "fg_gemm_w4: groups of %d columns are not supported (32, 64, 128)", group);
  FG_CHECK_ARG(K > 0 && K % group == 0, "fg_gemm_w4: K=%d is no multiple of the group of %d", K, group);
  FG_CHECK_ARG(ldx % 8 == 0 && ldx >= K && ldy >= (gated ? N / 2 : N), "fg_gemm_w4: row strides %d and %d", ldx, ldy);
  FG_CHECK_ARG((long long)N * (K / 8) < (1ll << 32) && (long long)M * ldx < (1ll << 32), "fg_gemm_w4: N=%d K=%d too large", N, K);
  FG_CHECK_ARG((((uintptr_t)x | (uintptr_t)w) & 15) == 0, "fg_gemm_w4: x and the codes must be 16-byte aligned");
  FG_CHECK_ARG(!gated || (N % 16 == 0 && bias == nullptr && out_dtype == FG_BF16), "fg_gemm_w4: a gated product of %d rows", N);
  FG_CHECK_ARG(act >= ACT_NONE && act <= ACT_RELU2, "fg_gemm_w4: unknown activation %d", act);
  const Epilogue4 epi{(const __nv_bfloat16*)bias, act, gated != 0};
  int rc;
  if (out_dtype == FG_BF16)
    rc = by_group<__nv_bfloat16>(group, x, ldx, w, scales, y, ldy, M, N, K, epi, stream);
  else if (out_dtype == FG_F32)
    rc = by_group<float>(group, x, ldx, w, scales, y, ldy, M, N, K, epi, stream);
  else
    FG_CHECK_ARG(false, "fg_gemm_w4: bad output dtype %d", out_dtype);
  if (rc) return rc;
  FG_CHECK_LAUNCH("fg_gemm_w4");
  return 0;
}
