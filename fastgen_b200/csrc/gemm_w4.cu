// Matrix product of a few tokens with 4-bit weights:
//   y[M, N] = x[M, K] * W[N, K]^T,   W[n, k] = (code[n, k] - 8) * scale[n, k / G],   G = 32, 64 or 128,
// x bfloat16, float32 accumulation, M <= 16.  (gemm_w4_tc5.cu has more tokens.)
//
// Bound by reading the codes once, half a byte a weight.  As in gemm_skinny.cu, 16 rows of W are the "M" side of
// mma.sync m16n8k16 and 8 tokens its "N" side, a thread streams its own pieces through a ring of cp.async stages that only it
// reads back, and the block's eight warps split K in chunks of 128 that are summed in warp order at the end.
//  * A 32-bit word holds eight columns of a row, the even columns in its low half's nibbles and the odd ones in its
//    high half's: the nibbles at bit 4 i of both halves are columns 2 i and 2 i + 1, so that one `and-or` with 0x4300 (128 in
//    bfloat16, whose last bit is then 1) makes the pair 128 + code of an operand register and one subtraction code - 8: 11
//    instructions for eight weights, all of them exact.
//  * The weights enter the product as the whole numbers they are; a group's sums are multiplied by the group's scale in
//    float32 on their way into the accumulators.  Nothing is rounded to 16 bits but the result.
//  * In a chunk a lane takes 32 neighbouring columns (one 16-byte piece a row).  Groups of 32 and 64 columns must not meet in
//    one instruction: there the four lanes of a row take a word each of the same 32 columns, four pieces of four bytes.
#include "skinny_product.cuh"

namespace {

using namespace fg_skinny;

constexpr int KCHUNK = 128;  // columns a warp takes at a time

__device__ __forceinline__ void cp_async_4(void* dst, const void* src, bool pred) {
  const int bytes = pred ? 4 : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes) : "memory");
}

// the columns 2 i and 2 i + 1 of a word's eight, as bfloat16
__device__ __forceinline__ uint32_t weights_of(uint32_t w, int i) {
  uint32_t v;
  asm("lop3.b32 %0, %1, 0x000f000f, 0x43004300, 0xea;\n" : "=r"(v) : "r"(w >> (4 * i)));  // (a & b) | c
  const uint32_t shift = 0x43084308u;  // 136
  const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), *reinterpret_cast<const __nv_bfloat162*>(&shift));
  return *reinterpret_cast<const uint32_t*>(&d);
}

// RT tiles of 16 rows and NT tiles of 8 tokens a block; G columns a group
template <int RT_, int NT_, int G_>
struct Plan4 {
  static constexpr int RT = RT_, NT = NT_, G = G_;
  static constexpr int PIECES = 2 * RT + 4 * NT;  // 16-byte pieces a thread copies per chunk
  static constexpr int STAGES = PIECES <= 6 ? 4 : PIECES <= 8 ? 3 : 2;
  static constexpr size_t RING = (size_t)STAGES * PIECES * THREADS * 16;
  static constexpr size_t SUMS = (size_t)WARPS * RT * ROWS * NT * 8 * 4;  // in the ring's memory once it is through
  static constexpr size_t SMEM = RING > SUMS ? RING : SUMS;
};

struct Epilogue4 {
  const __nv_bfloat16* bias;  // [N] or null
  int act;                    // ACT_*; with `gated`: 1 for a relu gate
  bool gated;                 // rows are gate and up in blocks of 8: y[M, N / 2]
};

template <typename P, typename TO>
__global__ void __launch_bounds__(THREADS)
gemm_w4_kernel(const __nv_bfloat16* x, int ldx, const uint32_t* __restrict__ w, int ldw, const __nv_bfloat16* __restrict__ scales,
               int lds, TO* __restrict__ y, int ldy, int M, int N, int K, Epilogue4 epi) {
  constexpr int RT = P::RT, NT = P::NT, PARTS = KCHUNK / P::G;  // groups of a chunk
  extern __shared__ __align__(16) unsigned char ring_raw[];
  uint4* ring = reinterpret_cast<uint4*>(ring_raw);  // [STAGES][PIECES][THREADS]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * (RT * ROWS);
  const int n_chunks = (K + KCHUNK - 1) / KCHUNK;
  const int mine = warp < n_chunks ? (n_chunks - warp + WARPS - 1) / WARPS : 0;
  pdl_trigger();

  auto issue_w = [&](int i) {
    uint4* slot = ring + (size_t)(i % P::STAGES) * P::PIECES * THREADS + tid;
    const int k = (warp + i * WARPS) * KCHUNK;
#pragma unroll
    for (int r = 0; r < 2 * RT; ++r) {
      const int n = n0 + r * 8 + g;
      const uint32_t* row = w + (size_t)min(n, N - 1) * ldw;
      if (P::G == KCHUNK) {
        const int at = k + 32 * t;
        cp_async_16<false>(slot + r * THREADS, row + (at < K ? at / 8 : 0), n < N && at < K);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int at = k + 32 * j + 8 * t;
          cp_async_4(reinterpret_cast<uint32_t*>(slot + r * THREADS) + j, row + (at < K ? at / 8 : 0), n < N && at < K);
        }
      }
    }
  };
  auto issue_x = [&](int i) {
    uint4* slot = ring + (size_t)(i % P::STAGES) * P::PIECES * THREADS + tid;
    const int k = (warp + i * WARPS) * KCHUNK;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int tok = nt * 8 + g;
      const __nv_bfloat16* row = x + (size_t)min(tok, M - 1) * ldx;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int at = k + (P::G == KCHUNK ? 32 * t + 8 * j : 32 * j + 8 * t);
        cp_async_16<true>(slot + (2 * RT + nt * 4 + j) * THREADS, row + (at < K ? at : 0), tok < M && at < K);
      }
    }
  };
  // the scales of a chunk: rows g + 8 r of the block, its groups
  auto fetch_scales = [&](int i, float (&s)[2 * RT][PARTS]) {
    const int k = (warp + i * WARPS) * KCHUNK;
#pragma unroll
    for (int r = 0; r < 2 * RT; ++r) {
      const int n = n0 + r * 8 + g;
#pragma unroll
      for (int p = 0; p < PARTS; ++p) {
        const int at = k + p * P::G;
        s[r][p] = i < mine && n < N && at < K ? __bfloat162float(scales[(size_t)n * lds + at / P::G]) : 0.f;
      }
    }
  };

  // weights and scales depend on nothing that is computed in the step: on their way before the wait
#pragma unroll
  for (int s = 0; s < P::STAGES - 1; ++s)
    if (s < mine) issue_w(s);
  float sc[2 * RT][PARTS];
  fetch_scales(0, sc);
  pdl_wait();
#pragma unroll
  for (int s = 0; s < P::STAGES - 1; ++s) {
    if (s < mine) issue_x(s);
    cp_async_commit();
  }
  float acc[RT][NT][4];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[rt][nt][e] = 0.f;

  for (int i = 0; i < mine; ++i) {
    if (i + P::STAGES - 1 < mine) {
      issue_w(i + P::STAGES - 1);
      issue_x(i + P::STAGES - 1);
    }
    cp_async_commit();
    float next[2 * RT][PARTS];
    fetch_scales(i + 1, next);
    cp_async_wait<P::STAGES - 1>();  // this thread's copies of chunk i have landed; only it reads them
    const uint4* slot = ring + (size_t)(i % P::STAGES) * P::PIECES * THREADS + tid;
    uint4 b[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 4; ++j) b[nt][j] = slot[(2 * RT + nt * 4 + j) * THREADS];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const uint4 lo = slot[(2 * rt) * THREADS], hi = slot[(2 * rt + 1) * THREADS];
      const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
      for (int p = 0; p < PARTS; ++p) {
        float part[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) part[nt][e] = 0.f;
#pragma unroll
        for (int j = p * 4 / PARTS; j < (p + 1) * 4 / PARTS; ++j) {
          const uint32_t a[4] = {weights_of(wl[j], 0), weights_of(wl[j], 1), weights_of(wl[j], 2), weights_of(wl[j], 3)};
          const uint32_t c[4] = {weights_of(wh[j], 0), weights_of(wh[j], 1), weights_of(wh[j], 2), weights_of(wh[j], 3)};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma(part[nt], a[0], c[0], a[1], c[1], b[nt][j].x, b[nt][j].y);
            mma(part[nt], a[2], c[2], a[3], c[3], b[nt][j].z, b[nt][j].w);
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          acc[rt][nt][0] = fmaf(part[nt][0], sc[2 * rt][p], acc[rt][nt][0]);
          acc[rt][nt][1] = fmaf(part[nt][1], sc[2 * rt][p], acc[rt][nt][1]);
          acc[rt][nt][2] = fmaf(part[nt][2], sc[2 * rt + 1][p], acc[rt][nt][2]);
          acc[rt][nt][3] = fmaf(part[nt][3], sc[2 * rt + 1][p], acc[rt][nt][3]);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < 2 * RT; ++r)
#pragma unroll
      for (int p = 0; p < PARTS; ++p) sc[r][p] = next[r][p];
  }
  cp_async_wait<0>();
  __syncthreads();  // the sums take the ring's memory
  typedef float Sums[RT * ROWS][NT * 8];
  Sums* red = reinterpret_cast<Sums*>(ring_raw);
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float* at = &red[warp][rt * ROWS + g][nt * 8 + 2 * t];
      at[0] = acc[rt][nt][0];
      at[1] = acc[rt][nt][1];
      at += 8 * NT * 8;
      at[0] = acc[rt][nt][2];
      at[1] = acc[rt][nt][3];
    }
  __syncthreads();
  auto total = [&](int row, int tok) {
    float s = 0.f;
#pragma unroll
    for (int wi = 0; wi < WARPS; ++wi) s += red[wi][row][tok];
    return s;
  };
  if (epi.gated) {
    for (int i = tid; i < RT * 8 * NT * 8; i += THREADS) {
      const int tok = i / (RT * 8), f = i - tok * (RT * 8), row = f / 8 * 16 + f % 8;
      if (tok < M && n0 + row + 8 < N) {
        // both are rounded to bfloat16 first, as a separate gate kernel would see them
        const float gr = __bfloat162float(__float2bfloat16_rn(total(row, tok)));
        const float ur = __bfloat162float(__float2bfloat16_rn(total(row + 8, tok)));
        y[(size_t)tok * ldy + n0 / 2 + f] = from_f32<TO>((epi.act ? fmaxf(gr, 0.f) : gr / (1.f + expf(-gr))) * ur);
      }
    }
    return;
  }
  for (int i = tid; i < RT * ROWS * NT * 8; i += THREADS) {
    const int tok = i / (RT * ROWS), row = i - tok * (RT * ROWS);  // consecutive threads write consecutive columns of y
    if (tok < M && n0 + row < N) {
      float v = total(row, tok);
      if (epi.bias != nullptr) v += __bfloat162float(epi.bias[n0 + row]);
      // the product is rounded to bfloat16 before the activation, as a separate kernel would see it
      if (epi.act != ACT_NONE) v = activate(__bfloat162float(__float2bfloat16_rn(v)), epi.act);
      y[(size_t)tok * ldy + n0 + row] = from_f32<TO>(v);
    }
  }
}

template <typename P, typename TO>
int launch(const void* x, int ldx, const void* w, const void* scales, void* y, int ldy, int M, int N, int K, const Epilogue4& epi,
           cudaStream_t stream) {
  auto kern = gemm_w4_kernel<P, TO>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)P::SMEM);
  FG_CHECK_ARG(e == cudaSuccess, "fg_gemm_w4: shared memory: %s", cudaGetErrorString(e));
  constexpr int R = P::RT * ROWS;
  fg_launch_pdl(kern, dim3((N + R - 1) / R), dim3(THREADS), P::SMEM, stream, (const __nv_bfloat16*)x, ldx, (const uint32_t*)w, K / 8,
                (const __nv_bfloat16*)scales, K / P::G, (TO*)y, ldy, M, N, K, epi);
  return 0;
}

template <int G, typename TO>
int choose(const void* x, int ldx, const void* w, const void* scales, void* y, int ldy, int M, int N, int K, const Epilogue4& epi,
           cudaStream_t stream) {
  const bool few = (N + ROWS - 1) / ROWS <= 2 * fg_sm_count();
  if (M <= 8)
    return few ? launch<Plan4<1, 1, G>, TO>(x, ldx, w, scales, y, ldy, M, N, K, epi, stream)
               : launch<Plan4<2, 1, G>, TO>(x, ldx, w, scales, y, ldy, M, N, K, epi, stream);
  return few ? launch<Plan4<1, 2, G>, TO>(x, ldx, w, scales, y, ldy, M, N, K, epi, stream)
             : launch<Plan4<2, 2, G>, TO>(x, ldx, w, scales, y, ldy, M, N, K, epi, stream);
}

template <typename TO>
int by_group(int group, const void* x, int ldx, const void* w, const void* scales, void* y, int ldy, int M, int N, int K,
             const Epilogue4& epi, cudaStream_t stream) {
  if (group == 128) return choose<128, TO>(x, ldx, w, scales, y, ldy, M, N, K, epi, stream);
  if (group == 64) return choose<64, TO>(x, ldx, w, scales, y, ldy, M, N, K, epi, stream);
  return choose<32, TO>(x, ldx, w, scales, y, ldy, M, N, K, epi, stream);
}

// The matrix in bfloat16, for products of many tokens: a thread eight columns.  Bound by its bytes: half of one read and two
// written a weight (28,672 x 4,096: FIGURE_X).
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

extern "C" int fg_gemm_w4_max_m() { return 16; }

// x: [M, K] bf16 (row stride ldx); w: codes [N, K / 8] words (see above); scales: bf16 [N, K / group]; y: [M, N] bf16 or float32,
// or with `gated` [M, N / 2] bf16: silu (relu with act 1) of the gate rows times the up rows, which lie in blocks of 8 in
// turn.  bias: bf16 [N] or null, added to the sums; act: ACT_* applied after it.
extern "C" int fg_gemm_w4(const void* x, int ldx, const void* w, const void* scales, int group, void* y, int ldy, int out_dtype,
                          int M, int N, int K, const void* bias, int act, int gated, cudaStream_t stream) {
  if (M == 0 || N == 0) return 0;
  FG_CHECK_ARG(M <= 16, "fg_gemm_w4: M=%d exceeds 16", M);
  FG_CHECK_ARG(group == 32 || group == 64 || group == 128, "fg_gemm_w4: groups of %d columns are not supported (32, 64, 128)", group);
  FG_CHECK_ARG(K > 0 && K % group == 0, "fg_gemm_w4: K=%d is no multiple of the group of %d", K, group);
  FG_CHECK_ARG(ldx % 8 == 0 && ldx >= K && ldy >= (gated ? N / 2 : N), "fg_gemm_w4: row strides %d and %d", ldx, ldy);
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
