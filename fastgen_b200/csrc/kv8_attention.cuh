// Attention of single tokens over the cache in 8 bits.
//
// The scheme of the 16-bit cache's persistent kernel: blocks stay on their SM and walk the (request, split of 128 keys,
// key/value head) items that exist; a producer warp streams codes through a ring of shared-memory slots, four consumer
// warps take 32 keys each, partials per split go to scratch and attention_combine_kernel merges them.  What differs is
// what 8 bits ask for:
//
//  * Codes become half precision on their way into a fragment, which is exact, by one conversion for two codes; bfloat16
//    operands would need four instructions for two.  Queries are bfloat16, whose range half precision does not have: a
//    head's query is multiplied by a power of two that brings its largest element to [2^14, 2^15), and the scores by its
//    inverse.  Elements 2^29 times smaller than the largest lose bits, the sum does not notice.
//  * A key's scale is a factor of its score.  A value's scale 2^f joins its weight, exponent to exponent: with s the base-2
//    score the weight of the second product is 2^(s + f - m), m the largest s + f, so that weights stay within half
//    precision whatever the pages' scales are, and the codes enter the product as they are.  The softmax's denominator is
//    the sum of 2^(s - m), taken apart.  Weights are held 2^15 times larger than their value (half precision then
//    reaches down to 2^-39 of the largest).
//  * A value word holds the codes of four neighbouring keys of one dimension, so that a conversion gives the pairs of keys
//    that an operand register wants.  Keys are dealt to the rows of the first product such that its result, transposed in
//    registers, has the same order: row r < 8 of a tile of 16 keys is key 4 (r / 2) + r % 2, row r + 8 that key + 2.
//
// Slots of pages behind the sequence's last position may hold anything, NaN codes of a former owner among it: their scores
// are masked and their value codes zeroed in shared memory before use.
#pragma once

#include <cuda.h>

#include "attention_mma.cuh"
#include "kv8.cuh"

namespace fg_kv8 {

using fg_mma::capped_score;
using fg_mma::mbar_arrive;
using fg_mma::mbar_arrive_expect;
using fg_mma::mbar_fence_init;
using fg_mma::mbar_init;
using fg_mma::mbar_wait;
using fg_mma::part_stride;
using fg_mma::smem_u32;

constexpr int SPLIT = fg_mma::DECODE_SPLIT;  // 128 key positions
constexpr int DECODE_THREADS = 160;          // 4 consumer warps + 1 producer warp
constexpr int CONSUMERS = 128;
constexpr int MAX_COLUMNS = 8;       // heads of a group that an item works on
constexpr int DECODE_MAX_SEQS = 4096;
constexpr float WEIGHT_SHIFT = 15.f;
constexpr int NO_PAGE = -1000;       // in an exponent's place

template <int HD>
__host__ __device__ constexpr int decode_slots() { return HD == 64 ? 6 : HD == 128 ? 4 : 2; }
template <int HD>
__host__ __device__ constexpr int decode_blocks_per_sm() { return HD == 64 ? 3 : 2; }
template <int HD>
__host__ __device__ constexpr int merge_ld() { return HD + 4; }

template <int HD>
inline size_t decode_smem_bytes(int group, int n_seqs) {
  const int columns = group < MAX_COLUMNS ? group : MAX_COLUMNS;
  // the ring, the merge buffer of the four warps (values, maxima, sums), positions and pair counts, alignment slack
  return (size_t)decode_slots<HD>() * SPLIT * HD + (size_t)4 * columns * merge_ld<HD>() * 4 + 2 * 4 * MAX_COLUMNS * 4 +
         (size_t)(2 * n_seqs + 1) * 4 + 1024;
}

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int c0, int c1, int c2, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t transposed_8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

// Shared memory holds a split's block in lines of 128 bytes, 16-byte pieces swizzled: piece c of line l is at c ^ (l & 7).
__device__ __forceinline__ int swizzled(int line, int piece) { return line * 128 + ((piece ^ (line & 7)) << 4); }

// The i-th 16-byte piece (of HD / 64) of a key's row that the lanes with lane % 4 == t load: such that eight lanes of two
// neighbouring keys meet eight different places.
template <int HD>
__device__ __forceinline__ int key_piece(int t, int i) {
  if constexpr (HD == 64) return t;
  else if constexpr (HD == 128) return 2 * t + i;
  else return 8 * (i >> 1) + ((t & 1) | ((t >> 1) << 2) | ((i & 1) << 1));
}
template <int HD>
__device__ __forceinline__ int key_offset(int key, int piece) {
  if constexpr (HD == 64) return swizzled(key >> 1, (key & 1) * 4 + piece);
  else return swizzled(key * (HD / 128) + (piece >> 3), piece & 7);
}
// The i-th 16-byte piece (of HD / 32) of a value group that the lanes with lane / 4 == g load: dimensions
// 4 (g + 8 i) .. + 3 of four keys
template <int HD>
__device__ __forceinline__ int value_offset(int group, int g, int i) { return swizzled(group * (HD / 32) + i, g); }

template <int HD, bool CHUNKS>
__global__ void __launch_bounds__(DECODE_THREADS, decode_blocks_per_sm<HD>())
kv8_decode_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, int layer,
                  const float* k_scales, const float* v_scales, const __nv_bfloat16* q, int q_stride,
                  const int* __restrict__ block_table, int table_width, int page_size, int n_pages,
                  const int* __restrict__ pos, const int* __restrict__ seq_req, const int* __restrict__ seq_tok, int n_seqs,
                  int n_heads, int n_kv_heads, int group, int window, float scale_log2, float cap_log2, float scale_by_cap,
                  float* __restrict__ scratch, long long max_pairs, int max_splits, int* status) {
  constexpr int SLOTS = decode_slots<HD>();
  constexpr int SLOT_BYTES = SPLIT * HD;
  constexpr int MLD = merge_ld<HD>();
  constexpr int KP = HD / 64, VP = HD / 32;  // 16-byte pieces a lane loads of a key's row and of a group of four values
  extern __shared__ unsigned char smem_unaligned[];
  unsigned char* ring = reinterpret_cast<unsigned char*>(((uintptr_t)smem_unaligned + 1023) & ~(uintptr_t)1023);
  const int columns = min(group, MAX_COLUMNS);
  float* wo = reinterpret_cast<float*>(ring + SLOTS * SLOT_BYTES);  // [4 warps][columns][MLD]
  float* wm = wo + 4 * columns * MLD;                               // [4][8] maxima
  float* wl = wm + 4 * MAX_COLUMNS;                                 // [4][8] sums
  int* s_pos = reinterpret_cast<int*>(wl + 4 * MAX_COLUMNS);        // [n_seqs] the token's position, -1: a padding lane
  int* s_cum = s_pos + n_seqs;                                      // [n_seqs + 1] (request, split) pairs before it
  __shared__ __align__(8) uint64_t full[SLOTS], empty[SLOTS];
  __shared__ int s_exp[SLOTS][SPLIT / 16];  // exponents of the slot's boxes
  __shared__ int gave_up;                   // set by a wait that ran out (see mbar_wait)

  pdl_trigger();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) {
    gave_up = 0;
    for (int i = 0; i < SLOTS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 4);  // one arrival a consumer warp
    }
    mbar_fence_init();
  }
  // positions, lists and block tables are inputs of the step: read while the kernel before this one finishes
  auto first_split = [&](int p) { return first_visible<CHUNKS>(p, window) / SPLIT; };
  auto n_splits = [&](int p) { return p < 0 ? 0 : min(p / SPLIT, max_splits - 1) - first_split(p) + 1; };
  for (int sq = tid; sq < n_seqs; sq += DECODE_THREADS) s_pos[sq] = seq_req[sq] < 0 ? -1 : pos[seq_tok[sq]];
  __syncthreads();
  if (warp == 0) {
    const int per_lane = (n_seqs + 31) / 32;
    const int lo = min(n_seqs, lane * per_lane), hi = min(n_seqs, lo + per_lane);
    int sum = 0;
    for (int sq = lo; sq < hi; ++sq) sum += n_splits(s_pos[sq]);
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    int run = incl - sum;
    for (int sq = lo; sq < hi; ++sq) {
      s_cum[sq] = run;
      run += n_splits(s_pos[sq]);
    }
    if (lane == 31) s_cum[n_seqs] = incl;
  }
  __syncthreads();

  const int box_rows = min(page_size, SPLIT);
  const int n_boxes = SPLIT / box_rows;
  int n_pairs = s_cum[n_seqs];
  if (n_pairs > max_pairs) {
    // the scratch was sized for fewer: report instead of writing past it
    if (tid == 0 && blockIdx.x == 0 && status) atomicOr(status, FG_STATUS_BAD_SPLITS);
    n_pairs = (int)max_pairs;
  }
  // items: (request, split) pair, key/value head, slice of up to eight heads of its group
  const int n_sub = (group + MAX_COLUMNS - 1) / MAX_COLUMNS;
  const long long total = (long long)n_pairs * n_kv_heads * n_sub;
  struct Item {
    int pair, seq, g, sub, p, k0, k_begin;
  };
  auto item_of = [&](long long item) {
    Item it;
    it.sub = (int)(item % n_sub);
    const long long r = item / n_sub;
    it.g = (int)(r % n_kv_heads);
    it.pair = (int)(r / n_kv_heads);
    int lo = 0, hi = n_seqs;  // the last request whose first pair is <= pair
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_cum[mid] <= it.pair) lo = mid; else hi = mid;
    }
    it.seq = lo;
    it.p = s_pos[lo];
    it.k0 = (first_split(it.p) + (it.pair - s_cum[lo])) * SPLIT;
    it.k_begin = first_visible<CHUNKS>(it.p, window);
    return it;
  };

  if (warp == 4) {
    // ================================ producer ================================
    // The step's own kernels write the page that holds the token's position (its cached entries may be rounded again at a
    // larger scale): splits that end before that page are loaded without waiting for them.
    bool waited = false;
    auto page_of = [&](const Item& it) {  // lane i: the page of box i of the item's split, or -1
      int page = -1;
      const int j0 = it.k0 + lane * box_rows;
      if (lane < n_boxes && j0 <= it.p && j0 + box_rows > it.k_begin) {
        const int logical = j0 / page_size;
        page = logical < table_width ? block_table[(size_t)seq_req[it.seq] * table_width + logical] : -1;
        if (page < 0 || page >= n_pages) {
          page = -1;
          if (status) atomicOr(status, FG_STATUS_BAD_PAGE);
        }
      }
      return page;
    };
    int n_fill = 0;  // an item's keys are fill 2i, its values fill 2i + 1
    Item it{};
    int page = -1;
    if ((long long)blockIdx.x < total) {
      it = item_of(blockIdx.x);
      page = page_of(it);
    }
    for (long long item = blockIdx.x; item < total; item += gridDim.x) {
      if (!waited && it.k0 + SPLIT > (it.p & ~(page_size - 1))) {
        pdl_wait();
        waited = true;
      }
      const size_t block = ((size_t)max(page, 0)) * n_kv_heads + it.g;
      const uint32_t ks = page >= 0 ? ld_global_4(k_scales + block) : 0u, vs = page >= 0 ? ld_global_4(v_scales + block) : 0u;
      // the next item's pages are on their way meanwhile
      Item next{};
      int next_page = -1;
      if (item + gridDim.x < total) {
        next = item_of(item + gridDim.x);
        next_page = page_of(next);
      }
      const unsigned valid = __ballot_sync(0xffffffffu, page >= 0);
      const int bytes = __popc(valid) * box_rows * HD;
      const int line0 = (it.k0 & (page_size - 1)) * HD / 128;  // 0 unless pages are longer than a split
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const int slot = n_fill % SLOTS;
        if (n_fill >= SLOTS) mbar_wait(&empty[slot], (n_fill / SLOTS - 1) & 1, status, &gave_up);
        if (lane < n_boxes) s_exp[slot][lane] = page >= 0 ? exponent_of_scale(__uint_as_float(kv ? vs : ks)) : NO_PAGE;
        __syncwarp();
        if (lane == 0) mbar_arrive_expect(&full[slot], bytes);
        __syncwarp();
        if (page >= 0)  // lane i issues box i's copy
          tma_load_3d(ring + slot * SLOT_BYTES + lane * box_rows * HD, kv ? &v_map : &k_map, 0, line0,
                      (int)(((size_t)layer * n_pages + page) * n_kv_heads + it.g), &full[slot]);
        ++n_fill;
      }
      it = next;
      page = next_page;
    }
    if (!waited) pdl_wait();
  } else {
    // ================================ consumers ================================
    pdl_wait();
    int n_item = 0;
    const int g8 = lane >> 2, t4 = lane & 3;
    for (long long item = blockIdx.x; item < total; item += gridDim.x) {
      const Item it = item_of(item);
      const int heads = min(MAX_COLUMNS, group - it.sub * MAX_COLUMNS);
      const int head0 = it.g * group + it.sub * MAX_COLUMNS;
      // the queries as the 8-column operand: column lane / 4 is a head, its elements in the order of the keys' pieces
      uint32_t qb[KP][4][2];
      float unscale;  // of head g8
      {
        const __nv_bfloat16* row = q + (size_t)seq_tok[it.seq] * q_stride + (head0 + min(g8, heads - 1)) * HD;
        uint4 raw[KP][2];
#pragma unroll
        for (int i = 0; i < KP; ++i) {
          raw[i][0] = ld_global_16(row + 16 * key_piece<HD>(t4, i));
          raw[i][1] = ld_global_16(row + 16 * key_piece<HD>(t4, i) + 8);
        }
        uint32_t top = 0;  // the largest magnitude's bits: bfloat16 order is the order of its bits
#pragma unroll
        for (int i = 0; i < KP; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t w[4] = {raw[i][h].x, raw[i][h].y, raw[i][h].z, raw[i][h].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) top = __vmaxu2(top, w[j] & 0x7fff7fffu);
          }
        int big = max(top & 0xffffu, top >> 16);
        big = max(big, __shfl_xor_sync(0xffffffffu, big, 1));
        big = max(big, __shfl_xor_sync(0xffffffffu, big, 2));
        const int up = min(14 - ((big >> 7) - 127), 126);  // power of two that the query is multiplied by
        const float f = exp2_int(up);
        unscale = exp2_int(-up);
#pragma unroll
        for (int i = 0; i < KP; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t w[4] = {raw[i][h].x, raw[i][h].y, raw[i][h].z, raw[i][h].w};
#pragma unroll
            for (int j = 0; j < 4; ++j)
              qb[i][2 * h + (j >> 1)][j & 1] =
                  g8 < heads ? pack_f16(__uint_as_float(w[j] << 16) * f, __uint_as_float(w[j] & 0xffff0000u) * f) : 0u;
          }
      }
      // of the two heads whose scores this thread gets
      const float un[2] = {__shfl_sync(0xffffffffu, unscale, 8 * t4), __shfl_sync(0xffffffffu, unscale, 8 * t4 + 4)};
      const int fk = 2 * n_item, fv = fk + 1;
      const int slot_k = fk % SLOTS, slot_v = fv % SLOTS;
      const unsigned char* Ks = ring + slot_k * SLOT_BYTES;
      unsigned char* Vs = ring + slot_v * SLOT_BYTES;

      // S^T[keys, heads] = K Q^T for this warp's 32 keys
      mbar_wait(&full[slot_k], (fk / SLOTS) & 1, status, &gave_up);
      float s[2][4];
      int ek[2];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        ek[mt] = s_exp[slot_k][(warp * 32 + mt * 16) / box_rows];
        s[mt][0] = s[mt][1] = s[mt][2] = s[mt][3] = 0.f;
        const int key = warp * 32 + mt * 16 + 4 * (g8 >> 1) + (g8 & 1);
#pragma unroll
        for (int i = 0; i < KP; ++i) {
          const int piece = key_piece<HD>(t4, i);
          const uint4 a = *reinterpret_cast<const uint4*>(Ks + key_offset<HD>(key, piece));
          const uint4 b = *reinterpret_cast<const uint4*>(Ks + key_offset<HD>(key + 2, piece));
          const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, bw[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
          for (int m = 0; m < 4; ++m)
            mma_f16(s[mt], halves_of_low(aw[m]), halves_of_low(bw[m]), halves_of_high(aw[m]), halves_of_high(bw[m]),
                    qb[i][m][0], qb[i][m][1]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[slot_k]);  // this warp is done with the keys

      // this thread's scores: keys of row g8 and that + 2, heads 2 t4 and 2 t4 + 1
      mbar_wait(&full[slot_v], (fv / SLOTS) & 1, status, &gave_up);
      float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
      float fe[2];
      const bool edge = it.k0 + warp * 32 < it.k_begin || it.k0 + warp * 32 + 31 > it.p || ek[0] == NO_PAGE || ek[1] == NO_PAGE;
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        const int ev = s_exp[slot_v][(warp * 32 + mt * 16) / box_rows];
        fe[mt] = (float)ev;
        const float ks = exp2_int(max(ek[mt], -126));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float raw = s[mt][e] * un[e & 1] * ks;
          float sc = capped_score(raw, scale_log2, cap_log2, scale_by_cap);
          if (edge) {
            const int j = it.k0 + warp * 32 + mt * 16 + 4 * (g8 >> 1) + (g8 & 1) + (e & 2);
            if (j < it.k_begin || j > it.p || ek[mt] == NO_PAGE) sc = -INFINITY;
          }
          s[mt][e] = sc;
          top[e & 1] = fmaxf(top[e & 1], sc + fe[mt]);
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], o));
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float m = top[e & 1];
          const float x = s[mt][e] == -INFINITY ? -INFINITY : s[mt][e] - m + WEIGHT_SHIFT;  // (m may be -inf: a NaN stays one)
          sum[e & 1] += ex2(x);
          s[mt][e] = ex2(x + fe[mt]);
        }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], o);
      // the weights as the 8-column operand: an 8 x 8 transposition in registers for each half tile
      uint32_t pb[2][2];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        pb[mt][0] = transposed_8x8(pack_f16(s[mt][0], s[mt][1]));
        pb[mt][1] = transposed_8x8(pack_f16(s[mt][2], s[mt][3]));
      }
      if (edge) {
        // codes of keys that are not seen: zero (a weight of zero times a NaN would be a NaN)
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          const int grp = warp * 8 + mt * 4 + t4;
          uint32_t mask = 0;
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const int j = it.k0 + 4 * grp + b;
            if (j >= it.k_begin && j <= it.p && ek[mt] != NO_PAGE) mask |= 0xffu << (8 * b);
          }
#pragma unroll
          for (int i = 0; i < VP; ++i) {
            uint4* at = reinterpret_cast<uint4*>(Vs + value_offset<HD>(grp, g8, i));
            uint4 w = *at;
            w.x &= mask, w.y &= mask, w.z &= mask, w.w &= mask;
            *at = w;
          }
        }
        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");  // the slot's next copy comes behind these stores
      }

      // O^T[dims, heads] = V^T P^T
      float o[VP][2][4];
#pragma unroll
      for (int i = 0; i < VP; ++i) {
#pragma unroll
        for (int h = 0; h < 2; ++h) o[i][h][0] = o[i][h][1] = o[i][h][2] = o[i][h][3] = 0.f;
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          // dimensions 4 (g8 + 8 i) + 0..3 of the four keys of group t4 of the tile
          const uint4 w = *reinterpret_cast<const uint4*>(Vs + value_offset<HD>(warp * 8 + mt * 4 + t4, g8, i));
          mma_f16(o[i][0], halves_of_low(w.x), halves_of_low(w.y), halves_of_high(w.x), halves_of_high(w.y), pb[mt][0], pb[mt][1]);
          mma_f16(o[i][1], halves_of_low(w.z), halves_of_low(w.w), halves_of_high(w.z), halves_of_high(w.w), pb[mt][0], pb[mt][1]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[slot_v]);  // ... and with the values

      // merge the four warps (heads of the item only)
      if (g8 == 0) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          wm[warp * MAX_COLUMNS + 2 * t4 + h] = top[h];
          wl[warp * MAX_COLUMNS + 2 * t4 + h] = sum[h];
        }
      }
#pragma unroll
      for (int i = 0; i < VP; ++i)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int head = 2 * t4 + c;
          // rows g8 and g8 + 8 of the two products are neighbouring dimensions
          if (head < heads)
            *reinterpret_cast<float4*>(wo + (warp * columns + head) * MLD + 4 * (g8 + 8 * i)) =
                make_float4(o[i][0][c], o[i][0][2 + c], o[i][1][c], o[i][1][2 + c]);
        }
      asm volatile("bar.sync 1, %0;\n" ::"n"(CONSUMERS) : "memory");
      for (int i = tid; i < heads * HD; i += CONSUMERS) {
        const int r = i / HD, d = i - r * HD;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) mm = fmaxf(mm, wm[w * MAX_COLUMNS + r]);
        float acc = 0.f, ll = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float mw = wm[w * MAX_COLUMNS + r];
          const float f = (mw == -INFINITY) ? 0.f : ex2(mw - mm);
          acc += f * wo[(w * columns + r) * MLD + d];
          ll += f * wl[w * MAX_COLUMNS + r];
        }
        float* dst = scratch + ((size_t)it.pair * n_heads + head0 + r) * part_stride<HD>();
        dst[d] = acc;
        if (d == 0) {
          dst[HD] = mm - WEIGHT_SHIFT;
          dst[HD + 1] = ll;
        }
      }
      asm volatile("bar.sync 1, %0;\n" ::"n"(CONSUMERS) : "memory");  // the merge buffer is free again
      ++n_item;
    }
  }
}

}  // namespace fg_kv8
