// Attention of single tokens over the cache in 8 bits.
//
// Blocks stay on their SM and walk the (request, key/value head, 128 keys) items that exist, each block a stretch of
// neighbours, an equal share of all.  The items of one request and head inside a block are one run: queries converted once,
// running maximum, sums and outputs in registers from item to item.  A run that holds all keys of its request is stored as the
// result; the others leave a partial (two a block at most), and the block whose partial of a request and head is counted last
// merges them in the order of the keys: one launch, nobody waits, the order of the sums is the walk's.  (A partial for
// every 128 keys and a merge in a launch of its own: 64 ragged requests of up to 2,800 keys, 32 / 8 heads of 128, 62.6 us
// against 45.7, batch 8 at 4,096 keys 21.1 against 17.7.)
// A producer warp streams codes through a ring of shared-memory slots ahead of four consumer warps.  In the first product a
// consumer warp has 32 keys; the weights go to shared memory, and in the second product it has a quarter of the dimensions
// of all 128 keys, so that there are no sums of warps to merge.
//
//  * Codes become half precision on their way into a fragment, which is exact, by one conversion for two codes; bfloat16
//    operands would need four instructions for two.  Queries are bfloat16, whose range half precision does not have: a
//    head's query is multiplied by a power of two that brings its largest element to [2^14, 2^15), and the scores by its
//    inverse.  Elements 2^29 times smaller than the largest lose bits, the sum does not notice.
//  * A key's scale is a factor of its score.  A value's scale 2^f joins its weight, exponent to exponent: with s the base-2
//    score the weight of the second product is 2^(s + f - m), m the largest s + f, so that weights stay within half
//    precision whatever the pages' scales are, and the codes enter the product as they are.  The softmax's denominator is
//    the sum of 2^(s - m), taken apart.  Weights are held 2^15 times larger than their value (half precision then
//    reaches down to 2^-39 of the largest); the denominator is not, for it lies between 2^-100 and 2^100 times the number
//    of keys (a value's scale is 2^-100 at the least and 2^100 at the most), within float32 for up to 2^27 keys.  Where scales
//    lie far apart, what brings a denominator to a new maximum is applied in two halves: 2^100 times 2^-200 is 2^-100.
//  * A value word holds the codes of four neighbouring keys of one dimension, so that a conversion gives the pairs of keys
//    that an operand register wants.  Keys are dealt to the rows of the first product such that its result, transposed in
//    registers, has the same order: row r < 8 of a tile of 16 keys is key 4 (r / 2) + r % 2, row r + 8 that key + 2.
//
// Slots of pages behind the sequence's last position may hold anything, NaN codes of a former owner among it: their scores
// are masked and their value codes zeroed in shared memory before use.
#pragma once

#include <cuda.h>

#include <type_traits>

#include "attention_mma.cuh"
#include "kv8.cuh"

namespace fg_kv8 {

using fg_mma::capped_score;
using fg_mma::mbar_arrive;
using fg_mma::mbar_fence_init;
using fg_mma::mbar_init;
using fg_mma::mbar_wait;
using fg_mma::smem_u32;

constexpr int SPLIT = 128;                   // key positions of an item
constexpr int DECODE_THREADS = 160;          // 4 consumer warps + 1 producer warp
constexpr int CONSUMERS = 128;
constexpr int MAX_COLUMNS = 8;       // heads of a group that an item works on
constexpr int DECODE_MAX_SEQS = 4096;
constexpr int WEIGHT_SHIFT = 15;
constexpr float WEIGHT_UNIT = 1.f / (1 << WEIGHT_SHIFT);
constexpr int SCALES_NEAR = 64;      // exponents of values' scales this close take the short way to a denominator
constexpr int NO_PAGE = -1000;       // in an exponent's place

// As many slots as an SM's blocks have room for.  (Fewer, 4 / 3 / 2, or eight of the smallest: every case within 2 %.)
template <int HD>
__host__ __device__ constexpr int decode_slots() { return HD == 64 ? 6 : HD == 128 ? 4 : 3; }
template <int HD>
__host__ __device__ constexpr int decode_blocks_per_sm() { return HD <= 128 ? 3 : 2; }
template <int HD>
__host__ __device__ constexpr int run_stride() { return HD + 4; }  // a run's partial of one head: outputs, maximum, sum

template <int HD>
inline size_t decode_smem_bytes(int n_seqs) {
  // the ring, positions and pair counts, alignment slack
  return (size_t)decode_slots<HD>() * SPLIT * HD + (size_t)(2 * n_seqs + 1) * 4 + 1024;
}

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int c0, int c1, int c2, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar))
      : "memory");
}

// bytes that a barrier's phase waits for, without an arrival
__device__ __forceinline__ void mbar_expect(uint64_t* bar, int bytes) {
  asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;\n" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
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

// ... down to float32's subnormal numbers
__device__ __forceinline__ float ex2_subnormal(float x) {
  float y;
  asm("ex2.approx.f32 %0, %1;\n" : "=f"(y) : "f"(x));
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

// What outputs relative to the base-2 maximum `top` are multiplied by, next to WEIGHT_UNIT: one over the sum of the weights,
// of which the head's sink (in natural units) is one more without a key.
__device__ __forceinline__ float finish(float top, float sum, const float* sinks, int head) {
  if (sinks == nullptr) return sum > 0.f || sum != sum ? 1.f / sum : 0.f;
  const float sink = sinks[head] * 1.4426950408889634f, m = fmaxf(top, sink);
  const float half = top == -INFINITY ? 0.f : ex2(0.5f * (top - m));
  return half * half / (sum * half * half + ex2(sink - m));
}

// Two neighbouring outputs, turned by position * frequency of their pair where a table is given.
__device__ __noinline__ float2 turned_pair(float a, float b, float freq, int p) {
  float sn, cs;
  sincosf((float)p * freq, &sn, &cs);
  return make_float2(a * cs - b * sn, b * cs + a * sn);
}
__device__ __forceinline__ void store_pair(__nv_bfloat16* dst, float a, float b, const float* freqs, int pair, int p) {
  if (freqs != nullptr) {
    const float2 v = turned_pair(a, b, freqs[pair], p);
    a = v.x;
    b = v.y;
  }
  *reinterpret_cast<__nv_bfloat162*>(dst) = __floats2bfloat162_rn(a, b);
}

template <int HD, bool CHUNKS, bool CAPPED>
__global__ void __launch_bounds__(DECODE_THREADS, decode_blocks_per_sm<HD>())
kv8_decode_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, int layer,
                  const float* k_scales, const float* v_scales, const __nv_bfloat16* q, int q_stride,
                  const int* __restrict__ block_table, int table_width, int page_size, int n_pages,
                  const int* __restrict__ pos, const int* __restrict__ seq_req, const int* __restrict__ seq_tok, int n_seqs,
                  int n_heads, int n_kv_heads, int group, int window, float scale_log2, float cap_log2, float scale_by_cap,
                  __nv_bfloat16* out, int out_stride, float* scratch, int* counters, const float* __restrict__ out_freqs,
                  const float* __restrict__ sinks, int* status) {
  constexpr int SLOTS = decode_slots<HD>();
  constexpr int SLOT_BYTES = SPLIT * HD;
  constexpr int KP = HD / 64;               // 16-byte pieces a lane loads of a key's row
  constexpr int VP = HD / 32;               // 16-byte pieces of a group of four values
  constexpr int TILES = SPLIT / 16;         // tiles of 16 keys
  constexpr int MINE = VP >= 4 ? VP / 4 : 1;  // pieces a warp has in the second product
  constexpr int HALVES = VP >= 4 ? 2 : 1;     // products (of 16 dimensions) of a piece: a warp has both, or one at HD = 64
  extern __shared__ unsigned char smem_unaligned[];
  unsigned char* ring = reinterpret_cast<unsigned char*>(((uintptr_t)smem_unaligned + 1023) & ~(uintptr_t)1023);
  int* s_pos = reinterpret_cast<int*>(ring + SLOTS * SLOT_BYTES);  // [n_seqs] the token's position, -1: a padding lane
  int* s_cum = s_pos + n_seqs;                                     // [n_seqs + 1] (request, split) pairs before it
  __shared__ __align__(8) uint64_t full[SLOTS], empty[SLOTS];
  __shared__ int s_exp[SLOTS][2][TILES];     // exponents of the keys' and the values' boxes, with the keys' slot
  __shared__ int s_apart[SLOTS];             // whether the values' scales of a run so far are far apart, with the keys' slot
  __shared__ __align__(8) uint2 s_weights[TILES][32];  // the second product's right operand
  __shared__ __align__(8) float s_top[4][MAX_COLUMNS], s_sum[4][MAX_COLUMNS];
  __shared__ __align__(16) int s_run[2][8];  // the block's partials: request, slice, token, position (-1: none), blocks from and to
  __shared__ int s_last[2];                  // ... and whether this block's was counted last
  __shared__ int gave_up;                    // set by a wait that ran out (see mbar_wait)

  pdl_trigger();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) {
    gave_up = 0;
    s_run[0][3] = s_run[1][3] = -1;
    for (int i = 0; i < SLOTS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 4);  // one arrival a consumer warp
    }
    mbar_fence_init();
  }
  // positions, lists and block tables are inputs of the step: read while the kernel before this one finishes
  auto first_split = [&](int p) { return first_visible<CHUNKS>(p, window) / SPLIT; };
  auto n_splits = [&](int p) { return p < 0 ? 0 : p / SPLIT - first_split(p) + 1; };
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
  const int n_boxes = SPLIT / box_rows, box_shift = 31 - __clz(box_rows), page_shift = 31 - __clz(page_size);
  // items: request, then (key/value head, slice of up to eight heads of its group), then split
  const int n_sub = (group + MAX_COLUMNS - 1) / MAX_COLUMNS, slices = n_kv_heads * n_sub;
  const long long total = (long long)s_cum[n_seqs] * slices;
  const int blocks = (int)min((long long)gridDim.x, total);  // that have items
  // (64-bit divisions take a few hundred cycles; what is divided fits 32 bits up to some ten million items)
  const bool narrow = (total + 1) * blocks < (1ll << 32);
  auto divided = [&](long long a, long long b) { return narrow ? (long long)((uint32_t)a / (uint32_t)b) : a / b; };
  auto begin_of = [&](int b) { return divided(total * b, blocks); };
  auto block_of = [&](long long item) { return (int)divided((item + 1) * blocks - 1, total); };
  const bool busy = (int)blockIdx.x < blocks;
  const long long begin = busy ? begin_of(blockIdx.x) : 0;
  const int count = busy ? (int)(begin_of(blockIdx.x + 1) - begin) : 0;
  struct Walk {
    int seq, slice, split, n, p, first, k_begin;  // split counts from `first`, the request's first one; n of them
  };
  auto enter = [&](Walk& w) {
    w.p = s_pos[w.seq];
    w.first = first_split(w.p);
    w.n = n_splits(w.p);
    w.k_begin = first_visible<CHUNKS>(w.p, window);
  };
  auto start = [&]() {
    Walk w{};
    if (count == 0) return w;
    int lo = 0, hi = n_seqs;  // the last request whose first item is <= begin
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if ((long long)s_cum[mid] * slices <= begin) lo = mid; else hi = mid;
    }
    w.seq = lo;
    enter(w);
    const int in = (int)(begin - (long long)s_cum[lo] * slices);
    w.slice = in / w.n;
    w.split = in - w.slice * w.n;
    return w;
  };
  // the next item; there is one
  auto advance = [&](Walk& w) {
    if (++w.split < w.n) return;
    w.split = 0;
    if (++w.slice < slices) return;
    w.slice = 0;
    do ++w.seq;
    while (s_cum[w.seq + 1] == s_cum[w.seq]);
    enter(w);
  };

  if (warp == 4) {
    // ================================ producer ================================
    auto page_of = [&](const Walk& w) {  // lane i: the page of box i of the item's split, or -1
      int page = -1;
      const int j0 = (w.first + w.split) * SPLIT + lane * box_rows;
      if (lane < n_boxes && j0 <= w.p && j0 + box_rows > w.k_begin) {
        const int logical = j0 >> page_shift;
        page = logical < table_width ? block_table[(size_t)seq_req[w.seq] * table_width + logical] : -1;
        if (page < 0 || page >= n_pages) {
          page = -1;
          if (status) atomicOr(status, FG_STATUS_BAD_PAGE);
        }
      }
      return page;
    };
    Walk w = start();
    int page = count > 0 ? page_of(w) : -1;
    // Any page may be what a kernel ahead has just written: nothing is loaded before those are over.  (Loading the splits
    // before the token's own page earlier saved 0.4 us of 7.4 for a short request, 1.9 of 50.6 for 64 ragged ones, and read
    // stale pages where a prompt's write is followed at once.)
    pdl_wait();
    int slot = 0, use = 0;
    int run_low = KV8_HIGHEST, run_top = KV8_LOWEST;  // exponents of the values' scales in the run so far
    for (int i = 0; i < count; ++i) {
      const int k0 = (w.first + w.split) * SPLIT, g = w.slice / n_sub, seq = w.seq, slice = w.slice;
      const size_t block = (size_t)max(page, 0) * n_kv_heads + g;
      const uint32_t ks = page >= 0 ? ld_global_4(k_scales + block) : 0u, vs = page >= 0 ? ld_global_4(v_scales + block) : 0u;
      const unsigned valid = __ballot_sync(0xffffffffu, page >= 0);
      const int bytes = __popc(valid) * box_rows * HD;
      const int line0 = (k0 & (page_size - 1)) * HD / 128;  // 0 unless pages are longer than a split
      const int k_slot = slot;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        if (use > 0) mbar_wait(&empty[slot], (use - 1) & 1, status, &gave_up);
        if (lane == 0) mbar_expect(&full[slot], bytes);
        __syncwarp();
        if (page >= 0)  // lane i issues box i's copy
          tma_load_3d(ring + slot * SLOT_BYTES + lane * box_rows * HD, kv ? &v_map : &k_map, 0, line0,
                      (int)(((size_t)layer * n_pages + page) * n_kv_heads + g), &full[slot]);
        if (++slot == SLOTS) {
          slot = 0;
          ++use;
        }
      }
      // the next item's pages and the scales come while the copies run; consumers read the scales behind the keys' arrival
      int next_page = -1;
      if (i + 1 < count) {
        advance(w);
        next_page = page_of(w);
      }
      const int ev = page >= 0 ? exponent_of_scale(__uint_as_float(vs)) : 0;
      if (lane < n_boxes) {
        s_exp[k_slot][0][lane] = page >= 0 ? exponent_of_scale(__uint_as_float(ks)) : NO_PAGE;
        s_exp[k_slot][1][lane] = ev;
      }
      run_low = min(run_low, __reduce_min_sync(0xffffffffu, page >= 0 ? ev : KV8_HIGHEST));
      run_top = max(run_top, __reduce_max_sync(0xffffffffu, page >= 0 ? ev : KV8_LOWEST));
      if (lane == 0) s_apart[k_slot] = run_top - run_low > SCALES_NEAR;
      if (w.seq != seq || w.slice != slice) run_low = KV8_HIGHEST, run_top = KV8_LOWEST;  // the next item begins a run
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&full[k_slot]);
        mbar_arrive(&full[k_slot + 1 == SLOTS ? 0 : k_slot + 1]);
      }
      page = next_page;
    }
    if (*reinterpret_cast<volatile int*>(&gave_up) != 0)
      // a wait ran out: the copies in flight land before the block leaves
      for (int f = max(0, 2 * count - SLOTS); f < 2 * count; ++f) mbar_wait(&full[f % SLOTS], f / SLOTS & 1, status);
  } else {
    // ================================ consumers ================================
    pdl_wait();
    const int g8 = lane >> 2, t4 = lane & 3;
    const int row_key = 4 * (g8 >> 1) + (g8 & 1);  // the key of row g8 of a tile; row g8 + 8 has that + 2
    // where this lane's pieces lie in a slot: a tile of 16 keys further on they lie 16 HD bytes further on, at the same place of
    // the swizzle's pattern
    int k_at[KP][2], v_at[MINE];
#pragma unroll
    for (int c = 0; c < KP; ++c) {
      k_at[c][0] = key_offset<HD>(warp * 32 + row_key, key_piece<HD>(t4, c));
      k_at[c][1] = key_offset<HD>(warp * 32 + row_key + 2, key_piece<HD>(t4, c));
    }
#pragma unroll
    for (int c = 0; c < MINE; ++c)
      v_at[c] = HALVES == 2 ? value_offset<HD>(t4, g8, warp + 4 * c) : value_offset<HD>(t4, g8, warp >> 1) + (warp & 1) * 8;
    Walk w = start();
    int slot = 0, use = 0;
    bool fresh = true;  // the item begins a run
    uint32_t qb[KP][4][2];
    float un[2] = {1.f, 1.f};  // what undoes the queries' scaling, of the two heads whose scores this thread gets
    int heads = 0, head0 = 0, tok = 0;
    float run_top[2], run_sum[2];  // of heads 2 t4 and 2 t4 + 1; the sum over this thread's keys
    float o[MINE][HALVES][4];
    for (int i = 0; i < count; ++i) {
      if (fresh) {
        run_top[0] = run_top[1] = -INFINITY;
        run_sum[0] = run_sum[1] = 0.f;
#pragma unroll
        for (int c = 0; c < MINE; ++c)
#pragma unroll
          for (int h = 0; h < HALVES; ++h) o[c][h][0] = o[c][h][1] = o[c][h][2] = o[c][h][3] = 0.f;
        const int g = w.slice / n_sub, sub = w.slice - g * n_sub;
        heads = min(MAX_COLUMNS, group - sub * MAX_COLUMNS);
        head0 = g * group + sub * MAX_COLUMNS;
        // the queries as the 8-column operand: column lane / 4 is a head, its elements in the order of the keys' pieces
        tok = seq_tok[w.seq];
        const __nv_bfloat16* row = q + (size_t)tok * q_stride + (head0 + min(g8, heads - 1)) * HD;
        uint4 raw[KP][2];
#pragma unroll
        for (int c = 0; c < KP; ++c) {
          raw[c][0] = ld_global_16(row + 16 * key_piece<HD>(t4, c));
          raw[c][1] = ld_global_16(row + 16 * key_piece<HD>(t4, c) + 8);
        }
        uint32_t top = 0;  // the largest magnitude's bits: bfloat16 order is the order of its bits
#pragma unroll
        for (int c = 0; c < KP; ++c)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t x[4] = {raw[c][h].x, raw[c][h].y, raw[c][h].z, raw[c][h].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) top = __vmaxu2(top, x[j] & 0x7fff7fffu);
          }
        int big = max(top & 0xffffu, top >> 16);
        big = max(big, __shfl_xor_sync(0xffffffffu, big, 1));
        big = max(big, __shfl_xor_sync(0xffffffffu, big, 2));
        const int up = min(14 - ((big >> 7) - 127), 126);  // power of two that the query is multiplied by
        const float f = exp2_int(up), unscale = exp2_int(-up);
#pragma unroll
        for (int c = 0; c < KP; ++c)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t x[4] = {raw[c][h].x, raw[c][h].y, raw[c][h].z, raw[c][h].w};
#pragma unroll
            for (int j = 0; j < 4; ++j)
              qb[c][2 * h + (j >> 1)][j & 1] =
                  g8 < heads ? pack_f16(__uint_as_float(x[j] << 16) * f, __uint_as_float(x[j] & 0xffff0000u) * f) : 0u;
          }
        un[0] = __shfl_sync(0xffffffffu, unscale, 8 * t4);
        un[1] = __shfl_sync(0xffffffffu, unscale, 8 * t4 + 4);
      }
      const int k0 = (w.first + w.split) * SPLIT;
      const bool edge = k0 < w.k_begin || k0 + SPLIT > w.p + 1;  // some keys of the split are not seen
      const int last = w.p, k_begin = w.k_begin;

      // S^T[keys, heads] = K Q^T for this warp's 32 keys
      const unsigned char* Ks = ring + slot * SLOT_BYTES;
      mbar_wait(&full[slot], use & 1, status, &gave_up);
      float s[2][4];
      int ek[2], ev[2];
      const bool apart = s_apart[slot] != 0;
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        const int box = (warp * 32 + mt * 16) >> box_shift;
        ek[mt] = s_exp[slot][0][box];
        ev[mt] = s_exp[slot][1][box];
        s[mt][0] = s[mt][1] = s[mt][2] = s[mt][3] = 0.f;
#pragma unroll
        for (int c = 0; c < KP; ++c) {
          const uint4 a = *reinterpret_cast<const uint4*>(Ks + k_at[c][0] + mt * 16 * HD);
          const uint4 b = *reinterpret_cast<const uint4*>(Ks + k_at[c][1] + mt * 16 * HD);
          const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, bw[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
          for (int m = 0; m < 4; ++m)
            mma_f16(s[mt], halves_of_low(aw[m]), halves_of_low(bw[m]), halves_of_high(aw[m]), halves_of_high(bw[m]),
                    qb[c][m][0], qb[c][m][1]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[slot]);  // this warp is done with the keys
      if (++slot == SLOTS) {
        slot = 0;
        ++use;
      }

      // this thread's scores: keys of row g8 and that + 2, heads 2 t4 and 2 t4 + 1
      // s becomes the base-2 score plus the exponent of the value's scale
      float top[2] = {run_top[0], run_top[1]};
      const float fe[2] = {(float)ev[0], (float)ev[1]};
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        const float ks = exp2_int(max(ek[mt], -126));
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if constexpr (CAPPED) {
            // (the query's power of two first: large keys' sums would leave float32 before a small query's brings them back)
            s[mt][h] = capped_score(s[mt][h] * un[h] * ks, scale_log2, cap_log2, scale_by_cap) + fe[mt];
            s[mt][2 + h] = capped_score(s[mt][2 + h] * un[h] * ks, scale_log2, cap_log2, scale_by_cap) + fe[mt];
          } else {
            const float f = ks * (un[h] * scale_log2);
            s[mt][h] = fmaf(s[mt][h], f, fe[mt]);
            s[mt][2 + h] = fmaf(s[mt][2 + h], f, fe[mt]);
          }
        }
      }
      if (edge || ek[0] == NO_PAGE || ek[1] == NO_PAGE) {
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int j = k0 + warp * 32 + mt * 16 + row_key + (e & 2);
            if (j < k_begin || j > last || ek[mt] == NO_PAGE) s[mt][e] = -INFINITY;
          }
      }
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int e = 0; e < 4; ++e) top[e & 1] = fmaxf(top[e & 1], s[mt][e]);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], o));
      if (g8 == 0) *reinterpret_cast<float2*>(&s_top[warp][2 * t4]) = make_float2(top[0], top[1]);
      asm volatile("bar.sync 1, %0;\n" ::"n"(CONSUMERS) : "memory");
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float2 other = *reinterpret_cast<const float2*>(&s_top[x][2 * t4]);
        top[0] = fmaxf(top[0], other.x);
        top[1] = fmaxf(top[1], other.y);
      }
      // what the run holds so far, relative to the new maximum
      float keep[2], down[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        down[h] = run_top[h] == -INFINITY ? -INFINITY : run_top[h] - top[h];
        keep[h] = ex2(down[h]);
        run_top[h] = top[h];
      }
      const float base[2] = {WEIGHT_SHIFT - (top[0] == -INFINITY ? 0.f : top[0]), WEIGHT_SHIFT - (top[1] == -INFINITY ? 0.f : top[1])};
      // The softmax's own weight is the value's weight over its scale, 2^-f: a multiplication where the scales of the run are
      // near one another.  (A weight that is zero in float32 is 2^-141 of the largest, over scales 2^64 apart 2^-77 of the
      // denominator; what `keep` loses of an earlier sum is 2^-62.)  Elsewhere an exponential of its own, to 2^-149 where
      // the denominator is 2^-100 or more.
      if (!apart) {
        run_sum[0] *= keep[0];
        run_sum[1] *= keep[1];
        const float inv[2] = {exp2_int(-ev[0] - WEIGHT_SHIFT), exp2_int(-ev[1] - WEIGHT_SHIFT)};
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s[mt][e] = ex2(s[mt][e] + base[e & 1]);
            run_sum[e & 1] = fmaf(s[mt][e], inv[mt], run_sum[e & 1]);
          }
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float half = ex2(0.5f * down[h]);
          run_sum[h] = run_sum[h] * half * half;
        }
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = s[mt][e] + base[e & 1];
            s[mt][e] = ex2(x);
            run_sum[e & 1] += ex2_subnormal(x - (fe[mt] + WEIGHT_SHIFT));
          }
      }
      // the weights as the 8-column operand: an 8 x 8 transposition in registers for each half tile
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
        s_weights[warp * 2 + mt][lane] =
            make_uint2(transposed_8x8(pack_f16(s[mt][0], s[mt][1])), transposed_8x8(pack_f16(s[mt][2], s[mt][3])));
      asm volatile("bar.sync 1, %0;\n" ::"n"(CONSUMERS) : "memory");

      // O^T[dims, heads] = V^T P^T: this warp's pieces of all keys
      const unsigned char* Vs = ring + slot * SLOT_BYTES;
      mbar_wait(&full[slot], use & 1, status, &gave_up);
#pragma unroll
      for (int c = 0; c < MINE; ++c)
#pragma unroll
        for (int h = 0; h < HALVES; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[c][h][e] *= keep[e & 1];
#pragma unroll
      for (int mt = 0; mt < TILES; ++mt) {
        const uint2 pb = s_weights[mt][lane];
        uint32_t mask = 0xffffffffu;
        if (edge) {
          // codes of keys that are not seen: zero (a weight of zero times a NaN of a page's former owner would be a NaN)
          mask = 0;
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const int j = k0 + mt * 16 + 4 * t4 + b;
            if (j >= k_begin && j <= last) mask |= 0xffu << (8 * b);
          }
        }
#pragma unroll
        for (int c = 0; c < MINE; ++c) {
          // dimensions 4 (g8 + 8 i) + 0..3 of the four keys of group t4 of the tile; at HD = 64 a warp has two of the four
          if constexpr (HALVES == 2) {
            uint4 v = *reinterpret_cast<const uint4*>(Vs + v_at[c] + mt * 16 * HD);
            if (edge) v.x &= mask, v.y &= mask, v.z &= mask, v.w &= mask;
            mma_f16(o[c][0], halves_of_low(v.x), halves_of_low(v.y), halves_of_high(v.x), halves_of_high(v.y), pb.x, pb.y);
            mma_f16(o[c][1], halves_of_low(v.z), halves_of_low(v.w), halves_of_high(v.z), halves_of_high(v.w), pb.x, pb.y);
          } else {
            uint2 v = *reinterpret_cast<const uint2*>(Vs + v_at[c] + mt * 16 * HD);
            if (edge) v.x &= mask, v.y &= mask;
            mma_f16(o[c][0], halves_of_low(v.x), halves_of_low(v.y), halves_of_high(v.x), halves_of_high(v.y), pb.x, pb.y);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[slot]);  // ... and with the values
      if (++slot == SLOTS) {
        slot = 0;
        ++use;
      }

      const Walk at = w;
      if (i + 1 < count) advance(w);
      fresh = i + 1 == count || w.seq != at.seq || w.slice != at.slice;
      if (!fresh) continue;
      if (i + 1 < count && g8 < min(MAX_COLUMNS, group)) {
        // the next run's queries on their way to L1
        const int g = w.slice / n_sub, first = g * group + (w.slice - g * n_sub) * MAX_COLUMNS;
        if (g8 < g * group + group - first) {
          const __nv_bfloat16* row = q + (size_t)seq_tok[w.seq] * q_stride + (first + g8) * HD;
          for (int c = t4; c < HD / 64; c += 4) asm volatile("prefetch.global.L1 [%0];\n" ::"l"(row + c * 64));
        }
      }

      // ---- the run ends: the four warps' sums, then the result or a partial ----
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) run_sum[h] += __shfl_xor_sync(0xffffffffu, run_sum[h], x);
      if (g8 == 0) *reinterpret_cast<float2*>(&s_sum[warp][2 * t4]) = make_float2(run_sum[0], run_sum[1]);
      asm volatile("bar.sync 1, %0;\n" ::"n"(CONSUMERS) : "memory");
      float sum[2] = {0.f, 0.f};
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float2 other = *reinterpret_cast<const float2*>(&s_sum[x][2 * t4]);
        sum[0] += other.x;
        sum[1] += other.y;
      }
      const long long run0 = (long long)s_cum[at.seq] * slices + (long long)at.slice * at.n;  // the request's first item of this head
      __nv_bfloat16* const dst = out + (size_t)tok * out_stride + head0 * HD;
      if (run0 >= begin && run0 + at.n <= begin + count) {
        // all keys of the request
        float f[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int head = head0 + min(2 * t4 + e, heads - 1);
          f[e] = finish(run_top[e], sum[e], sinks, head);
        }
#pragma unroll
        for (int c = 0; c < MINE; ++c)
#pragma unroll
          for (int h = 0; h < HALVES; ++h)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              // rows g8 and g8 + 8 of the product are neighbouring dimensions
              const int piece = HALVES == 2 ? warp + 4 * c : warp >> 1, which = HALVES == 2 ? h : warp & 1;
              const int d = 4 * (g8 + 8 * piece) + 2 * which;
              if (2 * t4 + e < heads)
                store_pair(dst + (2 * t4 + e) * HD + d, o[c][h][e] * WEIGHT_UNIT * f[e], o[c][h][2 + e] * WEIGHT_UNIT * f[e],
                           out_freqs, d / 2, at.p);
            }
        continue;
      }
      // a block's partials: of the run that reaches back behind its stretch, and of the one that goes on after it
      const int which_run = run0 >= begin;
      float* part = scratch + ((size_t)blockIdx.x * 2 + which_run) * MAX_COLUMNS * run_stride<HD>();
#pragma unroll
      for (int c = 0; c < MINE; ++c)
#pragma unroll
        for (int h = 0; h < HALVES; ++h)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int piece = HALVES == 2 ? warp + 4 * c : warp >> 1, which = HALVES == 2 ? h : warp & 1;
            if (2 * t4 + e < heads)
              *reinterpret_cast<float2*>(part + (2 * t4 + e) * run_stride<HD>() + 4 * (g8 + 8 * piece) + 2 * which) =
                  make_float2(o[c][h][e], o[c][h][2 + e]);
          }
      if (warp == 0 && g8 == 0)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (2 * t4 + e < heads)
            *reinterpret_cast<float2*>(part + (2 * t4 + e) * run_stride<HD>() + HD) = make_float2(run_top[e], sum[e]);
      if (tid == 0) {
        *reinterpret_cast<int4*>(s_run[which_run]) = make_int4(at.seq, at.slice, tok, at.p);
        s_run[which_run][4] = block_of(run0);
        s_run[which_run][5] = block_of(run0 + at.n - 1);
      }
    }

    // ---- the block's partials are counted when all its items are done: fence and counters cost their latency once ----
    asm volatile("bar.sync 1, %0;\n" ::"n"(CONSUMERS) : "memory");
    if (s_run[0][3] < 0 && s_run[1][3] < 0) return;
    if (tid == 0) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        s_last[x] = 0;
        if (s_run[x][3] < 0) continue;
        int* counter = counters + (size_t)s_run[x][0] * slices + s_run[x][1];
        int before;
        // (release for the whole block, whose stores are ordered before by the barrier; acquire for what the others stored)
        asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;\n" : "=r"(before) : "l"(counter) : "memory");
        if (before == s_run[x][5] - s_run[x][4]) {
          *counter = 0;  // for the launches behind this one
          s_last[x] = 1;
        }
      }
    }
    asm volatile("bar.sync 1, %0;\n" ::"n"(CONSUMERS) : "memory");
    for (int x = 0; x < 2; ++x) {
      if (!s_last[x]) continue;
      const int first_block = s_run[x][4], last_block = s_run[x][5], p = s_run[x][3];
      const int g = s_run[x][1] / n_sub, sub = s_run[x][1] - g * n_sub;
      const int heads = min(MAX_COLUMNS, group - sub * MAX_COLUMNS), head0 = g * group + sub * MAX_COLUMNS;
      __nv_bfloat16* const dst = out + (size_t)s_run[x][2] * out_stride + head0 * HD;
      // every partial of this request and head is there: a thread merges four neighbouring dimensions of a head, the
      // loads of sixteen partials in flight together, of eight where no more are left
      for (int y = tid; y < heads * (HD / 4); y += CONSUMERS) {
        const int r = y / (HD / 4), d = 4 * (y - r * (HD / 4));
        float m = -INFINITY, l = 0.f, a[4] = {0.f, 0.f, 0.f, 0.f};
        auto merged = [&](auto flight, int b0) {
          constexpr int FLIGHT = decltype(flight)::value;
          float2 ml[FLIGHT];
          float4 v[FLIGHT];
#pragma unroll
          for (int u = 0; u < FLIGHT; ++u) {
            const int b = b0 + u;
            const float* from = scratch + (((size_t)min(b, last_block) * 2 + (b == first_block)) * MAX_COLUMNS + r) * run_stride<HD>();
            // (volatile: all of them leave before the first is waited for)
            asm volatile("ld.global.cg.v2.f32 {%0,%1}, [%2];\n" : "=f"(ml[u].x), "=f"(ml[u].y) : "l"(from + HD) : "memory");
            asm volatile("ld.global.cg.v4.f32 {%0,%1,%2,%3}, [%4];\n"
                         : "=f"(v[u].x), "=f"(v[u].y), "=f"(v[u].z), "=f"(v[u].w)
                         : "l"(from + d)
                         : "memory");
          }
          float top = m, low = m == -INFINITY ? INFINITY : m;
#pragma unroll
          for (int u = 0; u < FLIGHT; ++u) {
            low = fminf(low, ml[u].x);
            if (b0 + u > last_block) ml[u] = make_float2(-INFINITY, 0.f);  // (the last one once more: nothing)
            top = fmaxf(top, ml[u].x);
          }
          const float keep = m == -INFINITY ? 0.f : ex2(m - top);
          const bool apart = low - top < -SCALES_NEAR;
          if (apart) {
            const float half = m == -INFINITY ? 0.f : ex2(0.5f * (m - top));
            l = l * half * half;
#pragma unroll
            for (int u = 0; u < FLIGHT; ++u) {
              const float h = ml[u].x == -INFINITY ? 0.f : ex2(0.5f * (ml[u].x - top));
              l += h * ml[u].y * h;
            }
          } else {
            l *= keep;
          }
          m = top;
#pragma unroll
          for (int e = 0; e < 4; ++e) a[e] *= keep;
#pragma unroll
          for (int u = 0; u < FLIGHT; ++u) {
            const float f = ml[u].x == -INFINITY ? 0.f : ex2(ml[u].x - top);
            if (!apart) l += f * ml[u].y;
            a[0] += f * v[u].x;
            a[1] += f * v[u].y;
            a[2] += f * v[u].z;
            a[3] += f * v[u].w;
          }
        };
        for (int b0 = first_block; b0 <= last_block;) {
          if (last_block - b0 >= 8) {
            merged(std::integral_constant<int, 16>(), b0);
            b0 += 16;
          } else {
            merged(std::integral_constant<int, 8>(), b0);
            b0 += 8;
          }
        }
        const float f = finish(m, l, sinks, head0 + r);
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] *= WEIGHT_UNIT;
        store_pair(dst + r * HD + d, a[0] * f, a[1] * f, out_freqs, d / 2, p);
        store_pair(dst + r * HD + d + 2, a[2] * f, a[3] * f, out_freqs, d / 2 + 1, p);
      }
    }
  }
}

}  // namespace fg_kv8
