// Writing and reading back the pages of the cache in 8 bits.
#pragma once

#include "kv8.cuh"

namespace fg_kv8 {

// ---------------------------------------------------------------------------------
// The write.  A page's new tokens are a run: consecutive tokens of the step with the same request and page.  Its scale
// needs the largest magnitude of the whole run (and the scale that the cached entries before it have), so a run is the
// work of one block, found on the device: a block looks at a stretch of tokens, PER a warp, and takes the runs that begin
// among them, keys and values of one key/value head.  A run of one token (a decoded token) is a warp's work; a longer run is
// the block's, a warp for four slots at a time, whose rows stay in registers between the search for the largest and the
// rounding.
//
// Bound by instructions at many tokens (each key/value head's block computes the angles anew) and by latencies at few: a block is a
// chain of positions, pages, rows, angles and codes.  Steps of many tokens take stretches of 64 tokens (PER = 4), a page of
// the usual size: with 16, three of four blocks found no run and left.  Queries have blocks of their own, a warp a token.
// (32 / 8 heads of 128: 2,048 prompt tokens beside 20 single ones 14.4 us, the write in 16 bits 9.4; 8,192 tokens 66.4 and 43.7.
// Without the exponents in doubt 14.1 and 65.6, without codes in doubt 12.3 and 53.8; with queries in the stretches' blocks and each thread looking
// through all places for the runs: 19.2 and 67.2.)
// ---------------------------------------------------------------------------------
constexpr int WRITE_WARPS = 16, WRITE_THREADS = 32 * WRITE_WARPS;
constexpr int Q_SLICE = 8, Q_FLIGHT = 8;  // query heads a block rotates, and those whose rows are in flight together

// A lane's E = HD / 32 neighbouring elements of a row.
template <int E, bool VEC>
__device__ __forceinline__ void load_lane(uint32_t (&w)[E / 2], const __nv_bfloat16* row, int lane) {
  const __nv_bfloat16* p = row + lane * E;
  if constexpr (VEC) {
    if constexpr (E == 2) {
      w[0] = ld_global_4(p);
    } else if constexpr (E == 4) {
      asm volatile("ld.global.v2.u32 {%0,%1}, [%2];\n" : "=r"(w[0]), "=r"(w[1]) : "l"(p) : "memory");
    } else {
      const uint4 v = ld_global_16(p);
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    }
  } else {
    const volatile unsigned short* s = reinterpret_cast<const volatile unsigned short*>(p);
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      const uint32_t lo = s[2 * i], hi = s[2 * i + 1];
      w[i] = lo | (hi << 16);
    }
  }
}
template <int E>
__device__ __forceinline__ void unpacked(float (&x)[E], const uint32_t (&w)[E / 2]) {
#pragma unroll
  for (int i = 0; i < E / 2; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

// A turned pair in 64 bits, for numbers whose code the float32 ones leave in doubt (one in some 40,000, and exact ties): w0 and w1
// are the norm's factors, the angle is float32 by definition.  To float32 with the last bit set where bits are lost, so that
// the rounding to a code is the only one.
__device__ __noinline__ float2 turned_exactly(const __nv_bfloat16* at, double w0, double w1, float angle, float magnitude) {
  const volatile unsigned short* raw = reinterpret_cast<const volatile unsigned short*>(at);
  const double a = (double)__uint_as_float((uint32_t)raw[0] << 16) * w0, b = (double)__uint_as_float((uint32_t)raw[1] << 16) * w1;
  double sn, cs;
  sincos((double)angle, &sn, &cs);
  auto narrowed = [](double x) {
    const float r = __double2float_rz(x);
    return (double)r == x ? r : __uint_as_float(__float_as_uint(r) | 1u);
  };
  return make_float2(narrowed((a * cs - b * sn) * magnitude), narrowed((b * cs + a * sn) * magnitude));
}

// A page's exponent: from the run's largest magnitude and, behind cached entries, no lower than theirs.
__device__ __forceinline__ int run_exponent(float amax, int slot, float before, int& old_e) {
  int e = scale_exponent(amax);
  old_e = e;
  if (slot > 0) {
    old_e = exponent_of_scale(before);
    e = max(e, old_e);
  }
  return e;
}

// Cached entries before `slot` rounded again at a larger scale, by `n` threads of which this is number `i`.
template <int HD>
__device__ __forceinline__ void rescale_entries(unsigned char* base, bool is_v, int slot, float f, int i, int n) {
  const int whole = is_v ? (slot & ~3) * HD : slot * HD;  // bytes of whole rows (of whole groups of four rows)
  for (int at = i * 4; at < whole; at += n * 4) {
    uint32_t* w = reinterpret_cast<uint32_t*>(base + at);
    *w = rescaled(ld_global_4(w), f);
  }
  if (is_v && (slot & 3)) {
    const uint32_t mask = (1u << (8 * (slot & 3))) - 1u;  // tokens of the last group that are cached
    for (int d = i; d < HD; d += n) {
      uint32_t* w = reinterpret_cast<uint32_t*>(base + whole) + d;
      const uint32_t old = ld_global_4(w);
      *w = (old & ~mask) | (rescaled(old, f) & mask);
    }
  }
}

// A lane's codes of one row.
template <int HD>
__device__ __forceinline__ void store_codes(unsigned char* base, bool is_v, const float (&x)[HD / 32], int slot, float inv, int lane) {
  constexpr int E = HD / 32;
  uint32_t c[E / 2];
#pragma unroll
  for (int i = 0; i < E / 2; ++i) c[i] = codes_of(x[2 * i] * inv, x[2 * i + 1] * inv);
  if (!is_v) {
    unsigned char* dst = base + slot * HD + lane * E;
    if constexpr (E == 2) *reinterpret_cast<uint16_t*>(dst) = (uint16_t)c[0];
    else if constexpr (E == 4) *reinterpret_cast<uint32_t*>(dst) = c[0] | (c[1] << 16);
    else *reinterpret_cast<uint2*>(dst) = make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
  } else {
    unsigned char* dst = base + (slot >> 2) * (4 * HD) + lane * (4 * E) + (slot & 3);
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      dst[8 * i] = (unsigned char)c[i];
      dst[8 * i + 4] = (unsigned char)(c[i] >> 8);
    }
  }
}

// A run of `n` tokens from slot `slot` and position p0 on, its keys (or its values) all in 64 bits, by the whole block, or by one
// warp without an s_amax: for runs whose largest magnitude float32 cannot tell from a border of the scales.  src: the run's first row; rstd: the norm's factor of
// its first token or null, `rstd_stride` apart; norm_w its weights or null; big: pairs that `magnitude` multiplies.
template <int HD>
__device__ __noinline__ void exact_run(const __nv_bfloat16* src, int src_stride, bool is_v, int n, int slot, int p0, const float* freqs,
                                       const float* rstd, int rstd_stride, const float* norm_w, float magnitude, int big,
                                       unsigned char* base, float* scale, float* s_amax) {
  constexpr int E = HD / 32;
  const int lane = threadIdx.x & 31, warp = s_amax ? threadIdx.x >> 5 : 0, warps = s_amax ? WRITE_WARPS : 1;
  auto sync = [&]() {
    if (s_amax) __syncthreads();
    else __syncwarp();
  };
  auto row = [&](float (&x)[E], int i) {
#pragma unroll 1
    for (int j = 0; j < E / 2; ++j) {
      const int pair = lane * (E / 2) + j;
      const __nv_bfloat16* at = src + (size_t)i * src_stride + 2 * pair;
      double w0 = rstd ? rstd[(size_t)i * rstd_stride] : 1.f, w1 = w0;
      if (norm_w) w0 *= norm_w[2 * pair], w1 *= norm_w[2 * pair + 1];
      const float2 v = freqs || rstd ? turned_exactly(at, w0, w1, freqs ? (float)(p0 + i) * freqs[pair] : 0.f, freqs && pair < big ? magnitude : 1.f)
                                     : make_float2(__bfloat162float(at[0]), __bfloat162float(at[1]));
      x[2 * j] = fabsf(v.x) == INFINITY ? __int_as_float(0x7fffffff) : v.x;
      x[2 * j + 1] = fabsf(v.y) == INFINITY ? __int_as_float(0x7fffffff) : v.y;
    }
  };
  float x[E], amax = 0.f;
  const float before = slot > 0 ? __uint_as_float(ld_global_4(scale)) : 1.f;
#pragma unroll 1
  for (int i = warp; i < n; i += warps) {
    row(x, i);
#pragma unroll
    for (int j = 0; j < E; ++j) amax = fmaxf(amax, fabsf(x[j]));
  }
  amax = warp_max(amax);
  if (s_amax) {
    __syncthreads();
    if (lane == 0) s_amax[warp] = amax;
    __syncthreads();
    amax = warp_max(s_amax[lane & (WRITE_WARPS - 1)]);
  }
  int old_e;
  const int e = run_exponent(amax, slot, before, old_e);
  if (e > old_e) rescale_entries<HD>(base, is_v, slot, exp2_int(max(old_e - e, -126)), warp * 32 + lane, warps * 32);
  sync();  // rescaled entries share words with new ones; every thread has read the old scale
#pragma unroll 1
  for (int i = warp; i < n; i += warps) {
    row(x, i);
    store_codes<HD>(base, is_v, x, slot + i, exp2_int(-e), lane);
  }
  if (warp + lane == 0 && (slot == 0 || e > old_e)) *scale = exp2_int(e);
}

template <int HD, bool VEC, int PER>
__global__ void __launch_bounds__(WRITE_THREADS, HD <= 128 ? 2 : 1)
kv8_write_kernel(const __nv_bfloat16* q, int q_stride, __nv_bfloat16* q_out, const __nv_bfloat16* k, int k_stride,
                 const __nv_bfloat16* v, int v_stride, const int* __restrict__ pos, const int* __restrict__ req,
                 const float* __restrict__ freqs, const float* __restrict__ v_freqs, unsigned char* k_pages,
                 unsigned char* v_pages, float* k_scales, float* v_scales, const int* __restrict__ block_table, int table_width,
                 int page_size, int n_pages, int n_tokens, int n_heads, int n_kv_heads, int* status, const float* rstd,
                 const float* __restrict__ qn_w, const float* __restrict__ kn_w, int rstd_heads, float magnitude,
                 int rot_pairs) {
  constexpr int E = HD / 32, STRETCH = WRITE_WARPS * PER;
  __shared__ int s_len[STRETCH], s_page[STRETCH], s_pos[STRETCH];
  __shared__ float s_amax[2][WRITE_WARPS];
  __shared__ int s_marked;
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // blocks of keys and values first, the heads of a stretch side by side; then those of queries
  const int kv_blocks = (n_tokens + STRETCH - 1) / STRETCH * n_kv_heads;

  // sine and cosine of the lane's pairs at position p
  auto turns = [&](float (&sn)[E / 2], float (&cs)[E / 2], const float* table, int p, float mag) {
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      sn[i] = 0.f;
      cs[i] = 1.f;
      if (table != nullptr) {
        const int j = lane * (E / 2) + i;
        sincosf((float)p * table[j], &sn[i], &cs[i]);
        if (mag != 1.f && j < rot_pairs) {
          sn[i] *= mag;
          cs[i] *= mag;
        }
      }
    }
  };
  auto turn = [&](float (&x)[E], const float (&sn)[E / 2], const float (&cs)[E / 2]) {
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      const float a = x[2 * i], b = x[2 * i + 1];
      x[2 * i] = a * cs[i] - b * sn[i];
      x[2 * i + 1] = b * cs[i] + a * sn[i];
    }
  };
  // the norm's factor of a token and head (column `at_head` of the factors, 0 or 1 where the whole projection shares one)
  auto normed = [&](float (&x)[E], int t, int at_head, int at_whole, const float* w) {
    if (rstd == nullptr) return;
    const float f = rstd_heads ? rstd[(size_t)t * rstd_heads + at_head] : rstd[2 * (size_t)t + at_whole];
#pragma unroll
    for (int i = 0; i < E; ++i) x[i] *= f * (w ? w[lane * E + i] : 1.f);
  };

  if ((int)blockIdx.x >= kv_blocks) {
    // ---- queries: a warp a token, the heads of the slice ----
    const int slices = (n_heads + Q_SLICE - 1) / Q_SLICE, at = blockIdx.x - kv_blocks;
    const int h0 = at % slices * Q_SLICE, h1 = min(n_heads, h0 + Q_SLICE), t = at / slices * WRITE_WARPS + warp;
    const bool real = t < n_tokens && req[t] >= 0;
    float sn[E / 2], cs[E / 2];
    if (real) turns(sn, cs, freqs, pos[t], magnitude);
    pdl_wait();
    if (real) {
#pragma unroll 1
      for (int hb = h0; hb < h1; hb += Q_FLIGHT) {
        uint32_t raw[Q_FLIGHT][E / 2];
#pragma unroll
        for (int i = 0; i < Q_FLIGHT; ++i)
          if (hb + i < h1) load_lane<E, VEC>(raw[i], q + (size_t)t * q_stride + (hb + i) * HD, lane);
#pragma unroll
        for (int i = 0; i < Q_FLIGHT; ++i) {
          const int h = hb + i;
          if (h >= h1) continue;
          float x[E];
          unpacked(x, raw[i]);
          normed(x, t, h, 0, qn_w ? qn_w + h * HD : nullptr);
          turn(x, sn, cs);
          __nv_bfloat162 out[E / 2];
#pragma unroll
          for (int e = 0; e < E / 2; ++e) out[e] = __floats2bfloat162_rn(x[2 * e], x[2 * e + 1]);
          __nv_bfloat16* dst = q_out + ((size_t)t * n_heads + h) * HD + lane * E;
          if constexpr (VEC) {
            if constexpr (E == 2) *reinterpret_cast<uint32_t*>(dst) = *reinterpret_cast<uint32_t*>(out);
            else if constexpr (E == 4) *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<uint2*>(out);
            else *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<uint4*>(out);
          } else {
#pragma unroll
            for (int e = 0; e < E / 2; ++e) dst[2 * e] = out[e].x, dst[2 * e + 1] = out[e].y;
          }
        }
      }
    }
    return;
  }

  // ---- keys and values of one head ----
  const int g = blockIdx.x % n_kv_heads, t0 = blockIdx.x / n_kv_heads * STRETCH;
  const __nv_bfloat16* const src[2] = {k + g * HD, v + g * HD};
  const int src_stride[2] = {k_stride, v_stride};
  unsigned char* const pool[2] = {k_pages, v_pages};
  float* const scales[2] = {k_scales, v_scales};
  const float* norm_w = kn_w ? kn_w + g * HD : nullptr;

  // the runs that begin at this warp's tokens: their lengths (0: none begins there) and pages
  bool any_long = false;
  const int mine = t0 + warp * PER;
  int reqs[PER + 1], positions[PER + 1];  // of the token before the warp's, and of the warp's: all on their way together
#pragma unroll
  for (int u = 0; u <= PER; ++u) {
    const int t = mine + u - 1;
    const bool there = t >= 0 && t < n_tokens;
    reqs[u] = there ? req[t] : -1;
    positions[u] = there ? pos[t] : 0;
  }
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int t = mine + u, r = reqs[u + 1], p = positions[u + 1];
    const int slot = p & (page_size - 1);
    int len = 0, page = -1;
    if (r >= 0 && (slot == 0 || reqs[u] != r || positions[u] != p - 1)) {
      const int logical = p / page_size;
      page = p >= 0 && logical < table_width ? block_table[(size_t)r * table_width + logical] : -1;
      const int most = min(page_size - slot, n_tokens - t);
      for (int at = 0; at < most; at += 32) {
        const int i = at + lane;
        const bool mine = i < most && req[t + i] == r && pos[t + i] == p + i;
        const unsigned all = __ballot_sync(0xffffffffu, mine);
        if (all != 0xffffffffu) {
          len += __ffs(~all) - 1;
          break;
        }
        len += 32;
      }
      if (page < 0 || page >= n_pages) {
        if (status && lane == 0) atomicOr(status, FG_STATUS_BAD_PAGE);
        len = 0;
      }
    }
    any_long = any_long || len > 1;
    if (lane == 0) {
      s_len[warp * PER + u] = len;
      s_page[warp * PER + u] = page;
      s_pos[warp * PER + u] = p;
    }
  }
  if (threadIdx.x == 0) s_marked = 0;
  any_long = __syncthreads_or(any_long);
  pdl_wait();

  // The largest finite magnitude (fmaxf passes over NaNs); infinities become NaNs, as they are stored.
  auto row_amax = [&](float (&x)[E]) {
    float a = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) a = fmaxf(a, fabsf(x[i]));
    if (a == INFINITY) {
      a = 0.f;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        if (fabsf(x[i]) == INFINITY) x[i] = __int_as_float(0x7fffffff);
        a = fmaxf(a, fabsf(x[i]));
      }
    }
    return a;
  };
  auto rescale = [&](int kv, size_t block, int slot, float f, int i, int n) {
    rescale_entries<HD>(pool[kv] + block * (size_t)page_size * HD, kv, slot, f, i, n);
  };
  auto store_row = [&](int kv, const float (&x)[E], size_t block, int slot, float inv) {
    store_codes<HD>(pool[kv] + block * (size_t)page_size * HD, kv, x, slot, inv, lane);
  };
  // Turned numbers are off by less than 2^-21 of their pair's magnitudes (sine and cosine 2^-23, two products and a sum 2^-24
  // each, and the square root of two from a pair to its turn), with a norm's factors or a magnitude less than 2^-20.  Where that
  // could change a code, and something has been rounded at all, the pair is computed in 64 bits.  (Without this one code in a
  // million is the neighbouring one; it takes 2 of the 14 us given above; doubts kept in a list and
  // settled behind the run 3.)
  const bool turned[2] = {freqs != nullptr || rstd != nullptr, v_freqs != nullptr};  // else the numbers are exact
  const float off = rstd != nullptr || magnitude != 1.f ? 0x1p-20f : 0x1p-21f;
  auto settled = [&](int kv, float (&x)[E], int t, int p, float inv) {
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      const float y0 = x[2 * i] * inv, y1 = x[2 * i + 1] * inv, d = (fabsf(y0) + fabsf(y1)) * off;
      if (d != 0.f && codes_of(y0 - d, y1 - d) != codes_of(y0 + d, y1 + d)) {
        const float* table = kv ? v_freqs : freqs;
        const int j = lane * (E / 2) + i;
        const float angle = table ? (float)p * table[j] : 0.f, factor = table && !kv && j < rot_pairs ? magnitude : 1.f;
        const bool normed_too = !kv && rstd != nullptr;
        if (angle == 0.f && factor == 1.f && !normed_too) continue;
        double w0 = 1.0, w1 = 1.0;
        if (normed_too) {
          w0 = w1 = rstd_heads ? rstd[(size_t)t * rstd_heads + n_heads + g] : rstd[2 * (size_t)t + 1];
          if (norm_w) w0 *= norm_w[2 * j], w1 *= norm_w[2 * j + 1];
        }
        const float2 v = turned_exactly(src[kv] + (size_t)t * src_stride[kv] + 2 * j, w0, w1, angle, factor);
        x[2 * i] = v.x;
        x[2 * i + 1] = v.y;
      }
    }
  };
  // The largest magnitude is off by less than 2^-19 of itself, for its pair's other number is no larger.  Where that leaves the
  // exponent in doubt (the borders are 1.75 times powers of two: within 32 of its last places, 2^-23 each, of one),
  // the run is marked by a negative length and left to exact_run, behind the others.  (Its keys or values may have been written
  // before: once more is the same.)
  auto in_doubt = [&](int kv, float amax) {
    return __builtin_expect(turned[kv] && ((__float_as_uint(amax) - (0x600000u - 32u)) & 0x7fffffu) <= 64u, 0);
  };
  auto exact = [&](int kv, int t, int n, int p, int page, float* amax) {
    const int slot = p & (page_size - 1);
    const size_t block = (size_t)page * n_kv_heads + g;
    const float* factor = kv || rstd == nullptr ? nullptr : rstd_heads ? rstd + (size_t)t * rstd_heads + n_heads + g : rstd + 2 * (size_t)t + 1;
    exact_run<HD>(src[kv] + (size_t)t * src_stride[kv], src_stride[kv], kv, n, slot, p, kv ? v_freqs : freqs, factor,
                  rstd_heads ? rstd_heads : 2, kv ? nullptr : norm_w, kv ? 1.f : magnitude, kv ? 0 : rot_pairs,
                  pool[kv] + block * (size_t)page_size * HD, scales[kv] + block, amax);
  };
  auto scale_before = [&](int kv, size_t block, int slot) {
    return slot > 0 ? __uint_as_float(ld_global_4(scales[kv] + block)) : 1.f;
  };

#pragma unroll 1
  for (int u = 0; u < PER; ++u) {
    if (s_len[warp * PER + u] != 1) continue;
    const int t = t0 + warp * PER + u, p = s_pos[warp * PER + u], slot = p & (page_size - 1);
    const size_t block = (size_t)s_page[warp * PER + u] * n_kv_heads + g;
    uint32_t raw[2][E / 2];
    load_lane<E, VEC>(raw[0], src[0] + (size_t)t * src_stride[0], lane);
    load_lane<E, VEC>(raw[1], src[1] + (size_t)t * src_stride[1], lane);
    const float before[2] = {scale_before(0, block, slot), scale_before(1, block, slot)};
    bool left = false;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      float x[E];
      unpacked(x, raw[kv]);
      if (kv == 0) normed(x, t, n_heads + g, 1, norm_w);
      if (kv == 0 || v_freqs != nullptr) {
        float sn[E / 2], cs[E / 2];
        turns(sn, cs, kv ? v_freqs : freqs, p, kv ? 1.f : magnitude);
        turn(x, sn, cs);
      }
      const float amax = warp_max(row_amax(x));
      if (in_doubt(kv, amax)) {
        left = true;
        continue;
      }
      int old_e;
      const int e = run_exponent(amax, slot, before[kv], old_e);
      if (e > old_e) {
        rescale(kv, block, slot, exp2_int(max(old_e - e, -126)), lane, 32);
        __syncwarp();
      }
      if (turned[kv]) settled(kv, x, t, p, exp2_int(-e));
      store_row(kv, x, block, slot, exp2_int(-e));
      if (lane == 0 && (slot == 0 || e > old_e)) scales[kv][block] = exp2_int(e);
    }
    if (left && lane == 0) s_len[warp * PER + u] = -1, s_marked = 1;
  }
  if (!any_long) {
    __syncwarp();
#pragma unroll 1
    for (int u = 0; u < PER; ++u)
      if (__builtin_expect(s_len[warp * PER + u] < 0, 0)) {
        exact(0, mine + u, 1, s_pos[warp * PER + u], s_page[warp * PER + u], nullptr);
        exact(1, mine + u, 1, s_pos[warp * PER + u], s_page[warp * PER + u], nullptr);
      }
    return;
  }

  unsigned todo = 0;  // runs of two and more tokens among 32 of the stretch's tokens
#pragma unroll 1
  for (int w = -1;;) {
    todo &= todo - 1;
    while (todo == 0 && (w | 31) + 1 < STRETCH) {
      w = (w | 31) + 1;
      todo = __ballot_sync(0xffffffffu, w + lane < STRETCH && s_len[(w + lane) % STRETCH] > 1);
    }
    if (todo == 0) break;
    w = (w & ~31) + __ffs(todo) - 1;
    const int n = s_len[w];
    const int first = t0 + w, p0 = s_pos[w], slot = p0 & (page_size - 1);
    const size_t block = (size_t)s_page[w] * n_kv_heads + g;
    const float before[2] = {scale_before(0, block, slot), scale_before(1, block, slot)};
    // four slots a warp and round; pages of up to 64 slots need one round, whose rows stay in registers
    const int rounds = (page_size + 4 * WRITE_WARPS - 1) / (4 * WRITE_WARPS);
    uint32_t raw[2][4][E / 2];
    float x[4][E];  // keys, turned
    float amax[2] = {0.f, 0.f};
    auto turned_v = [&](float (&y)[E], int i, int s) {
      unpacked(y, raw[1][i]);
      if (v_freqs != nullptr) {
        float sn[E / 2], cs[E / 2];
        turns(sn, cs, v_freqs, p0 + s - slot, 1.f);
        turn(y, sn, cs);
      }
      return row_amax(y);
    };
    auto load_round = [&](int c) {
      const int s0 = 4 * (warp + WRITE_WARPS * c);
#pragma unroll
      for (int kv = 0; kv < 2; ++kv)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int s = s0 + i;
#pragma unroll
          for (int j = 0; j < E / 2; ++j) raw[kv][i][j] = 0;
          if (s >= slot && s < slot + n) load_lane<E, VEC>(raw[kv][i], src[kv] + (size_t)(first + s - slot) * src_stride[kv], lane);
        }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int s = s0 + i;
        unpacked(x[i], raw[0][i]);
        if (s < slot || s >= slot + n) continue;
        float sn[E / 2], cs[E / 2];
        turns(sn, cs, freqs, p0 + s - slot, magnitude);
        normed(x[i], first + s - slot, n_heads + g, 1, norm_w);
        turn(x[i], sn, cs);
        amax[0] = fmaxf(amax[0], row_amax(x[i]));
      }
    };
    for (int c = 0; c < rounds; ++c) {
      load_round(c);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float y[E];
        amax[1] = fmaxf(amax[1], turned_v(y, i, 4 * (warp + WRITE_WARPS * c) + i));
      }
    }
    amax[0] = warp_max(amax[0]);
    amax[1] = warp_max(amax[1]);
    __syncthreads();  // the run before is through with s_amax
    if (lane == 0) {
      s_amax[0][warp] = amax[0];
      s_amax[1][warp] = amax[1];
    }
    __syncthreads();
    int e[2], old_e[2];
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) amax[kv] = warp_max(s_amax[kv][lane & (WRITE_WARPS - 1)]);
    if (__builtin_expect(in_doubt(0, amax[0]) || in_doubt(1, amax[1]), 0)) {  // (every thread has the same numbers)
      if (threadIdx.x == 0) s_len[w] = -n, s_marked = 1;
      continue;
    }
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      e[kv] = run_exponent(amax[kv], slot, before[kv], old_e[kv]);
      if (e[kv] > old_e[kv]) rescale(kv, block, slot, exp2_int(max(old_e[kv] - e[kv], -126)), threadIdx.x, WRITE_THREADS);
    }
    if (slot > 0) __syncthreads();  // rescaled entries share words with new ones; every thread has read the old scales
    const float inv[2] = {exp2_int(-e[0]), exp2_int(-e[1])};
    for (int c = 0; c < rounds; ++c) {
      if (rounds > 1) load_round(c);
      const int s0 = 4 * (warp + WRITE_WARPS * c);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (s0 + i >= slot && s0 + i < slot + n) {
          if (turned[0]) settled(0, x[i], first + s0 + i - slot, p0 + s0 + i - slot, inv[0]);
          store_row(0, x[i], block, s0 + i, inv[0]);
        }
#pragma unroll
      for (int i = 0; i < 4; ++i) turned_v(x[i], i, s0 + i);  // now the values
      if (turned[1])
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (s0 + i >= slot && s0 + i < slot + n) settled(1, x[i], first + s0 + i - slot, p0 + s0 + i - slot, inv[1]);
      if (s0 >= slot && s0 + 4 <= slot + n) {
        // a whole group of four tokens: words
        uint32_t* dst = reinterpret_cast<uint32_t*>(v_pages + block * (size_t)page_size * HD + (size_t)s0 * HD) + lane * E;
        uint32_t wd[E];
#pragma unroll
        for (int j = 0; j < E; ++j)
          wd[j] = codes_of(x[0][j] * inv[1], x[1][j] * inv[1]) | (codes_of(x[2][j] * inv[1], x[3][j] * inv[1]) << 16);
        if constexpr (E == 2) {
          *reinterpret_cast<uint2*>(dst) = make_uint2(wd[0], wd[1]);
        } else {
#pragma unroll
          for (int j = 0; j < E; j += 4) *reinterpret_cast<uint4*>(dst + j) = make_uint4(wd[j], wd[j + 1], wd[j + 2], wd[j + 3]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (s0 + i >= slot && s0 + i < slot + n) store_row(1, x[i], block, s0 + i, inv[1]);
      }
    }
    if (threadIdx.x < 2) {
      const int kv = threadIdx.x;
      const int mine = kv ? e[1] : e[0], old = kv ? old_e[1] : old_e[0];
      if (slot == 0 || mine > old) scales[kv][block] = exp2_int(mine);
    }
  }

  __syncthreads();
  if (s_marked == 0) return;
#pragma unroll 1
  for (int w = 0; w < STRETCH; ++w) {
    if (s_len[w] >= 0) continue;
    exact(0, t0 + w, -s_len[w], s_pos[w], s_page[w], s_amax[0]);
    exact(1, t0 + w, -s_len[w], s_pos[w], s_page[w], s_amax[1]);
  }
}

// ---------------------------------------------------------------------------------
// What pages stand for, in bfloat16 [page, head, slot, HD]
// ---------------------------------------------------------------------------------
constexpr int EXPAND_THREADS = 256;

__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// One (page, head) block: slots in [lo, hi) as what they stand for, the others as zeros.
template <int HD>
__device__ __forceinline__ void expand_block(const unsigned char* in, __nv_bfloat16* out, float scale, int page_size, bool is_v,
                                             int lo, int hi) {
  // a thread takes eight dimensions of four slots: four pieces of 16 bytes of the output
  constexpr int PIECES = HD / 8;
  for (int i = threadIdx.x; i < page_size / 4 * PIECES; i += EXPAND_THREADS) {
    const int grp = i / PIECES, d = (i - grp * PIECES) * 8;
    uint2 rows[4];  // eight codes of each slot
    if (is_v) {
      const uint4 a = ld_global_16(in + (size_t)grp * 4 * HD + d * 4), b = ld_global_16(in + (size_t)grp * 4 * HD + d * 4 + 16);
      // word j holds dimension d + j of the four slots: a 4 x 4 transposition of bytes, twice
      auto transpose = [](uint4 w, uint32_t (&o)[4]) {
        const uint32_t x = __byte_perm(w.x, w.y, 0x5140), y = __byte_perm(w.z, w.w, 0x5140);
        const uint32_t u = __byte_perm(w.x, w.y, 0x7362), v = __byte_perm(w.z, w.w, 0x7362);
        o[0] = __byte_perm(x, y, 0x5410);
        o[1] = __byte_perm(x, y, 0x7632);
        o[2] = __byte_perm(u, v, 0x5410);
        o[3] = __byte_perm(u, v, 0x7632);
      };
      uint32_t lo4[4], hi4[4];
      transpose(a, lo4);
      transpose(b, hi4);
#pragma unroll
      for (int s = 0; s < 4; ++s) rows[s] = make_uint2(lo4[s], hi4[s]);
    } else {
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const unsigned char* src = in + (size_t)(grp * 4 + s) * HD + d;
        asm volatile("ld.global.v2.u32 {%0,%1}, [%2];\n" : "=r"(rows[s].x), "=r"(rows[s].y) : "l"(src) : "memory");
      }
    }
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int slot = grp * 4 + s;
      uint4 o = make_uint4(0, 0, 0, 0);
      if (slot >= lo && slot < hi) {
        const float2 a = floats_of(halves_of_low(rows[s].x)), b = floats_of(halves_of_high(rows[s].x));
        const float2 c = floats_of(halves_of_low(rows[s].y)), e = floats_of(halves_of_high(rows[s].y));
        o = make_uint4(bf16_pair(a.x * scale, a.y * scale), bf16_pair(b.x * scale, b.y * scale),
                       bf16_pair(c.x * scale, c.y * scale), bf16_pair(e.x * scale, e.y * scale));
      }
      *reinterpret_cast<uint4*>(out + (size_t)slot * HD + d) = o;
    }
  }
}

template <int HD>
__global__ void __launch_bounds__(EXPAND_THREADS)
kv8_values_kernel(const unsigned char* k_pages, const unsigned char* v_pages, const float* k_scales, const float* v_scales,
                  const int* pages, __nv_bfloat16* k_out, __nv_bfloat16* v_out, int page_size, int n_pages, int n_kv_heads,
                  int* status) {
  pdl_trigger();
  pdl_wait();
  const bool is_v = blockIdx.z == 1;
  const int g = blockIdx.y, page = (int)ld_global_4(pages + blockIdx.x);
  const size_t bytes = (size_t)page_size * HD;
  __nv_bfloat16* out = (is_v ? v_out : k_out) + ((size_t)blockIdx.x * n_kv_heads + g) * bytes;
  if (page < 0 || page >= n_pages) {
    if (status && threadIdx.x == 0) atomicOr(status, FG_STATUS_BAD_PAGE);
    for (size_t i = threadIdx.x; i < bytes / 8; i += EXPAND_THREADS) reinterpret_cast<uint4*>(out)[i] = make_uint4(0, 0, 0, 0);
    return;
  }
  const size_t block = (size_t)page * n_kv_heads + g;
  const float scale = __uint_as_float(ld_global_4((is_v ? v_scales : k_scales) + block));
  expand_block<HD>((is_v ? v_pages : k_pages) + block * bytes, out, scale, page_size, is_v, 0, page_size);
}

// For prompt portions: blocks walk the (page, head) pairs that the sequences of two and more new tokens read.  Bound by
// its bytes: a code in, two bytes out for each entry.
template <int HD>
__global__ void __launch_bounds__(EXPAND_THREADS)
kv8_expand_kernel(const unsigned char* k_pages, const unsigned char* v_pages, const float* k_scales, const float* v_scales,
                  const int* __restrict__ block_table, int table_width, const int* __restrict__ seq_slot,
                  const int* __restrict__ seq_start, const int* __restrict__ seq_cached, int n_seqs, __nv_bfloat16* k_out,
                  __nv_bfloat16* v_out, int page_size, int n_pages, int n_kv_heads, int window, int* status) {
  __shared__ int s_slot[EXPAND_THREADS], s_cached[EXPAND_THREADS], s_last[EXPAND_THREADS], s_n;
  pdl_trigger();
  const size_t bytes = (size_t)page_size * HD;
  const int grid = gridDim.x;
  bool waited = false;
  int before = 0;  // items of the sequences before, modulo the grid
  for (int base = 0; base < n_seqs; base += EXPAND_THREADS) {
    // the sequences of two and more tokens among the next EXPAND_THREADS, in any order of their own: every block must
    // find the same one, so the first warp alone lists them
    __syncthreads();
    if (threadIdx.x < 32) {
      int n = 0;
      for (int s0 = base; s0 < min(n_seqs, base + EXPAND_THREADS); s0 += 32) {
        const int s = s0 + (int)threadIdx.x;
        const int slot = s < n_seqs ? seq_slot[s] : -1;
        const int fresh = slot >= 0 ? seq_start[s + 1] - seq_start[s] : 0;
        const unsigned some = __ballot_sync(0xffffffffu, fresh >= 2);
        if (fresh >= 2) {
          const int at = n + __popc(some & ((1u << threadIdx.x) - 1u));
          s_slot[at] = slot;
          s_cached[at] = seq_cached[s];
          s_last[at] = seq_cached[s] + fresh - 1;
        }
        n += __popc(some);
      }
      if (threadIdx.x == 0) s_n = n;
    }
    __syncthreads();
    for (int s = 0; s < s_n; ++s) {
      const int last = s_last[s];
      const int lo_page = first_visible(s_cached[s], window) / page_size;
      const int items = (last / page_size - lo_page + 1) * n_kv_heads * 2;
      // the blocks take the items of all sequences in turn
      const int first = ((int)blockIdx.x - before + grid) % grid;
      before = (before + items) % grid;
      for (int it = first; it < items; it += grid) {
        const bool is_v = it & 1;
        const int g = (it >> 1) % n_kv_heads, logical = lo_page + (it >> 1) / n_kv_heads;
        const int page = logical < table_width ? block_table[(size_t)s_slot[s] * table_width + logical] : -1;
        if (page < 0 || page >= n_pages) {
          if (status && threadIdx.x == 0) atomicOr(status, FG_STATUS_BAD_PAGE);
          continue;
        }
        if (!waited) {
          pdl_wait();
          waited = true;
        }
        const size_t block = (size_t)page * n_kv_heads + g;
        const float scale = __uint_as_float(ld_global_4((is_v ? v_scales : k_scales) + block));
        expand_block<HD>((is_v ? v_pages : k_pages) + block * bytes, (is_v ? v_out : k_out) + block * bytes, scale, page_size,
                         is_v, 0, last - logical * page_size + 1);
      }
    }
  }
  if (!waited) pdl_wait();
}

}  // namespace fg_kv8
