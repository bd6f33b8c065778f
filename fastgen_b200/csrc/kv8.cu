// The paged cache in 8 bits (see kv8.cuh for what it holds): the write of a step's keys and values with the
// rotation, the codes' values in bfloat16, and attention of single tokens.  Compiled for one head size,
// -DFG_HEAD_DIM=<64, 128 or 256>.
#include <string.h>

#include "kv8_attention.cuh"
#include "kv8_pages.cuh"

#ifndef FG_HEAD_DIM
#error "compile with -DFG_HEAD_DIM=<head size>"
#endif
static_assert(FG_HEAD_DIM == 64 || FG_HEAD_DIM == 128 || FG_HEAD_DIM == 256, "head sizes 64, 128 and 256");

static int check_pages(const char* name, const void* k_pages, const void* v_pages, const float* k_scales,
                       const float* v_scales, int page_size, int n_pages, int n_kv_heads, int head_dim) {
  FG_CHECK_ARG(head_dim == FG_HEAD_DIM, "%s: library built for head size %d, got %d", name, FG_HEAD_DIM, head_dim);
  FG_CHECK_ARG(page_size >= 16 && page_size <= 256 && (page_size & (page_size - 1)) == 0,
               "%s: pages of %d slots are not supported (powers of two from 16 to 256)", name, page_size);
  FG_CHECK_ARG(n_kv_heads > 0 && n_kv_heads <= 8192 && n_pages > 0, "%s: %d key/value heads, %d pages", name, n_kv_heads, n_pages);
  FG_CHECK_ARG(k_pages && v_pages && k_scales && v_scales, "%s: pools and scales are needed", name);
  FG_CHECK_ARG((((uintptr_t)k_pages | (uintptr_t)v_pages) & 15) == 0, "%s: pools must be 16-byte aligned", name);
  return 0;
}

// Queries rotated into q_out [T, n_heads * HD]; rotated keys and values into their pages.  Options as in
// fg_rope_kv_write.  A sequence's tokens are neighbours in the step, in ascending order of position.
extern "C" int fg_kv8_write(const void* q, int q_stride, void* q_out, const void* k, int k_stride, const void* v, int v_stride,
                            const int* pos, const int* req, const float* freqs, const float* v_freqs, void* k_pages,
                            void* v_pages, float* k_scales, float* v_scales, const int* block_table, int table_width,
                            int page_size, int n_pages, int n_tokens, int n_heads, int n_kv_heads, int head_dim, int* status,
                            const float* rstd, const float* qn_w, const float* kn_w, int rstd_heads, float magnitude,
                            int rot_pairs, cudaStream_t stream) {
  using namespace fg_kv8;
  if (n_tokens == 0) return 0;
  if (check_pages("fg_kv8_write", k_pages, v_pages, k_scales, v_scales, page_size, n_pages, n_kv_heads, head_dim)) return -1;
  FG_CHECK_ARG(n_heads > 0 && n_heads % n_kv_heads == 0, "fg_kv8_write: %d heads over %d kv heads", n_heads, n_kv_heads);
  constexpr int ALIGN = 2 * (FG_HEAD_DIM / 32);  // a lane's part of a row
  const bool vec = (((uintptr_t)q | (uintptr_t)q_out | (uintptr_t)k | (uintptr_t)v) % ALIGN) == 0 &&
                   ((2 * (long long)q_stride) % ALIGN) == 0 && ((2 * (long long)k_stride) % ALIGN) == 0 &&
                   ((2 * (long long)v_stride) % ALIGN) == 0;
  const int q_slices = (n_heads + Q_SLICE - 1) / Q_SLICE;
  auto launch = [&](auto kern, int per) -> int {
    const int stretch = WRITE_WARPS * per;
    const long long blocks = (long long)(n_tokens + stretch - 1) / stretch * n_kv_heads +
                             (long long)(n_tokens + WRITE_WARPS - 1) / WRITE_WARPS * q_slices;
    FG_CHECK_ARG(blocks < (1ll << 31), "fg_kv8_write: %d tokens of %d heads", n_tokens, n_heads);
    fg_launch_pdl(kern, dim3((unsigned)blocks), dim3(WRITE_THREADS), 0, stream,
                  (const __nv_bfloat16*)q, q_stride, (__nv_bfloat16*)q_out, (const __nv_bfloat16*)k, k_stride,
                  (const __nv_bfloat16*)v, v_stride, pos, req, freqs, v_freqs, (unsigned char*)k_pages, (unsigned char*)v_pages,
                  k_scales, v_scales, block_table, table_width, page_size, n_pages, n_tokens, n_heads, n_kv_heads, status, rstd,
                  qn_w, kn_w, rstd_heads, magnitude, rot_pairs);
    return 0;
  };
  // Few tokens: a warp a token.  us by that and by four tokens a warp (32 / 8 heads of 128, pages of 64): one prompt of 256 tokens 9.4
  // and 8.6, of 512 9.6 and 9.9, of 1,024 11.6 and 10.5, two of 1,024 16.9 and 14.1; 500 single tokens 7.1 and 11.9, 1,000 10.0 and 12.0.
  // (Pages of 16, where a stretch holds four runs, want the first: 512 tokens 9.2 and 26.3, 1,024 16.6 and 27.9.)
  const int rc = n_tokens <= 512 ? launch(vec ? kv8_write_kernel<FG_HEAD_DIM, true, 1> : kv8_write_kernel<FG_HEAD_DIM, false, 1>, 1)
                                 : launch(vec ? kv8_write_kernel<FG_HEAD_DIM, true, 4> : kv8_write_kernel<FG_HEAD_DIM, false, 4>, 4);
  if (rc) return rc;
  FG_CHECK_LAUNCH("fg_kv8_write");
  return 0;
}

// What the pages pages[0 .. n) stand for, bfloat16 [n, n_kv_heads, page, HD] each, every slot of them.
extern "C" int fg_kv8_values(const void* k_pages, const void* v_pages, const float* k_scales, const float* v_scales,
                             const int* pages, int n, void* k_out, void* v_out, int page_size, int n_pages, int n_kv_heads,
                             int head_dim, int* status, cudaStream_t stream) {
  using namespace fg_kv8;
  if (n == 0) return 0;
  if (check_pages("fg_kv8_values", k_pages, v_pages, k_scales, v_scales, page_size, n_pages, n_kv_heads, head_dim)) return -1;
  FG_CHECK_ARG((((uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0, "fg_kv8_values: outputs must be 16-byte aligned");
  fg_launch_pdl(kv8_values_kernel<FG_HEAD_DIM>, dim3(n, n_kv_heads, 2), dim3(EXPAND_THREADS), 0, stream,
                (const unsigned char*)k_pages, (const unsigned char*)v_pages, k_scales, v_scales, pages,
                (__nv_bfloat16*)k_out, (__nv_bfloat16*)v_out, page_size, n_pages, n_kv_heads, status);
  FG_CHECK_LAUNCH("fg_kv8_values");
  return 0;
}

// The pages that prompt portions read (sequences that bring two tokens or more), in bfloat16 at the same page ids of a
// pool of one layer: keys and values that some query of the sequence sees, zeros in the pages' other slots.
extern "C" int fg_kv8_expand(const void* k_pages, const void* v_pages, const float* k_scales, const float* v_scales,
                             const int* block_table, int table_width, const int* seq_slot, const int* seq_start,
                             const int* seq_cached, int n_seqs, void* k_out, void* v_out, int page_size, int n_pages,
                             int n_kv_heads, int head_dim, int window, int* status, cudaStream_t stream) {
  using namespace fg_kv8;
  if (n_seqs == 0) return 0;
  if (check_pages("fg_kv8_expand", k_pages, v_pages, k_scales, v_scales, page_size, n_pages, n_kv_heads, head_dim)) return -1;
  FG_CHECK_ARG((((uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0, "fg_kv8_expand: outputs must be 16-byte aligned");
  fg_launch_pdl(kv8_expand_kernel<FG_HEAD_DIM>, dim3(8 * fg_sm_count()), dim3(EXPAND_THREADS), 0, stream,
                (const unsigned char*)k_pages, (const unsigned char*)v_pages, k_scales, v_scales, block_table, table_width,
                seq_slot, seq_start, seq_cached, n_seqs, (__nv_bfloat16*)k_out, (__nv_bfloat16*)v_out, page_size, n_pages,
                n_kv_heads, window, status);
  FG_CHECK_LAUNCH("fg_kv8_expand");
  return 0;
}

// What fg_kv8_attention_decode needs: floats of scratch, whatever the step, and zeroed counters, one for every sequence and
// slice of up to eight heads of a group, which a launch leaves at zero.
extern "C" int fg_kv8_decode_scratch_floats() {
  using namespace fg_kv8;
  return decode_blocks_per_sm<FG_HEAD_DIM>() * fg_sm_count() * 2 * MAX_COLUMNS * run_stride<FG_HEAD_DIM>();
}
static int decode_counters(int n_seqs, int n_heads, int n_kv_heads) {
  const int group = n_heads / n_kv_heads;
  return n_seqs * n_kv_heads * ((group + fg_kv8::MAX_COLUMNS - 1) / fg_kv8::MAX_COLUMNS);
}

// Attention of single tokens; pools as tensor maps made by fg_make_kv8_tensor_map, `layer` the run's index in them.
extern "C" int fg_kv8_attention_decode(const void* q, int q_stride, void* out, int out_stride, const void* k_map,
                                       const void* v_map, int layer, const float* k_scales, const float* v_scales,
                                       const int* block_table, int table_width, int page_size, int n_pages, const int* pos,
                                       const int* seq_req, const int* seq_tok, int n_seqs, int n_heads, int n_kv_heads,
                                       int head_dim, int window, float scale, float softcap, float* scratch, int scratch_floats,
                                       int* counters, int n_counters, const float* out_freqs, const float* sinks, int* status,
                                       cudaStream_t stream) {
  using namespace fg_kv8;
  if (n_seqs == 0) return 0;
  if (check_pages("fg_kv8_attention_decode", q, out, k_scales, v_scales, page_size, n_pages, n_kv_heads, head_dim)) return -1;
  FG_CHECK_ARG(n_heads > 0 && n_heads % n_kv_heads == 0 && n_seqs <= DECODE_MAX_SEQS,
               "fg_kv8_attention_decode: %d heads over %d kv heads, %d sequences (at most %d)", n_heads, n_kv_heads, n_seqs,
               DECODE_MAX_SEQS);
  FG_CHECK_ARG(scratch != nullptr && scratch_floats >= fg_kv8_decode_scratch_floats() && counters != nullptr &&
                   n_counters >= decode_counters(n_seqs, n_heads, n_kv_heads) && ((uintptr_t)scratch & 15) == 0,
               "fg_kv8_attention_decode: scratch of %d floats, %d counters are too few", scratch_floats, n_counters);
  FG_CHECK_ARG(q_stride % 8 == 0 && out_stride % 2 == 0, "fg_kv8_attention_decode: row strides %d and %d", q_stride, out_stride);
  const int group = n_heads / n_kv_heads;
  CUtensorMap km, vm;
  memcpy(&km, k_map, sizeof(CUtensorMap));
  memcpy(&vm, v_map, sizeof(CUtensorMap));
  const size_t smem = decode_smem_bytes<FG_HEAD_DIM>(n_seqs);
  auto kern = window < 0 ? (softcap > 0.f ? kv8_decode_kernel<FG_HEAD_DIM, true, true> : kv8_decode_kernel<FG_HEAD_DIM, true, false>)
                         : (softcap > 0.f ? kv8_decode_kernel<FG_HEAD_DIM, false, true> : kv8_decode_kernel<FG_HEAD_DIM, false, false>);
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  FG_CHECK_ARG(e == cudaSuccess, "fg_kv8_attention_decode: shared memory: %s", cudaGetErrorString(e));
  const float log2e = 1.4426950408889634f;
  fg_launch_pdl(kern, dim3(decode_blocks_per_sm<FG_HEAD_DIM>() * fg_sm_count()), dim3(DECODE_THREADS), smem, stream, km, vm,
                layer, k_scales, v_scales, (const __nv_bfloat16*)q, q_stride, block_table, table_width, page_size, n_pages, pos,
                seq_req, seq_tok, n_seqs, n_heads, n_kv_heads, group, window, scale * log2e, softcap * log2e,
                softcap > 0.f ? scale / softcap : 0.f, (__nv_bfloat16*)out, out_stride, scratch, counters, out_freqs, sinks,
                status);
  FG_CHECK_LAUNCH("fg_kv8_attention_decode");
  return 0;
}
