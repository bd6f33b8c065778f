// What the two products with 4-bit weights share (see gemm_w4.cu for the weights' form).
#pragma once

#include "skinny_product.cuh"

namespace fg_w4 {

// the columns 2 i and 2 i + 1 of a word's eight, as bfloat16: one `and-or` with 0x4300 makes the pair 128 + code
__device__ __forceinline__ uint32_t weights_of(uint32_t w, int i) {
  uint32_t v;
  asm("lop3.b32 %0, %1, 0x000f000f, 0x43004300, 0xea;\n" : "=r"(v) : "r"(w >> (4 * i)));  // (a & b) | c
  const uint32_t shift = 0x43084308u;  // 136
  const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), *reinterpret_cast<const __nv_bfloat162*>(&shift));
  return *reinterpret_cast<const uint32_t*>(&d);
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
__device__ __forceinline__ float ld_cluster(uint32_t addr, uint32_t rank) {
  uint32_t remote;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(remote) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];\n" : "=f"(v) : "r"(remote) : "memory");
  return v;
}

struct Epilogue4 {
  const __nv_bfloat16* bias;  // [N] or null
  int act;                    // ACT_*; with `gated`: 1 for a relu gate
  bool gated;                 // rows are gate and up in blocks of 8: y[M, N / 2]
};

}  // namespace fg_w4
