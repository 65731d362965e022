// TMA access to a page pool: a 4-D tensor map [page][kv head][token][d] of
// 16-bit elements whose boxes are `keys` tokens x 64 dims of one page and
// head, 128-byte swizzled.
#pragma once
#include <cuda.h>

#include "device_cache.cuh"
#include "paged.cuh"

namespace nnz {

// One lane of the warp, known as such to the compiler: behind a plain test of
// the lane it takes every tcgen05.mma for divergent code (S: 900 -> 585 cycles
// for its 8 instructions, P V: 1900 -> 700).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred q;\n elect.sync _|q, 0xffffffff;\n selp.u32 %0, 1, 0, q;\n}\n" : "=r"(p));
  return p != 0;
}

// x: dim (0 or 64), y: token within the page.
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* tm, int x, int y, int head, int page, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(tm)), "r"(x), "r"(y), "r"(head), "r"(page), "r"(smem_u32(bar))
      : "memory");
}

// False if the driver entry point is missing or it refuses the strides.
bool paged_tensor_map(CUtensorMap* tm, const PagedPool& kv, const void* base, int hd, uint32_t keys);
// Rows of q as [token][head][d]: boxes of `heads` heads x `tokens` tokens x 64 dims.
bool paged_q_map(CUtensorMap* tm, const PagedAttnArgs& a, int hd, uint32_t heads, uint32_t tokens);

}  // namespace nnz
