// Ragged serving over a paged KV cache: per-head norm + rotation into pages,
// attention of new tokens over pages (declarations; include/nnz_b200.h has
// the contracts).
#pragma once
#include "common.cuh"

namespace nnz {

enum RaggedDtype : int { RD_F16 = 0, RD_BF16 = 1 };

// The two 16-bit types of the page pools.
template <typename T>
struct T16;
template <>
struct T16<__half> {
  static constexpr bool kBf16 = false;
  static __device__ __forceinline__ float2 to_f2(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <>
struct T16<__nv_bfloat16> {
  static constexpr bool kBf16 = true;
  static __device__ __forceinline__ float2 to_f2(uint32_t u) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

// Not 0: a non-finite element among the two (exponent all ones).
template <bool BF16>
__device__ __forceinline__ uint32_t bad_any(uint32_t w) {
  constexpr uint32_t e = BF16 ? 0x7F807F80u : 0x7C007C00u, one = BF16 ? 0x00800080u : 0x04000400u;
  return ((w & e) + one) & 0x80008000u;
}

// A page pool as the kernels see it (strides in elements).
struct PagedPool {
  uint16_t* k;
  uint16_t* v;
  uint32_t num_pages, page_size, n_kv;
  int64_t page_stride, head_stride, token_stride;
};

struct NormRopeArgs {
  PagedPool kv;
  const uint16_t* qkv;
  int64_t qkv_stride;
  uint32_t tokens, n_q;
  const float* q_norm;
  const float* k_norm;
  float eps;
  int rope_style;
  const float2* table;
  uint32_t table_positions;
  const int* positions;
  const long long* slots;
  uint16_t* q_out;
  int64_t q_stride;
  int* err;
};

struct PagedAttnArgs {
  PagedPool kv;
  const uint16_t* q;
  int64_t q_stride;
  uint32_t tokens, n_q, num_seqs, max_new;
  const int* q_start;
  const int* kv_len;
  const int* page_table;
  uint32_t table_stride;
  float scale;
  uint16_t* out;
  int64_t out_stride;
  void* ws;
  int num_sms;
  int* err;
};

cudaError_t rope_table_launch(float theta, uint32_t hd, uint32_t positions, float2* table, cudaStream_t st);
cudaError_t norm_rope_launch(const NormRopeArgs& a, int dtype, int hd, cudaStream_t st);
// Any page size and any strides: one warp per (new token, query head).
cudaError_t paged_attn_any_launch(const PagedAttnArgs& a, int dtype, int hd, cudaStream_t st);

}  // namespace nnz
