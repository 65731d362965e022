// Ragged serving over a paged KV cache: entry points, the rotation table,
// the per-head norm + rotation kernel and the any-layout attention kernel.
#include <cuda_runtime.h>
#include <math.h>

#include <algorithm>

#include "op_entry.cuh"
#include "paged_sched.cuh"
#include "paged_tma.cuh"
#include "rope_dev.cuh"

namespace nnz {

namespace {

// ---------------------------------------------------------------------------
// rotation table
// ---------------------------------------------------------------------------
__global__ void rope_table_kernel(double l2theta, uint32_t half, uint32_t positions, float2* table) {
  const uint64_t n = (uint64_t)positions * half;
  for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (uint64_t)gridDim.x * blockDim.x) {
    const double f = exp2(-l2theta * (double)(i % half) / (double)half);
    double s, c;
    sincos((double)(i / half) * f, &s, &c);
    table[i] = make_float2((float)c, (float)s);
  }
}

// ---------------------------------------------------------------------------
// per-head RMSNorm + rotation -> q_out and the pages
// ---------------------------------------------------------------------------
// y = x * rsqrt(mean(x^2) + eps) * w over one head, then each pair (a, b) ->
// (a cos - b sin, a sin + b cos); pairs are (2i, 2i + 1) or (i, i + HD / 2).
// Bound by bytes: every head is read and written once in 16-byte chunks, HD /
// 8 lanes to a head, f32 arithmetic, one rounding.  One CTA of 4 warps per
// token; a thread asks for all its chunks (up to kNrUnroll) before it waits
// for the position, the table row that depends on it, or the slot, so a CTA
// pays two memory latencies and the 8 CTAs of an SM keep 64 KB in flight.
// Measured (16 / 8 heads of 128): 8191 tokens 29.4 us, 4.7 TB/s (memory is the
// first reason of stalls, and 2.6 of 4 instructions a cycle issue); 512 tokens 4.0
// us, 1 token 2.45 us, which is the launch and those two latencies.
// A lane holds four pairs of a head whole: 8 elements in a row (pairwise), or 4
// of each half (half split: two 8-byte chunks; with 16-byte chunks the pairs
// would meet by 8 shuffles more per chunk).
constexpr int kNrThreads = 128, kNrUnroll = 4;

template <int STYLE>
__device__ __forceinline__ uint4 nr_load(const uint16_t* head, uint32_t hl, int hd) {
  if constexpr (STYLE == ROPE_PAIRWISE) return __ldcs(reinterpret_cast<const uint4*>(head) + hl);
  const uint2 a = __ldcs(reinterpret_cast<const uint2*>(head) + hl), b = __ldcs(reinterpret_cast<const uint2*>(head + hd / 2) + hl);
  return make_uint4(a.x, a.y, b.x, b.y);
}
template <int STYLE>
__device__ __forceinline__ void nr_store(uint16_t* head, uint32_t hl, int hd, const uint4& v) {
  if constexpr (STYLE == ROPE_PAIRWISE) {
    reinterpret_cast<uint4*>(head)[hl] = v;
  } else {
    reinterpret_cast<uint2*>(head)[hl] = make_uint2(v.x, v.y);
    reinterpret_cast<uint2*>(head + hd / 2)[hl] = make_uint2(v.z, v.w);
  }
}

template <typename T, int HD, int STYLE>
__global__ void __launch_bounds__(kNrThreads, 8) norm_rope_kernel(const NormRopeArgs a) {
  constexpr int LPH = HD / 8;                          // lanes per head
  constexpr uint32_t HPS = kNrThreads / LPH;            // heads per step of the CTA
  const uint32_t tok = blockIdx.x;
  const uint32_t hl = threadIdx.x % LPH, hg = threadIdx.x / LPH;
  const uint32_t n_kv = a.kv.n_kv, heads = a.n_q + 2 * n_kv;
  const uint16_t* src = a.qkv + (int64_t)tok * a.qkv_stride;
  uint4 u[kNrUnroll];
#pragma unroll
  for (int i = 0; i < kNrUnroll; ++i) {
    const uint32_t h = hg + i * HPS;
    u[i] = h < heads ? nr_load<STYLE>(src + h * HD, hl, HD) : make_uint4(0u, 0u, 0u, 0u);
  }
  const int pos = a.positions[tok];
  const long long slot = a.slots[tok];
  // element e of the lane: 8 hl + e, or 4 hl + e of the first (e < 4) or second half
  float4 wq[2], wk[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t at = STYLE == ROPE_PAIRWISE ? hl * 8 + 4 * i : hl * 4 + i * (HD / 2);
    wq[i] = __ldg(reinterpret_cast<const float4*>(a.q_norm + at));
    wk[i] = __ldg(reinterpret_cast<const float4*>(a.k_norm + at));
  }
  const bool bad_pos = pos < 0 || (uint32_t)pos >= a.table_positions;
  const bool bad_slot = slot >= (long long)a.kv.num_pages * a.kv.page_size;
  const bool bad = bad_pos || bad_slot;
  if (bad && threadIdx.x == 0) atomicOr(a.err, bad_pos ? ERR_BAD_POS : ERR_BAD_PAGE);
  float4 cs[2];             // (cos, sin) of the lane's pairs 4 hl .. 4 hl + 3
  {
    const float4* tab = reinterpret_cast<const float4*>(a.table + (size_t)(bad_pos ? 0 : pos) * (HD / 2)) + hl * 2;
    cs[0] = __ldg(tab);
    cs[1] = __ldg(tab + 1);
  }
  int64_t page_off = 0;
  if (!bad && slot >= 0) {
    const long long pg = slot >> 32 ? slot / a.kv.page_size : (long long)((uint32_t)slot / a.kv.page_size);
    page_off = pg * a.kv.page_stride + (slot - pg * a.kv.page_size) * a.kv.token_stride;
  }
  for (uint32_t h0 = 0; h0 < heads; h0 += kNrUnroll * HPS) {
#pragma unroll
    for (int i = 0; i < kNrUnroll; ++i) {
      const uint32_t h = h0 + i * HPS + hg;
      if (h0 + i * HPS >= heads) break;               // the same for every thread
      const bool is_q = h < a.n_q, is_v = h >= a.n_q + n_kv;
      uint4 y = u[i];
      if (!__all_sync(0xffffffffu, is_v)) {            // a query or key head among the warp's
        const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
        float x[8], ss = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = T16<T>::to_f2(w[e]);
          x[2 * e] = f.x;
          x[2 * e + 1] = f.y;
          ss = fmaf(f.x, f.x, ss);
          ss = fmaf(f.y, f.y, ss);
        }
#pragma unroll
        for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float r = rsqrtf(ss * (1.f / HD) + a.eps);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float4 nw = is_q ? wq[e] : wk[e];
          x[4 * e] *= r * nw.x;
          x[4 * e + 1] *= r * nw.y;
          x[4 * e + 2] *= r * nw.z;
          x[4 * e + 3] *= r * nw.w;
        }
        const float c[4] = {cs[0].x, cs[0].z, cs[1].x, cs[1].z}, s[4] = {cs[0].y, cs[0].w, cs[1].y, cs[1].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int ia = STYLE == ROPE_PAIRWISE ? 2 * e : e, ib = STYLE == ROPE_PAIRWISE ? 2 * e + 1 : e + 4;
          const float p = x[ia], q = x[ib];
          x[ia] = p * c[e] - q * s[e];
          x[ib] = p * s[e] + q * c[e];
        }
        if (!is_v)
          y = make_uint4(T16<T>::pack(x[0], x[1]), T16<T>::pack(x[2], x[3]), T16<T>::pack(x[4], x[5]), T16<T>::pack(x[6], x[7]));
      }
      if (is_q) {
        if (bad) y = make_uint4(0u, 0u, 0u, 0u);
        nr_store<STYLE>(a.q_out + (int64_t)tok * a.q_stride + h * HD, hl, HD, y);
      } else if (h < heads && !bad && slot >= 0) {
        const uint32_t kh = h - a.n_q - (is_v ? n_kv : 0u);
        nr_store<STYLE>((is_v ? a.kv.v : a.kv.k) + page_off + (int64_t)kh * a.kv.head_stride, hl, HD, y);
      }
      const uint32_t hn = h + kNrUnroll * HPS;
      if (hn < heads) u[i] = nr_load<STYLE>(src + hn * HD, hl, HD);
    }
  }
}

// ---------------------------------------------------------------------------
// attention over any page size and strides: one warp per (row, query head)
// ---------------------------------------------------------------------------
// Scores one key at a time (HD / 32 elements per lane, warp sum), online
// softmax in f32.  No tensor cores and no split over the keys: pages that the
// tiled kernels cannot load (a size that is no multiple of 8) are served
// right, not fast.  Bound by the latency of a key's loads and warp sum: 64
// single tokens over 2017 .. 4032 keys 2629 us with pages of 12, against 139 us
// with pages of 8 in the streaming kernel.
template <typename T, int HD>
__global__ void __launch_bounds__(128) paged_attn_any_kernel(const PagedAttnArgs a) {
  constexpr int EPL = HD / 32;   // elements per lane, in 2-element words
  const int lane = threadIdx.x & 31;
  if (blockIdx.x == 0)      // ranges and lengths are looked at here: no row need come across them
    for (uint32_t s = threadIdx.x; s < a.num_seqs; s += blockDim.x)
      if (seq_bad(a, seq_info(a, s))) atomicOr(a.err, ERR_BAD_PAGE);
  const uint64_t unit = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const uint32_t row = (uint32_t)(unit / a.n_q), h = (uint32_t)(unit % a.n_q);
  if (row >= a.tokens) return;
  // the sequence of this row: the last s with q_start[s] <= row
  uint32_t lo = 0, hi = a.num_seqs;
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if ((int64_t)a.q_start[mid] <= (int64_t)row) lo = mid;
    else hi = mid;
  }
  const int64_t qs = a.q_start[lo], qe = a.q_start[lo + 1];
  if (row < qs || row >= qe || qs < 0 || row - qs >= (int64_t)a.max_new) return;
  const int64_t cap = (int64_t)a.table_stride * a.kv.page_size;
  int64_t len = a.kv_len[lo];
  bool bad = false;         // a page outside the pool
  const int64_t last = min(len, len - (qe - qs) + (row - qs) + 1);   // keys [0, last) are visible
  len = min(last, cap);
  const uint16_t* qp = a.q + (int64_t)row * a.q_stride + h * HD;
  float q[EPL], o[EPL];
#pragma unroll
  for (int e = 0; e < EPL; e += 2) {
    const float2 f = T16<T>::to_f2(*reinterpret_cast<const uint32_t*>(qp + lane * EPL + e));
    q[e] = f.x * a.scale;
    q[e + 1] = f.y * a.scale;
    o[e] = o[e + 1] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  const int64_t head_off = (int64_t)(h / (a.n_q / a.kv.n_kv)) * a.kv.head_stride + lane * EPL;
  const int* pages = a.page_table + (size_t)lo * a.table_stride;
  for (int64_t j0 = 0; j0 < len; j0 += a.kv.page_size) {
    const int pg = pages[j0 / a.kv.page_size];
    if (pg >= (int64_t)a.kv.num_pages) bad = true;
    if (pg < 0 || (uint32_t)pg >= a.kv.num_pages) continue;
    const int64_t base = (int64_t)pg * a.kv.page_stride + head_off;
    const int n = (int)min((int64_t)a.kv.page_size, len - j0);
    for (int t = 0; t < n; ++t) {
      const uint16_t* kp = a.kv.k + base + t * a.kv.token_stride;
      const uint16_t* vp = a.kv.v + base + t * a.kv.token_stride;
      float s = 0.f, v[EPL];
#pragma unroll
      for (int e = 0; e < EPL; e += 2) {
        const float2 f = T16<T>::to_f2(*reinterpret_cast<const uint32_t*>(kp + e));
        const float2 g = T16<T>::to_f2(*reinterpret_cast<const uint32_t*>(vp + e));
        s = fmaf(q[e], f.x, fmaf(q[e + 1], f.y, s));
        v[e] = g.x;
        v[e + 1] = g.y;
      }
      s = warp_sum(s);
      if (s > m) {
        const float c = expf(m - s);   // 0 at the first key
        l *= c;
#pragma unroll
        for (int e = 0; e < EPL; ++e) o[e] *= c;
        m = s;
      }
      const float p = s == -INFINITY ? 0.f : expf(s - m);
      l += p;
#pragma unroll
      for (int e = 0; e < EPL; ++e) o[e] = fmaf(p, v[e], o[e]);
    }
  }
  if (bad && lane == 0) atomicOr(a.err, ERR_BAD_PAGE);
  const float r = l == 0.f ? 0.f : 1.f / l;
  uint16_t* op = a.out + (int64_t)row * a.out_stride + h * HD + lane * EPL;
#pragma unroll
  for (int e = 0; e < EPL; e += 2) *reinterpret_cast<uint32_t*>(op + e) = T16<T>::pack(o[e] * r, o[e + 1] * r);
}

}  // namespace

namespace {

// The tiled kernel's parts, [HD / 4][R][4] (128 KB each: one CTA alone would
// need 13 us for four of them): a block takes 32 rows of one split task, lane =
// row, a warp HD / 8 dims, so every load is 512 bytes in a row and a lane's
// output whole sectors.  About 6 us for 19 MB of parts, launch included.
template <typename T, int HD>
__global__ void __launch_bounds__(256) paged_merge_tile_kernel(const PagedAttnArgs a, const PartWs ws) {
  constexpr int N4 = HD / 32;          // float4 per thread
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t G = a.n_q / a.kv.n_kv;
  pdl_wait();
  const PartHeader h = ws.head[blockIdx.x];
  const uint32_t row = blockIdx.y * 32 + lane;
  if (row >= h.rows || h.parts == 0) return;
  float m = -INFINITY, l = 0.f, o[N4][4];
#pragma unroll
  for (int i = 0; i < N4; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
  for (uint32_t k0 = 0; k0 < h.parts; k0 += 2) {
    float pm[2], pl[2];
    float4 po[2][N4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t k = k0 + j;
      pm[j] = -INFINITY;
      pl[j] = 0.f;
#pragma unroll
      for (int i = 0; i < N4; ++i) po[j][i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (k < h.parts) {
        const float* p = ws.slot(blockIdx.x + k, k == 0 ? 1 : 0, HD);
        pm[j] = __ldcg(p + row);
        pl[j] = __ldcg(p + ws.R + row);
        const float4* q = reinterpret_cast<const float4*>(p + 2 * ws.R) + row;
#pragma unroll
        for (int i = 0; i < N4; ++i) po[j][i] = __ldcg(q + (size_t)(warp * N4 + i) * ws.R);
      }
    }
    const float mn = fmaxf(m, fmaxf(pm[0], pm[1]));
    const float ms = mn == -INFINITY ? 0.f : mn;
    const float c = exp2f(m - ms), f0 = exp2f(pm[0] - ms), f1 = exp2f(pm[1] - ms);
    m = mn;
    l = l * c + f0 * pl[0] + f1 * pl[1];
#pragma unroll
    for (int i = 0; i < N4; ++i) {
      o[i][0] = o[i][0] * c + f0 * po[0][i].x + f1 * po[1][i].x;
      o[i][1] = o[i][1] * c + f0 * po[0][i].y + f1 * po[1][i].y;
      o[i][2] = o[i][2] * c + f0 * po[0][i].z + f1 * po[1][i].z;
      o[i][3] = o[i][3] * c + f0 * po[0][i].w + f1 * po[1][i].w;
    }
  }
  const float il = l == 0.f ? 0.f : 1.f / l;
  uint16_t* op = a.out + ((int64_t)h.row0 + row / G) * a.out_stride + ((int64_t)h.kvh * G + row % G) * HD + warp * N4 * 4;
#pragma unroll
  for (int i = 0; i < N4; i += 2)
    *reinterpret_cast<uint4*>(op + 4 * i) = make_uint4(T16<T>::pack(o[i][0] * il, o[i][1] * il), T16<T>::pack(o[i][2] * il, o[i][3] * il),
                                                       T16<T>::pack(o[i + 1][0] * il, o[i + 1][1] * il),
                                                       T16<T>::pack(o[i + 1][2] * il, o[i + 1][3] * il));
}

}  // namespace

cudaError_t paged_merge_tile_launch(const PagedAttnArgs& a, const PartWs& ws, uint32_t workers, int dtype, int hd, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(workers, (ws.R + 31) / 32);
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (dtype == RD_F16)
    return hd == 128 ? cudaLaunchKernelEx(&cfg, &paged_merge_tile_kernel<__half, 128>, a, ws)
                     : cudaLaunchKernelEx(&cfg, &paged_merge_tile_kernel<__half, 64>, a, ws);
  return hd == 128 ? cudaLaunchKernelEx(&cfg, &paged_merge_tile_kernel<__nv_bfloat16, 128>, a, ws)
                   : cudaLaunchKernelEx(&cfg, &paged_merge_tile_kernel<__nv_bfloat16, 64>, a, ws);
}

namespace {

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encode_fn() {
  static const EncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeFn>(p);
  }();
  return fn;
}

bool encode16(CUtensorMap* tm, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box) {
  const EncodeFn enc = encode_fn();
  const cuuint32_t es[5] = {1, 1, 1, 1, 1};
  return enc && enc(tm, CU_TENSOR_MAP_DATA_TYPE_UINT16, (cuuint32_t)rank, const_cast<void*>(base), dims, strides, box, es,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace

bool paged_tensor_map(CUtensorMap* tm, const PagedPool& kv, const void* base, int hd, uint32_t keys) {
  const cuuint64_t dims[4] = {(cuuint64_t)hd, kv.page_size, kv.n_kv, kv.num_pages};
  // a dimension of one element takes any stride
  const cuuint64_t strides[3] = {(cuuint64_t)kv.token_stride * 2, (cuuint64_t)(kv.n_kv > 1 ? kv.head_stride : kv.token_stride) * 2,
                                 (cuuint64_t)(kv.num_pages > 1 ? kv.page_stride : kv.token_stride) * 2};
  const cuuint32_t box[4] = {64, keys, 1, 1};
  return encode16(tm, base, 4, dims, strides, box);
}

bool paged_q_map(CUtensorMap* tm, const PagedAttnArgs& a, int hd, uint32_t heads, uint32_t tokens) {
  const cuuint64_t dims[3] = {(cuuint64_t)hd, a.n_q, a.tokens};
  const cuuint64_t strides[2] = {(cuuint64_t)hd * 2, (cuuint64_t)a.q_stride * 2};
  const cuuint32_t box[3] = {64, heads, tokens};
  return encode16(tm, a.q, 3, dims, strides, box);
}

cudaError_t rope_table_launch(float theta, uint32_t hd, uint32_t positions, float2* table, cudaStream_t st) {
  const uint64_t n = (uint64_t)positions * (hd / 2);
  const uint32_t grid = (uint32_t)std::min<uint64_t>((n + 255) / 256, 148 * 8);
  rope_table_kernel<<<grid, 256, 0, st>>>(log2((double)theta), hd / 2, positions, table);
  return cudaGetLastError();
}

template <typename T, int HD>
static cudaError_t norm_rope_t(const NormRopeArgs& a, cudaStream_t st) {
  if (a.rope_style == ROPE_PAIRWISE) norm_rope_kernel<T, HD, ROPE_PAIRWISE><<<a.tokens, kNrThreads, 0, st>>>(a);
  else norm_rope_kernel<T, HD, ROPE_HALF_SPLIT><<<a.tokens, kNrThreads, 0, st>>>(a);
  return cudaGetLastError();
}

cudaError_t norm_rope_launch(const NormRopeArgs& a, int dtype, int hd, cudaStream_t st) {
  if (dtype == RD_F16) return hd == 128 ? norm_rope_t<__half, 128>(a, st) : norm_rope_t<__half, 64>(a, st);
  return hd == 128 ? norm_rope_t<__nv_bfloat16, 128>(a, st) : norm_rope_t<__nv_bfloat16, 64>(a, st);
}

cudaError_t paged_attn_any_launch(const PagedAttnArgs& a, int dtype, int hd, cudaStream_t st) {
  const uint64_t grid = ((uint64_t)a.tokens * a.n_q + 3) / 4;
  if (grid > 0x7FFFFFFFull) return cudaErrorInvalidValue;
  if (dtype == RD_F16) {
    if (hd == 128) paged_attn_any_kernel<__half, 128><<<(uint32_t)grid, 128, 0, st>>>(a);
    else paged_attn_any_kernel<__half, 64><<<(uint32_t)grid, 128, 0, st>>>(a);
  } else {
    if (hd == 128) paged_attn_any_kernel<__nv_bfloat16, 128><<<(uint32_t)grid, 128, 0, st>>>(a);
    else paged_attn_any_kernel<__nv_bfloat16, 64><<<(uint32_t)grid, 128, 0, st>>>(a);
  }
  return cudaGetLastError();
}

}  // namespace nnz

using namespace nnz;

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// nullptr if `kv` can be used, else what is wrong with it.
const char* pool_error(const nnz_paged_kv* kv) {
  if (!kv || !kv->k || !kv->v) return "paged kv: null pool";
  if (kv->dtype != NNZ_DT_F16 && kv->dtype != NNZ_DT_BF16) return "paged kv: dtype must be f16 or bf16";
  if (kv->head_dim != 64 && kv->head_dim != 128) return "paged kv: head_dim must be 64 or 128";
  if (kv->num_kv_heads == 0 || kv->num_kv_heads > 65535) return "paged kv: num_kv_heads";
  if (kv->num_pages == 0 || kv->num_pages > 0x7FFFFFFFu) return "paged kv: num_pages";
  if (kv->page_size == 0 || kv->page_size > 65536) return "paged kv: page_size must be 1 .. 65536";
  if (kv->page_stride % 8 || kv->head_stride % 8 || kv->token_stride % 8 || kv->page_stride < 0 || kv->head_stride < 0 ||
      kv->token_stride < 0)
    return "paged kv: strides must be multiples of 8 elements";
  if (kv->token_stride < kv->head_dim || (kv->num_kv_heads > 1 && kv->head_stride < kv->head_dim) ||
      (kv->num_pages > 1 && kv->page_stride < kv->head_dim))
    return "paged kv: strides smaller than a head";
  if (!aligned16(kv->k) || !aligned16(kv->v)) return "paged kv: k and v must be 16-byte aligned";
  return nullptr;
}

PagedPool pool_of(const nnz_paged_kv* kv) {
  return {static_cast<uint16_t*>(kv->k), static_cast<uint16_t*>(kv->v), kv->num_pages, kv->page_size, kv->num_kv_heads,
          kv->page_stride, kv->head_stride, kv->token_stride};
}

int dtype_of(const nnz_paged_kv* kv) { return kv->dtype == NNZ_DT_BF16 ? RD_BF16 : RD_F16; }

}  // namespace

extern "C" {

int nnz_rope_table(float theta, uint32_t head_dim, uint32_t positions, float* table, void* stream) {
  if (!table || positions == 0 || head_dim == 0 || head_dim % 2 || !(theta > 0.f) || (reinterpret_cast<uintptr_t>(table) & 7))
    return refuse(NNZ_EINVAL, "nnz_rope_table: invalid arguments");
  return cuda_rc(rope_table_launch(theta, head_dim, positions, reinterpret_cast<float2*>(table), static_cast<cudaStream_t>(stream)),
                 "nnz_rope_table");
}

int nnz_qk_norm_rope_paged(const nnz_paged_kv* kv, const nnz_norm_rope_args* p, void* stream) {
  if (const char* why = pool_error(kv)) return refuse(NNZ_EINVAL, why);
  if (!p) return refuse(NNZ_EINVAL, "nnz_qk_norm_rope_paged: null argument");
  if (p->tokens == 0) return NNZ_OK;
  if (!p->qkv || !p->q_norm || !p->k_norm || !p->rope_table || !p->positions || !p->slots || !p->q_out)
    return refuse(NNZ_EINVAL, "nnz_qk_norm_rope_paged: null argument");
  const int64_t hd = kv->head_dim;
  if (p->num_query_heads == 0 || p->num_query_heads > 65535 || p->tokens > 0x7FFFFFFFu || p->table_positions == 0 ||
      (p->rope_style != NNZ_ROPE_PAIRWISE && p->rope_style != NNZ_ROPE_HALF_SPLIT) || !(p->eps >= 0.f))
    return refuse(NNZ_EINVAL, "nnz_qk_norm_rope_paged: heads, tokens, table, eps or rope_style");
  if (p->qkv_stride % 8 || p->qkv_stride < (p->num_query_heads + 2 * (int64_t)kv->num_kv_heads) * hd || p->q_stride % 8 ||
      p->q_stride < p->num_query_heads * hd)
    return refuse(NNZ_EINVAL, "nnz_qk_norm_rope_paged: row strides must be multiples of 8 elements that hold the heads");
  if (!aligned16(p->qkv) || !aligned16(p->q_out) || !aligned16(p->q_norm) || !aligned16(p->k_norm) ||
      (reinterpret_cast<uintptr_t>(p->rope_table) & 15))
    return refuse(NNZ_EINVAL, "nnz_qk_norm_rope_paged: pointers must be 16-byte aligned");
  NormRopeArgs a{};
  int sms = 0;
  if (const int rc = op_device(&a.err, &sms)) return rc;
  a.kv = pool_of(kv);
  a.qkv = static_cast<const uint16_t*>(p->qkv);
  a.qkv_stride = p->qkv_stride;
  a.tokens = p->tokens;
  a.n_q = p->num_query_heads;
  a.q_norm = p->q_norm;
  a.k_norm = p->k_norm;
  a.eps = p->eps;
  a.rope_style = p->rope_style;
  a.table = reinterpret_cast<const float2*>(p->rope_table);
  a.table_positions = p->table_positions;
  a.positions = p->positions;
  a.slots = reinterpret_cast<const long long*>(p->slots);
  a.q_out = static_cast<uint16_t*>(p->q_out);
  a.q_stride = p->q_stride;
  return cuda_rc(norm_rope_launch(a, dtype_of(kv), (int)hd, static_cast<cudaStream_t>(stream)), "nnz_qk_norm_rope_paged");
}

size_t nnz_paged_attn_workspace(const nnz_paged_kv* kv, uint32_t num_query_heads) {
  if (pool_error(kv) || num_query_heads == 0 || num_query_heads % kv->num_kv_heads) return 0;
  int* err = nullptr;
  int sms = 0;
  if (op_device(&err, &sms)) sms = 148;   // no device: the size for a full B200
  return std::max(paged_stream_ws(sms, (int)kv->head_dim), paged_umma_ws(sms, (int)kv->head_dim));
}

int nnz_paged_attn(const nnz_paged_kv* kv, const nnz_paged_attn_args* p, void* stream) {
  if (const char* why = pool_error(kv)) return refuse(NNZ_EINVAL, why);
  if (!p) return refuse(NNZ_EINVAL, "nnz_paged_attn: null argument");
  const int64_t hd = kv->head_dim;
  if (p->num_query_heads == 0 || p->num_query_heads % kv->num_kv_heads || p->num_query_heads / kv->num_kv_heads > 64)
    return refuse(NNZ_EINVAL, "nnz_paged_attn: num_query_heads must be a multiple (<= 64x) of num_kv_heads");
  if (p->tokens == 0 || p->num_seqs == 0 || p->max_new == 0) return NNZ_OK;
  if (!p->q || !p->q_start || !p->kv_len || !p->page_table || !p->out || !p->workspace)
    return refuse(NNZ_EINVAL, "nnz_paged_attn: null argument");
  if (p->tokens > 0x7FFFFFFFu || p->num_seqs > 0x7FFFFFFFu || p->table_stride == 0 ||
      (uint64_t)p->table_stride * kv->page_size > 0x7FFF0000u || !(p->scale >= 0.f && isfinite(p->scale)))
    return refuse(NNZ_EINVAL, "nnz_paged_attn: tokens, num_seqs, table_stride or scale");
  if (p->q_stride % 8 || p->q_stride < p->num_query_heads * hd || p->out_stride % 8 || p->out_stride < p->num_query_heads * hd)
    return refuse(NNZ_EINVAL, "nnz_paged_attn: row strides must be multiples of 8 elements that hold the heads");
  if (!aligned16(p->q) || !aligned16(p->out) || (reinterpret_cast<uintptr_t>(p->workspace) & 255))
    return refuse(NNZ_EINVAL, "nnz_paged_attn: q and out must be 16-byte, workspace 256-byte aligned");
  if (p->workspace_bytes < nnz_paged_attn_workspace(kv, p->num_query_heads))
    return refuse(NNZ_EINVAL, "nnz_paged_attn: workspace too small");
  PagedAttnArgs a{};
  if (const int rc = op_device(&a.err, &a.num_sms)) return rc;
  a.kv = pool_of(kv);
  a.q = static_cast<const uint16_t*>(p->q);
  a.q_stride = p->q_stride;
  a.tokens = p->tokens;
  a.n_q = p->num_query_heads;
  a.num_seqs = p->num_seqs;
  a.max_new = p->max_new;
  a.q_start = p->q_start;
  a.kv_len = p->kv_len;
  a.page_table = p->page_table;
  a.table_stride = p->table_stride;
  a.scale = p->scale > 0.f ? p->scale : 1.f / sqrtf((float)hd);
  a.out = static_cast<uint16_t*>(p->out);
  a.out_stride = p->out_stride;
  a.ws = p->workspace;
  // The tiled kernels copy boxes of 8 keys or more of one page; a page whose
  // size is no multiple of 8 would end inside one.  Up to 16 rows of a kv head
  // fit one mma tile and are streamed by single warps (us, against the tcgen05
  // kernel: 64 single tokens of 2017 .. 4032 keys 137 / 192, one of 515 7.2 /
  // 17.7, 16 rows of 8000 keys 23.8 / 26.6, 32 x 16 rows of 1000 .. 4000 keys 85
  // / 97); more rows need several such tiles, and go to tcgen05.
  const bool tiled = kv->page_size % 8 == 0;
  const uint64_t rows = (uint64_t)a.max_new * (a.n_q / a.kv.n_kv);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int dt = dtype_of(kv);
  const cudaError_t e = !tiled ? paged_attn_any_launch(a, dt, (int)hd, st)
                      : rows <= kStreamRows ? paged_stream_launch(a, dt, (int)hd, st) : paged_umma_launch(a, dt, (int)hd, st);
  return cuda_rc(e, "nnz_paged_attn");
}

}  // extern "C"
