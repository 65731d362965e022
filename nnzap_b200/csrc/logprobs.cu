// Log probabilities of given tokens, the row's entropy and its most probable
// tokens, from one read of the logits (contract: nnz_token_logprobs in
// include/nnz_b200.h; the reference's softmax over the same logits is
// sampleToken, nnmetal/src/transformer.zig:3833-3869).
//
// With M = max x, s = sum exp(x - M) and t = sum exp(x - M) (x - M):
//   log p(i) = (x_i - M) - ln s,   H = -sum p ln p = ln s - t / s.
// Every thread keeps (M, s, t) of its elements and rescales them when its
// maximum grows; two such triples merge as s' = s e^d, t' = (t + s d) e^d with
// d = M - M'.  x - M is formed before the multiplication by log2 e, so the
// error stays relative to the difference, not to the logits' size.
//
// Most probable tokens cost the stream nothing but a store: every thread's
// maximum of each step (16 or 32 elements) goes to shared memory.  The k-th
// largest of 64 overall maxima (each of 4 threads) bounds the CTA's k best
// from below; the steps whose maximum reaches it (about k of them) are read
// again, 64 bytes each, and their elements that reach it sorted as 64-bit
// (value, index) keys, 32 to a list, one per lane of a warp.
//
// A row is cut over a cluster of CTAs (1 to 16) whose triples and lists meet
// in the first CTA's shared memory: no workspace, no atomics on memory, the
// same result every time.
//
// Bound by the read of the logits where there are many rows: 512 rows of
// 151936 f32 61 us, 5.1 TB/s.  64 rows of 151669 bf16 14.2 us and one row of
// 151936 f32 7.5 us are the launch of the cluster, one latency of memory, the
// selection (3 - 4 us) and the merge.
#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "device_cache.cuh"
#include "op_entry.cuh"

namespace cg = cooperative_groups;

namespace nnz {

namespace {

constexpr int kLpThreads = 256;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpVec = 4;              // 16-byte loads per thread and step
constexpr uint32_t kLpMaxCluster = 16;
constexpr float kLog2e = 1.4426950408889634f;

struct LpArgs {
  const void* x;
  uint32_t rows, n;
  int64_t stride;
  const int* tokens;
  uint32_t num_tokens, top_k;
  float* logprob;
  float* entropy;
  float* lse;
  int* top_ids;
  float* top_lp;
  int* err;
};

struct LpStat {
  float m, s, t;
};

// exp of anything below is 0 in f32; differences are cut here so that
// -infinity and the types' lowest values add 0 to t (0 times the cut).
constexpr float kLpLow = -200.f;

__device__ __forceinline__ LpStat lp_merge(const LpStat& a, const LpStat& b) {
  const float m = fmaxf(a.m, b.m);
  const float da = a.m == m ? 0.f : fmaxf(a.m - m, kLpLow), db = b.m == m ? 0.f : fmaxf(b.m - m, kLpLow);
  const float ea = expf(da), eb = expf(db);
  return {m, a.s * ea + b.s * eb, (a.t + a.s * da) * ea + (b.t + b.s * db) * eb};
}

// Larger key = larger value, then lower index; 0 = no element.
__device__ __forceinline__ unsigned long long lp_key(float v, uint32_t idx) { return argmax_pack(v + 0.f, idx); }
__device__ __forceinline__ float lp_value(unsigned long long k) {
  const uint32_t u = (uint32_t)(k >> 32);
  return __uint_as_float((u & 0x80000000u) ? (u & 0x7FFFFFFFu) : ~u);
}

__device__ __forceinline__ unsigned long long lp_exchange(unsigned long long k, int lane, int o, bool desc) {
  const unsigned long long other = __shfl_xor_sync(0xffffffffu, k, o);
  const bool keep_max = ((lane & o) == 0) == desc;
  return keep_max ? (k > other ? k : other) : (k < other ? k : other);
}

__device__ __forceinline__ uint32_t lp_exchange(uint32_t k, int lane, int o, bool desc) {
  const uint32_t other = __shfl_xor_sync(0xffffffffu, k, o);
  return ((lane & o) == 0) == desc ? max(k, other) : min(k, other);
}

// 32 keys, one per lane, into descending order (bitonic sort).
template <typename K>
__device__ __forceinline__ K lp_sort32(K k, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size *= 2)
#pragma unroll
    for (int o = size / 2; o > 0; o >>= 1) k = lp_exchange(k, lane, o, (lane & size) == 0);
  return k;
}

// The best 32 of two descending lists, descending.
template <typename K>
__device__ __forceinline__ K lp_merge32(K a, K b, int lane) {
  const K r = __shfl_sync(0xffffffffu, b, 31 - lane);
  a = a > r ? a : r;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) a = lp_exchange(a, lane, o, true);
  return a;
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

template <typename T>
__device__ __forceinline__ float lp_load1(const T* p) {
  if constexpr (std::is_same_v<T, float>) return *p;
  else if constexpr (std::is_same_v<T, __half>) return __half2float(*p);
  else return __bfloat162float(*p);
}

// The 16 / sizeof(T) elements of one 16-byte vector as floats.
template <typename T>
__device__ __forceinline__ void lp_unpack(const uint4& u, float* x) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  if constexpr (std::is_same_v<T, float>) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(w[i]);
  } else if constexpr (std::is_same_v<T, __half>) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
}

constexpr int kLpSlots = 24;      // step maxima kept per thread; longer slices keep one per 2, 4, .. steps

constexpr int kLpPool = kLpWarps * 64;

struct LpShared {
  float smax[kLpSlots][kLpThreads];
  unsigned long long pool[kLpPool];                             // candidates
  uint32_t count;
  unsigned long long list[kLpWarps][32];
  uint32_t tmax[kLpWarps][32];
  unsigned long long peer[kLpMaxCluster][32];                  // the cluster's lists (first CTA)
  LpStat stat[kLpWarps];
  LpStat peer_stat[kLpMaxCluster];
};
struct LpSharedNoTop {
  LpStat stat[kLpWarps];
  LpStat peer_stat[kLpMaxCluster];
};

// Butterfly over groups of W lanes.
template <int W>
__device__ __forceinline__ LpStat lp_warp_merge(LpStat st) {
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) {
    LpStat b;
    b.m = __shfl_xor_sync(0xffffffffu, st.m, o);
    b.s = __shfl_xor_sync(0xffffffffu, st.s, o);
    b.t = __shfl_xor_sync(0xffffffffu, st.t, o);
    st = lp_merge(st, b);
  }
  return st;
}

// The CTA's best 32 from one descending list per warp: in warp 0's `mine` and
// in lists[0], after a barrier of the CTA.
template <typename K>
__device__ __forceinline__ void lp_tree(K (*lists)[32], K& mine, int warp, int lane) {
  lists[warp][lane] = mine;
  __syncthreads();
#pragma unroll
  for (int w = kLpWarps / 2; w > 0; w >>= 1) {
    if (warp < w) {
      mine = lp_merge32(mine, lists[warp + w][lane], lane);
      lists[warp][lane] = mine;
    }
    __syncthreads();
  }
}

// CTAs per SM: 4 for f32 (512 rows in one wave: 61 us, with 3 and more
// registers 84); 16-bit steps hold twice the elements and want the registers
// (64 rows: 14.2 us, with 4 CTAs and spills 17.5).
template <typename T, bool TOP>
__global__ void __launch_bounds__(kLpThreads, sizeof(T) == 4 ? 4 : 3) logprobs_kernel(const LpArgs a) {
  constexpr int EPV = 16 / (int)sizeof(T);
  constexpr int E = kLpVec * EPV;
  __shared__ std::conditional_t<TOP, LpShared, LpSharedNoTop> sh;
  cg::cluster_group cl = cg::this_cluster();
  const uint32_t C = cl.num_blocks(), rank = cl.block_rank();
  const uint32_t row = blockIdx.x / C;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T* xr = static_cast<const T*>(a.x) + (int64_t)row * a.stride;
  // 16-byte granules that the row touches; element i of granule g is the
  // row's element g EPV + i - skew
  const uint32_t skew = (uint32_t)(reinterpret_cast<uintptr_t>(xr) & 15) / (uint32_t)sizeof(T);
  const uint4* g0 = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(xr) & ~uintptr_t(15));
  const uint32_t ng = (uint32_t)(((uint64_t)a.n + skew + EPV - 1) / EPV);
  const uint32_t gb = (uint32_t)((uint64_t)ng * rank / C), ge = (uint32_t)((uint64_t)ng * (rank + 1) / C);

  // one granule; elements outside the row read as -infinity (a granule that
  // is partly outside is read element by element)
  auto load = [&](uint32_t g) -> uint4 {
    constexpr uint32_t neg = std::is_same_v<T, float> ? 0xFF800000u : std::is_same_v<T, __half> ? 0xFC00FC00u : 0xFF80FF80u;
    if (g >= ge) return make_uint4(neg, neg, neg, neg);
    const int64_t e0 = (int64_t)g * EPV - skew;
    if (e0 >= 0 && e0 + EPV <= (int64_t)a.n) return __ldg(g0 + g);
    uint32_t w[4] = {neg, neg, neg, neg};
#pragma unroll
    for (int i = 0; i < EPV; ++i)
      if (e0 + i >= 0 && e0 + i < (int64_t)a.n) {
        if constexpr (sizeof(T) == 4) {
          w[i] = reinterpret_cast<const uint32_t*>(xr)[e0 + i];
        } else {
          const uint32_t h = reinterpret_cast<const uint16_t*>(xr)[e0 + i];
          w[i / 2] = (i & 1) ? (w[i / 2] & 0xFFFFu) | (h << 16) : (w[i / 2] & 0xFFFF0000u) | h;
        }
      }
    return make_uint4(w[0], w[1], w[2], w[3]);
  };

  LpStat st{-INFINITY, 0.f, 0.f};
  constexpr uint32_t STEP = kLpThreads * kLpVec;
  uint4 nxt[kLpVec];
#pragma unroll
  for (int u = 0; u < kLpVec; ++u) nxt[u] = load(gb + u * kLpThreads + threadIdx.x);
  const uint32_t steps = (ge - gb + STEP - 1) / STEP;
  int shift = 0;                     // 2^shift steps share a slot of smax
  while ((steps + (1u << shift) - 1) >> shift > (uint32_t)kLpSlots) ++shift;
  float slot_max = -INFINITY;
  uint32_t step = 0;
  for (uint32_t g = gb; g < ge; g += STEP, ++step) {
    float x[E];
#pragma unroll
    for (int u = 0; u < kLpVec; ++u) lp_unpack<T>(nxt[u], x + u * EPV);
    if (g + STEP < ge) {
#pragma unroll
      for (int u = 0; u < kLpVec; ++u) nxt[u] = load(g + STEP + u * kLpThreads + threadIdx.x);
    }
    float cm = x[0];
#pragma unroll
    for (int i = 1; i < E; ++i) cm = fmaxf(cm, x[i]);
    if (cm > st.m) {
      const float d = fmaxf(st.m - cm, kLpLow), f = expf(d);
      st.t = (st.t + st.s * d) * f;
      st.s *= f;
      st.m = cm;
    }
    const float mm = st.m == -INFINITY ? 0.f : st.m;
    float s0 = 0.f, t0 = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const float d = max_nan(x[i] - mm, kLpLow);
      const float e = ex2(d * kLog2e);
      s0 += e;
      t0 = fmaf(e, d, t0);
    }
    st.s += s0;
    st.t += t0;
    if constexpr (TOP) {
      slot_max = (step & ((1u << shift) - 1)) == 0 ? cm : fmaxf(slot_max, cm);
      sh.smax[step >> shift][threadIdx.x] = slot_max;
    }
  }

  const float thread_max = st.m;
  // warp -> CTA
  st = lp_warp_merge<32>(st);
  if (lane == 0) sh.stat[warp] = st;
  unsigned long long best = 0;          // lane i: the i-th best so far
  if constexpr (TOP) {
    // The k-th largest of 64 maxima, each over 4 threads (every warp finds it
    // for itself: two sorts side by side and a merge).
    sh.tmax[warp][lane] = float_key(thread_max + 0.f);
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    const uint32_t g0 = lp_sort32(max(max(sh.tmax[0][lane], sh.tmax[1][lane]), max(sh.tmax[2][lane], sh.tmax[3][lane])), lane);
    const uint32_t g1 = lp_sort32(max(max(sh.tmax[4][lane], sh.tmax[5][lane]), max(sh.tmax[6][lane], sh.tmax[7][lane])), lane);
    const uint32_t tk = __shfl_sync(0xffffffffu, lp_merge32(g0, g1, lane), (int)a.top_k - 1);
    const float floor_ = lp_value((unsigned long long)tk << 32);

    // The steps of this warp's threads that reach it are read again, four
    // loads at a time; lane: vector lane / EPV of the step, element lane % EPV.
    // f(value, index): one call per lane and element, the warp together.
    const uint32_t slots = (steps + (1u << shift) - 1) >> shift;
    auto again = [&](auto f) {
      uint32_t mine = 0;                 // slots of this thread
      for (uint32_t sl = 0; sl < slots; ++sl) {
        const float v = sh.smax[sl][threadIdx.x];
        if (v >= floor_ && v > -INFINITY) mine |= 1u << sl;
      }
      uint32_t src = 0, sl = 0, sub = 0;   // thread (lane), slot and step of the next load
      uint32_t owners = __ballot_sync(0xffffffffu, mine != 0);
      while (owners || sub) {
        float xv[4];
        uint32_t idx[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          xv[q] = -INFINITY;
          idx[q] = 0;
          if (!(owners || sub)) continue;
          if (sub == 0) {
            src = (uint32_t)__ffs(owners) - 1;
            sl = (uint32_t)__ffs(__shfl_sync(0xffffffffu, mine, (int)src)) - 1;
            if ((uint32_t)lane == src) mine &= mine - 1;
            owners = __ballot_sync(0xffffffffu, mine != 0);
          }
          const uint32_t gr = gb + ((sl << shift) + sub) * STEP + (lane / EPV) * kLpThreads + warp * 32 + src;
          const int64_t e = (int64_t)gr * EPV + lane % EPV - skew;
          if (lane < E && gr < ge && e >= 0 && e < (int64_t)a.n) xv[q] = lp_load1(xr + e);
          idx[q] = (uint32_t)e;
          sub = (sub + 1) & ((1u << shift) - 1);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) f(xv[q], idx[q]);
      }
    };
    // They are few (about k for any but contrived rows): one pool for the CTA.
    again([&](float v, uint32_t i) {
      if (v >= floor_ && v > -INFINITY) {
        const uint32_t at = atomicAdd(&sh.count, 1u);
        if (at < (uint32_t)kLpPool) sh.pool[at] = lp_key(v, i);
      }
    });
    __syncthreads();
    const uint32_t count = sh.count;
    if (count <= (uint32_t)kLpPool) {
      if (warp == 0) {
        best = lp_sort32((uint32_t)lane < count ? sh.pool[lane] : 0ull, lane);
        for (uint32_t at = 32; at < count; at += 32)
          best = lp_merge32(best, lp_sort32(at + lane < count ? sh.pool[at + lane] : 0ull, lane), lane);
      }
    } else {
      // many equal or nearly equal largest logits: a list per warp, 32
      // candidates at a time, those that beat its k-th
      __syncthreads();                   // the pool becomes the warps' buffers
      unsigned long long* buf = sh.pool + warp * 64;
      uint32_t cnt = 0;
      unsigned long long kth = 0;
      auto flush = [&]() {
        __syncwarp();
        const unsigned long long k = (uint32_t)lane < cnt ? buf[lane] : 0ull;
        const unsigned long long rest = (uint32_t)lane + 32 < cnt ? buf[lane + 32] : 0ull;
        __syncwarp();
        buf[lane] = rest;
        cnt = cnt > 32 ? cnt - 32 : 0;
        best = lp_merge32(best, lp_sort32(k, lane), lane);
        kth = __shfl_sync(0xffffffffu, best, (int)a.top_k - 1);
        __syncwarp();
      };
      again([&](float v, uint32_t i) {
        const unsigned long long key = v >= floor_ && v > -INFINITY ? lp_key(v, i) : 0ull;
        const bool take = key > kth;
        const uint32_t b = __ballot_sync(0xffffffffu, take);
        if (take) buf[cnt + __popc(b & ((1u << lane) - 1u))] = key;
        cnt += __popc(b);
        if (cnt >= 32) flush();
      });
      if (cnt) flush();
      lp_tree(sh.list, best, warp, lane);
    }
  } else {
    __syncthreads();
  }
  // CTA -> first CTA of the cluster (whose shared memory exists once every
  // CTA of the cluster has started)
  if (C > 1) {
    cl.sync();
    if (warp == 0) {
      st = lp_warp_merge<kLpWarps>(sh.stat[lane % kLpWarps]);
      auto* dst = cl.map_shared_rank(&sh, 0);
      if (lane == 0) dst->peer_stat[rank] = st;
      if constexpr (TOP) dst->peer[rank][lane] = best;
    }
    cl.sync();
    if (rank != 0) return;
    if constexpr (TOP) {
      best = 0;
      for (uint32_t r = warp; r < C; r += kLpWarps) best = lp_merge32(best, sh.peer[r][lane], lane);
      lp_tree(sh.list, best, warp, lane);
    }
    if (warp != 0) return;
    st = (uint32_t)lane % kLpMaxCluster < C ? sh.peer_stat[lane % kLpMaxCluster] : LpStat{-INFINITY, 0.f, 0.f};
    st = lp_warp_merge<(int)kLpMaxCluster>(st);
  } else {
    if (warp != 0) return;
    st = lp_warp_merge<kLpWarps>(sh.stat[lane % kLpWarps]);
  }
  const float ls = logf(st.s);
  // a row with nothing allowed: every log probability -infinity, entropy 0
  const bool empty = st.m == -INFINITY && st.s == 0.f;
  if (lane == 0) {
    if (a.entropy) a.entropy[row] = empty ? 0.f : ls - st.t / st.s;
    if (a.lse) a.lse[row] = empty ? -INFINITY : st.m + ls;
  }
  for (uint32_t j = lane; j < a.num_tokens; j += 32) {
    const int t = a.tokens[(size_t)row * a.num_tokens + j];
    float v = 0.f;
    if (t >= (int64_t)a.n) {
      atomicOr(a.err, ERR_BAD_TOKEN);
      v = NAN;
    } else if (t >= 0) {
      v = empty ? -INFINITY : (lp_load1(xr + t) - st.m) - ls;
    }
    a.logprob[(size_t)row * a.num_tokens + j] = v;
  }
  if constexpr (TOP) {
    if ((uint32_t)lane < a.top_k) {
      const float v = lp_value(best);
      const bool none = best == 0 || v == -INFINITY;
      a.top_ids[(size_t)row * a.top_k + lane] = none ? -1 : (int)argmax_index(best);
      a.top_lp[(size_t)row * a.top_k + lane] = none ? (st.s == st.s ? -INFINITY : NAN) : (v - st.m) - ls;
    }
  }
}

template <typename T, bool TOP>
cudaError_t logprobs_go(const LpArgs& a, int sms, cudaStream_t st) {
  const auto fn = &logprobs_kernel<T, TOP>;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kLpThreads);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  // The largest cluster: 16 CTAs where the device takes them, else the 8 that every one does.
  static PerDevice largest;
  const uint32_t most = (uint32_t)largest.get([&] {
    int n = 0;
    at[0].val.clusterDim.x = kLpMaxCluster;
    cfg.gridDim = dim3(kLpMaxCluster);
    if (cudaFuncSetAttribute((const void*)fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess &&
        cudaOccupancyMaxActiveClusters(&n, fn, &cfg) == cudaSuccess && n > 0)
      return (int)kLpMaxCluster;
    cudaGetLastError();
    return 8;
  });
  // CTAs per row: as many as keep the row's CTAs within two per SM, each with
  // a step of work or more (a CTA's sorts and merges cost it 3 - 4 us: 64 rows
  // of 151669 bf16 take 14.5 us with 4, 17.8 with 8, 16.9 with 2; 512 rows of
  // 151936 f32 60.9 us with 1, 69.8 with 2; one row 8.3 us with 16, 11.2 with 4)
  const uint64_t bytes = (uint64_t)a.n * sizeof(T);
  uint32_t C = 1;
  while (C < most && (uint64_t)a.rows * 2 * C <= (uint64_t)sms * 2 && bytes / (2 * C) >= kLpThreads * kLpVec * 16) C *= 2;
  if ((uint64_t)a.rows * C > 0x7FFFFFFFull) return cudaErrorInvalidValue;
  cfg.gridDim = dim3(a.rows * C);
  at[0].val.clusterDim.x = C;
  return cudaLaunchKernelEx(&cfg, fn, a);
}

template <typename T>
cudaError_t logprobs_t(const LpArgs& a, int sms, cudaStream_t st) {
  return a.top_k ? logprobs_go<T, true>(a, sms, st) : logprobs_go<T, false>(a, sms, st);
}

}  // namespace
}  // namespace nnz

extern "C" int nnz_token_logprobs(const nnz_logprobs_args* p, void* stream) {
  using namespace nnz;
  if (!p) return refuse(NNZ_EINVAL, "nnz_token_logprobs: null argument");
  if (p->rows == 0) return NNZ_OK;
  if (p->dtype != NNZ_DT_F32 && p->dtype != NNZ_DT_F16 && p->dtype != NNZ_DT_BF16)
    return refuse(NNZ_EINVAL, "nnz_token_logprobs: dtype must be f32, f16 or bf16");
  const uintptr_t esz = p->dtype == NNZ_DT_F32 ? 4 : 2;
  if (!p->logits || (reinterpret_cast<uintptr_t>(p->logits) % esz) || p->n == 0 || p->n > 0x7FFFFFF0u || p->rows > 0x7FFFFFFu ||
      p->stride < (int64_t)p->n)
    return refuse(NNZ_EINVAL, "nnz_token_logprobs: logits, rows, n or stride");
  if (p->top_k > 32 || (p->top_k && (!p->top_ids || !p->top_logprobs)))
    return refuse(NNZ_EINVAL, "nnz_token_logprobs: top_k must be 0 .. 32, with top_ids and top_logprobs");
  if (p->num_tokens && (!p->tokens || !p->logprob)) return refuse(NNZ_EINVAL, "nnz_token_logprobs: tokens need logprob");
  LpArgs a{};
  int sms = 0;
  if (const int rc = op_device(&a.err, &sms)) return rc;
  a.x = p->logits;
  a.rows = p->rows;
  a.n = p->n;
  a.stride = p->stride;
  a.tokens = p->tokens;
  a.num_tokens = p->num_tokens;
  a.top_k = p->top_k;
  a.logprob = p->logprob;
  a.entropy = p->entropy;
  a.lse = p->logsumexp;
  a.top_ids = p->top_ids;
  a.top_lp = p->top_logprobs;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = p->dtype == NNZ_DT_F32 ? logprobs_t<float>(a, sms, st)
                      : p->dtype == NNZ_DT_F16 ? logprobs_t<__half>(a, sms, st) : logprobs_t<__nv_bfloat16>(a, sms, st);
  return cuda_rc(e, "nnz_token_logprobs");
}
