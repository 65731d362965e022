// Attention of many query rows over paged K/V on tcgen05: prompt chunks, alone
// or mixed with single tokens.
//
// A task is 2 x 128 rows, (token, head) pairs of one sequence and kv head
// with the G heads fastest, so the heads of a group share every K/V tile; its
// units are tiles of 128 keys, and the units of all tasks are cut into equal
// runs, one per CTA and SM (paged_sched.cuh).  Per unit, for each of the two
// row tiles:
//   S = Q K^T           tcgen05.mma, operands in shared memory, f32 in TMEM
//   P = 2^(S c - m)     two threads per row: online softmax out of TMEM, P in
//                       the pool's type over the S it came from
//   O += P V            tcgen05.mma, P from TMEM, V as stored (MN-major B)
// so while one row tile's softmax runs, the tensor cores work for the other.
// m need not be the row's maximum: any m gives the same quotient as long as no
// P overflows and the largest does not fall so low that the others are lost
// below the 16-bit type's range.  A unit's P is computed with the m that the row
// has, in one pass over S without looking for a maximum, and only if the sum of
// 64 P turns out to be 2^15 or more (or, among the first keys that a row sees,
// less than kLeast) does the row take a new m, from its maximum, rescale O and
// compute the unit again, which after the first units is rare.
// f16: m starts at -4 and is set 4 below the maximum, so P has 4 bits more
// towards zero, and 64 P that sum to 64 have one of 1 or more: what P loses below
// 2^-14 is 2^-25 of the row's largest a key.  bf16 has f32's range: m starts at 0,
// is set to the maximum, and a sum of 1/4 will do.  (f16 with m from 0 and a sum
// of 64 took 37.4 us for 512 tokens, whose units were often computed twice;
// from -4 36.5.)
// Sums are f32, and of the P before they are rounded.  P enters the second
// product in the pool's type because the tensor cores multiply 16-bit operands
// at twice the rate of wider ones: an error of half a unit in its last place in
// every weight, as much again as the result's own rounding at the most.
// (The tensor cores add a product to O with about 2^-25 of O's size: tens of
// thousands of keys that weigh less than that each are lost, in any type.)
//
// Roles: warps 0-7 and 8-15 softmax and epilogue of row tiles 0 and 1 (TMEM lane
// = row; warps 0-3 of a tile have keys 0-63 of a unit and the lower half of the
// output's dims, 4-7 the others; together they clean the V tiles at the
// diagonal and at the end), warp 16 finds the CTA's run of units, hands its
// parts to the others and loads them (Q, then K and V tiles into one ring,
// boxes of one page each), warp 17 MMA issue.  Boxes of absent
// pages and past the length are loaded from beyond the pool's last page: the
// copy engine fills them with zeros, so no stale byte meets the product.
//
// Measured (16 / 8 heads of 128): 4096 tokens behind 4096 keys 214 us, 960
// TFLOP/s of the visible pairs' products; 512 behind 4096 36.7 us.  Over the 4096
// tokens the tensor pipe is busy 56 % of the time and the special-function units
// 57 %; neither is the limit, the order between them is.  A unit
// takes a CTA about 3900 cycles, its four products 2100 to 2800 of them: S, the
// softmax, P V and the next S of a row tile follow one another, TMEM is full
// with one S and one O of each, and the special-function units alone need 2048
// cycles for a unit's exponentials.  (Steps of 64 keys with two S of each row
// tile took 256 us: products of 64 columns are bound by the queries' way from
// shared memory.)  Of the 512 tokens' time about 7 us are the way to the first
// S (lengths, cut, page numbers, first tiles) and 6 us the merge of the parts.
//
// TMEM: S of the two row tiles at columns 0 and 128, O at 256 and 384; P of keys
// 0-63 and 64-127 over the first 32 columns of their halves of S.
#include <cuda_runtime.h>
#include <math.h>

#include <atomic>
#include <type_traits>

#include "paged_sched.cuh"
#include "paged_tma.cuh"
#include "umma.cuh"

namespace nnz {

namespace {

constexpr int kUmKeys = 128;
// 96 registers a thread.  (A fifth whole warpgroup that gave its registers to
// the softmax warps, 104 / 64, took 36.4 instead of 34.9 us for 512 tokens: the
// warps that load and issue then spill.)
constexpr int kUmThreads = 576;
constexpr uint32_t kUmTries = 1u << 18;          // polls of a wait: every wait is for this CTA's own warps and copies
constexpr int kWTma = 16, kWMma = 17;             // warps
constexpr uint32_t kHalfB = 128 * 128;           // 128 rows x 64 dims, swizzled
constexpr int kSegs = 4;                          // segments in flight
constexpr uint32_t kPartCost = 3;                 // what a part costs besides its units, in units (queries, epilogue, merge)
constexpr int kPres = 8;                          // units whose page masks are kept
// sum of 64 P: below kMost (no P overflows), at first kLeast at least
constexpr float kMost = 32768.f;
template <typename T>
constexpr float kLeast = T16<T>::kBf16 ? 0.25f : 64.f;
template <typename T>
constexpr float kLift = T16<T>::kBf16 ? 0.f : 4.f;         // m is this much below the maximum

template <int HD>
struct UmShape {
  static constexpr uint32_t kTileB = (HD / 64) * kHalfB;      // Q, K or V tile of 128 rows
  static constexpr int kStages = HD == 128 ? 5 : 8;
  static constexpr uint32_t OFF_KV = 2 * kTileB;
  static constexpr uint32_t OFF_BAR = OFF_KV + kStages * kTileB;
  static constexpr int kBars = 2 * kStages + 9 + 3 * kPres + 2 * kSegs;
  static constexpr uint32_t OFF_MISC = OFF_BAR + kBars * 8;
  static constexpr uint32_t OFF_SEG = OFF_MISC + 80, OFF_XT = OFF_SEG + kSegs * 80;
  static constexpr uint32_t kSmem = OFF_XT + 1024 + 1024;
};

struct UmArgs {
  CUtensorMap tmQ, tmK, tmV;
  PagedAttnArgs a;
  PartWs ws;
  uint32_t workers;
  uint32_t box;       // keys per copy: 8 .. 128
  uint32_t pt;        // tokens per row tile: 128 / G
  float sl2;          // scale * log2(e)
};

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* tm, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(tm)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void mbar_arrive1(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// D(tmem) (+)= A(tmem) B(smem), kind::f16.
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc));
}

// 32 columns of this thread's TMEM lane; complete only after tm_wait_ld.
__device__ __forceinline__ void tm_ld32(uint32_t taddr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]),
        "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]),
        "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tm_ld16(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tm_wait_ld(uint32_t (&v)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]),
                 "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])
               :
               : "memory");
}
// Waits for this thread's TMEM loads; v is tied to the wait so that no use of
// it can be scheduled before.
__device__ __forceinline__ void tm_wait_ld(uint32_t (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]),
                 "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])
               :
               : "memory");
  asm volatile("" : "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]),
                    "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31]));
}
// Two f32 at a time (one instruction each).
__device__ __forceinline__ uint64_t pair2(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float2 split2(uint64_t a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a));
  return r;
}

// Sets the scores of 64 keys of a row that it does not see to -infinity, in
// TMEM: it sees the first `end`, on pages whose bit is set (one bit per 2^sh
// keys).  (Rolled: this runs a few times per task, and instructions have to
// be fetched.)
__device__ __forceinline__ void um_mask(uint32_t tS, int end, uint32_t bits, uint32_t sh) {
#pragma unroll 1
  for (int c = 0; c < 2; ++c) {
    uint32_t see = end >= 32 * c + 32 ? 0xFFFFFFFFu : end <= 32 * c ? 0u : (1u << (end - 32 * c)) - 1u;
    const uint32_t pg = bits >> ((32 * c) >> sh);          // first page bit of this quarter
    if (sh >= 5) {
      if (!(pg & 1u)) see = 0;
    } else {
      for (int e = 0; e < 32; e += 1 << sh)
        if (!((pg >> (e >> sh)) & 1u)) see &= ~(((1u << (1 << sh)) - 1u) << e);
    }
    if (__all_sync(0xffffffffu, see == 0xFFFFFFFFu)) continue;
    uint32_t v[32];
    tm_ld32(tS + 32 * c, v);
    tm_wait_ld(v);
#pragma unroll
    for (int e = 0; e < 32; ++e) v[e] = (see >> e) & 1u ? v[e] : 0xFF800000u;
    tmem_st32(tS + 32 * c, v);
  }
}

// The largest of 64 scores of a row.
__device__ __forceinline__ float um_top(uint32_t tS) {
  float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll 1
  for (int c = 0; c < 2; ++c) {
    uint32_t v[32];
    tm_ld32(tS + 32 * c, v);
    tm_wait_ld(v);
#pragma unroll
    for (int e = 0; e < 32; ++e) mx[e & 1] = fmaxf(mx[e & 1], __uint_as_float(v[e]));
  }
  return fmaxf(mx[0], mx[1]);
}

// P = 2^(S sl2 - ms) of 64 keys of a row as 32 words of the pool's type; their
// f32 sum.  The next 16 of S are on their way while some are worked on.
template <typename T>
__device__ __forceinline__ float um_pass(uint32_t tS, float sl2, float ms, uint32_t (&w)[32]) {
  const uint64_t k2 = pair2(sl2, sl2), m2 = pair2(-ms, -ms);
  uint64_t acc[2] = {0ull, 0ull};
  uint32_t v[2][16];
  tm_ld16(tS, v[0]);
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    tm_wait_ld(v[c & 1]);
    if (c < 3) tm_ld16(tS + 16 * (c + 1), v[(c + 1) & 1]);
#pragma unroll
    for (int e = 0; e < 16; e += 2) {
      const float2 y = split2(fma2(pair2(__uint_as_float(v[c & 1][e]), __uint_as_float(v[c & 1][e + 1])), k2, m2));
      // (all on the special-function units: a polynomial for every fourth on
      // the FMA pipe made it 235 instead of 229 us for 4096 tokens)
      const float2 q = make_float2(ex2(y.x), ex2(y.y));
      acc[(e >> 1) & 1] = add2(acc[(e >> 1) & 1], pair2(q.x, q.y));
      w[8 * c + e / 2] = T16<T>::pack(q.x, q.y);
    }
    // the words stay before the wait for the next ones
    uint32_t* q = w + 8 * c;
    asm volatile("" : "+r"(q[0]), "+r"(q[1]), "+r"(q[2]), "+r"(q[3]), "+r"(q[4]), "+r"(q[5]), "+r"(q[6]), "+r"(q[7]));
  }
  const float2 t = split2(add2(acc[0], acc[1]));
  return t.x + t.y;
}

// The two warps that share 32 rows: whether any of their 64 threads says so.
__device__ __forceinline__ bool pair_any(int bar, bool p) {
  uint32_t r;
  asm volatile(
      "{\n .reg .pred a, b;\n setp.ne.u32 a, %2, 0;\n bar.red.or.pred b, %1, 64, a;\n selp.u32 %0, 1, 0, b;\n}\n"
      : "=r"(r)
      : "r"(bar), "r"((uint32_t)p)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ void pair_sync(int bar) { asm volatile("bar.sync %0, 64;" ::"r"(bar) : "memory"); }
// The value of the row's thread of half `from`.
__device__ __forceinline__ float pair_tell(int bar, volatile uint32_t* at, int half, int from, float v) {
  if (half == from) *at = __float_as_uint(v);
  pair_sync(bar);
  const float r = __uint_as_float(*at);
  pair_sync(bar);
  return r;
}

template <bool BF16>
__host__ __device__ constexpr uint32_t um_idesc(int M, int N) {
  return idesc_f16(M, N) | (BF16 ? (1u << 7) | (1u << 10) : 0u);
}

// 16-bit words with a non-finite element (exponent all ones).
template <bool BF16>
__device__ __forceinline__ uint32_t bad_mask(uint32_t w) {
  constexpr uint32_t e = BF16 ? 0x7F80u : 0x7C00u;
  return ((w & e) == e ? 0xFFFFu : 0u) | (((w >> 16) & e) == e ? 0xFFFF0000u : 0u);
}

// The part of one task in a CTA's run, as warp 16 hands it to the others.
struct Segment {
  uint32_t take;       // units (0: the run is over)
  uint32_t unit;       // first unit within the task
  uint32_t n[2];       // units that each row tile looks at (from the first)
  uint32_t parts;      // 0: the whole task; else the parts it is split into
  uint32_t gaps;       // a page of its keys is absent
  uint32_t s, kvh;
  int row0;            // q / out row of the task's first token
  int rows;            // tokens of the task
  uint32_t marks[8];   // keys with a non-finite V, among the task's last 256
  int d, e;            // token i of the task sees keys [0, clamp(d + i, 0, e))

  __device__ __forceinline__ int seen(int i) const { return max(0, min(d + i, e)); }
};
// Adds the non-finite V elements d0 .. d0 + 31 of the marked keys that the
// row sees (a NaN or an infinity times a positive probability is itself).
template <bool BF16>
__device__ __forceinline__ void add_nonfinite(const PagedAttnArgs& a, const Segment& g, const volatile uint32_t* marks, int limit, int d0, float (&o)[32]) {
  const int base = max(0, g.seen(g.rows - 1) - 256);
  for (int w = 0; w < 8; ++w) {
    uint32_t bits = marks[w];
    while (bits) {
      const int key = base + 32 * w + __ffs(bits) - 1;
      bits &= bits - 1;
      if (key >= limit) continue;
      const uint32_t pi = (uint32_t)key / a.kv.page_size;
      const int pg = __ldg(a.page_table + (size_t)g.s * a.table_stride + pi);
      if ((uint32_t)pg >= a.kv.num_pages) continue;      // (a mark of a tile that never landed, after a wait that gave up)
      const uint16_t* vp = a.kv.v + (int64_t)pg * a.kv.page_stride + (int64_t)g.kvh * a.kv.head_stride +
                           (int64_t)((uint32_t)key - pi * a.kv.page_size) * a.kv.token_stride + d0;
#pragma unroll
      for (int d = 0; d < 32; d += 2) {
        const uint32_t e = *reinterpret_cast<const uint32_t*>(vp + d);
        const uint32_t b = bad_mask<BF16>(e);
        const float2 f = T16<std::conditional_t<BF16, __nv_bfloat16, __half>>::to_f2(e & b);
        o[d] += f.x;
        o[d + 1] += f.y;
      }
    }
  }
}

template <typename T, int HD>
__global__ void __launch_bounds__(kUmThreads, 1) paged_umma_kernel(const __grid_constant__ UmArgs t) {
  using S = UmShape<HD>;
  constexpr bool BF = T16<T>::kBf16;
  constexpr int NH = HD / 64;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const PagedAttnArgs& a = t.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint64_t* kv_full = reinterpret_cast<uint64_t*>(sm + S::OFF_BAR);
  uint64_t* kv_empty = kv_full + S::kStages;
  uint64_t* q_full = kv_empty + S::kStages;
  uint64_t* q_empty = q_full + 1;
  uint64_t* drained = q_empty + 1;       // every product is complete (after a wait that gave up)
  uint64_t* s_full = drained + 1;        // [2] S of a row tile complete
  uint64_t* p_full = s_full + 2;         // [2] P written, O rescaled (8 warps)
  uint64_t* pv_done = p_full + 2;        // [2] P V complete
  uint64_t* v_ready = pv_done + 2;       // [kPres] a unit's V tile has been cleaned (units that need it; 16 warps)
  uint64_t* v_go = v_ready + kPres;      // [kPres] such a tile is there (it stays until it has been cleaned)
  uint64_t* pres_full = v_go + kPres;    // [kPres] page mask of a unit written
  uint64_t* seg_full = pres_full + kPres;   // [kSegs]
  uint64_t* seg_empty = seg_full + kSegs;   // [kSegs] the 17 other warps are done with it
  uint32_t* tslot = reinterpret_cast<uint32_t*>(sm + S::OFF_MISC);
  volatile uint32_t* pres = tslot + 1;   // [kPres] one bit per box of the unit: page present
  Segment* segs = reinterpret_cast<Segment*>(sm + S::OFF_SEG);
  static_assert(sizeof(Segment) <= 80 && S::kSmem <= 232448);
  uint32_t* xt = reinterpret_cast<uint32_t*>(sm + S::OFF_XT);     // [2][128] what the two threads of a row tell each other (before: the cut's pairs)
  const uint32_t G = a.n_q / a.kv.n_kv;
  const int PT = (int)t.pt, QT = 2 * PT;
  // every barrier by its own thread; arrivals: a warp each for P (8), a clean V
  // tile (16) and a part's end (17), else 1
  static_assert(S::kBars <= kUmThreads);
  if (threadIdx.x < 8) tslot[1 + kPres + threadIdx.x] = 0;
  if (threadIdx.x < (uint32_t)S::kBars) {
    uint64_t* b = kv_full + threadIdx.x;
    mbar_init(b, b == p_full || b == p_full + 1 ? 8 : b >= v_ready && b < v_go ? 16 : b >= seg_empty ? 17 : 1);
    fence_barrier_init();
  }
  if (warp == kWTma && lane < 3) {
    const CUtensorMap* tm = lane == 0 ? &t.tmQ : lane == 1 ? &t.tmK : &t.tmV;
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(tm)) : "memory");
  }
  if (warp == kWMma) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tslot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tslot;
  pdl_launch();       // the merge kernel may be set up (it waits for this one's end)
  // Bounded waits: one that gives up leaves no tries to the later ones, and the
  // error is reported at the end (nothing but the poll stands in the loop).
  // Who gave up stops at its next part, all lanes of a warp and both warps of
  // a pair together, or those left would wait at barriers that have no bound; a
  // part that is not finished with is not replaced, no tile is given back that
  // may not have landed, and copies and products under way are waited for
  // (`landed`) before the CTA ends.
  uint32_t tries = kUmTries;
  auto gave_up = [&] { return __any_sync(0xffffffffu, tries == 0) != 0; };
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    for (uint32_t n = 0; !mbar_try_wait(bar, parity & 1u);)
      if (++n > tries) {
        tries = 0;
        break;
      }
  };

  auto landed = [&](uint64_t* bar, uint32_t parity) {
    for (uint32_t n = 0; n < kUmTries && !mbar_try_wait(bar, parity & 1u);) ++n;
  };

  // part k of the run; warp 17, and 0-15 likewise, take them in order from warp 16
  // (fields are read into registers one by one: a copy indexed by the row tile
  // would live in local memory, which with this much shared memory means L2)
  auto segment = [&](uint32_t k) -> const Segment* {
    wait(seg_full + k % kSegs, k / kSegs);
    const Segment* g = segs + k % kSegs;
    return !gave_up() && g->take != 0 ? g : nullptr;
  };
  auto segment_done = [&](uint32_t k) {
    __syncwarp();
    if (lane == 0) mbar_arrive1(seg_empty + k % kSegs);
  };

  if (warp >= 16) {
  if (warp == kWTma) {
    // ---------------- the run, and its TMA ----------------
    Cursor c;
    PartRun run{0, 0, 0};
    uint64_t u = 0, u1 = 0;
    uint32_t per = 1;
    bool even = true, more = false;
    const uint32_t P = t.workers;
    // One part per CTA where that costs no more than kPartCost units over the
    // even cut (us, against the even cut: 512 tokens of 4608 keys 38.4 / 43.0,
    // 1024 of 2048 35.2 / 38.7, 31 single tokens and a chunk of 449 34.6 / 43.2;
    // 128 of 1024 22.6 / 22.5).
    even = !warp_parts<5>(a, QT, kUmKeys, lane, P, [](uint32_t) { return kPartCost; }, blockIdx.x == 0, blockIdx.x, xt, c, run);
    more = run.parts != 0;
    if (even) {
      uint64_t mine = 0;
      const uint64_t total = warp_total(a, QT, kUmKeys, lane, blockIdx.x == 0, mine);
      per = max(1u, (uint32_t)div_up(total, P));
      u = (uint64_t)blockIdx.x * per;
      u1 = min(u + per, total);
      more = u < u1;
      if (more) warp_find(a, QT, kUmKeys, lane, u, mine, c);
    }
    const uint32_t nb = kUmKeys / t.box;
    const uint32_t bi = (uint32_t)lane % nb;      // this lane's box of a unit
    uint32_t stage_use = 0, unit_no = 0, q_use = 0;
    for (uint32_t seg = 0;; ++seg) {
      // ---- the next part: to the other warps ----
      Segment o{};
      if (more) {
        o.take = even ? (uint32_t)min((uint64_t)(c.units - c.unit), u1 - u) : run.end - c.unit;
        o.unit = c.unit;
        o.s = c.s;
        o.kvh = c.kvh;
        const int tok0 = c.qt * QT;
        o.row0 = (int)c.q.row0 + tok0;
        o.rows = min(QT, c.q.rows - tok0);
        o.e = (int)min(max(c.q.len, (int64_t)0), c.q.cap);
        o.d = (int)max(c.q.len - c.q.n + 1 + tok0, (int64_t)-(1 << 30));
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (i * PT < o.rows) {
            const uint32_t un = max(1u, ((uint32_t)o.seen(min((i + 1) * PT, o.rows) - 1) + kUmKeys - 1) / kUmKeys);
            o.n[i] = un > c.unit ? min(un - c.unit, o.take) : 0;
          }
        if (!even) {
          o.parts = run.parts > 1 ? run.parts : 0;
        } else if (o.take != c.units) {
          const uint64_t t0 = u - c.unit;
          o.parts = (uint32_t)((t0 + c.units - 1) / per - t0 / per + 1);
        }
      }
      auto publish = [&] {
        if (o.take) {     // (softmax warps ask per part, not per unit: shared memory is slow to answer while MMAs read it)
          const uint32_t k0 = o.unit * kUmKeys, k1 = min((o.unit + o.take) * kUmKeys, (uint32_t)o.seen(o.rows - 1));
          const uint32_t p0 = k0 / a.kv.page_size, p1 = k1 > k0 ? (k1 - 1) / a.kv.page_size + 1 : p0;
          bool gap = false;
          for (uint32_t p = p0 + lane; p < p1; p += 32) gap |= (uint32_t)__ldg(a.page_table + (size_t)o.s * a.table_stride + p) >= a.kv.num_pages;
          o.gaps = __any_sync(0xffffffffu, gap) ? 1u : 0u;
        }
        if (seg >= kSegs) wait(seg_empty + seg % kSegs, seg / kSegs - 1);
        if (gave_up()) return;
        if (lane == 0) {
          segs[seg % kSegs] = o;
          mbar_arrive1(seg_full + seg % kSegs);
        }
      };
      // (the first part's loads go first: nobody can use it before they land)
      if (seg || !o.take) publish();
      if (gave_up() || o.take == 0) break;
      u += o.take;
      more = even && u < u1 && cursor_next_task(a, c, QT, kUmKeys);

      // ---- its loads ----
      const int last = o.seen(o.rows - 1);
      const int* pages = a.page_table + (size_t)o.s * a.table_stride;
      // page of this lane's box of unit i; -1 where there is none
      auto page_of = [&](uint32_t i, uint32_t& at) -> int {
        const uint32_t key = (o.unit + i) * kUmKeys + bi * t.box;
        at = 0;
        if (key >= (uint32_t)last) return -1;
        const uint32_t pi = key / a.kv.page_size;
        at = key - pi * a.kv.page_size;
        const int p = __ldg(pages + pi);
        if ((uint32_t)p < a.kv.num_pages) return p;
        if (p >= 0) atomicOr(a.err, ERR_BAD_PAGE);
        return -1;
      };
      uint32_t at, nat = 0;
      int pg = page_of(0, at), npg = -1;
      // the queries: at once for the first part, later once the previous part's
      // products have read theirs (its first K tile does not wait for that)
      auto queries = [&] {
        if (seg) wait(q_empty, seg - 1);
        if (gave_up()) return;
        ++q_use;
        const int tiles = PT < o.rows ? 2 : 1;
        if (lane == 0) {
          mbar_arrive_expect_tx(q_full, (uint32_t)tiles * NH * G * PT * 128);
          for (int x = 0; x < tiles; ++x)
            for (int h = 0; h < NH; ++h)
              tma_load_3d(sm + x * S::kTileB + h * kHalfB, &t.tmQ, h * 64, (int)(o.kvh * G), o.row0 + x * PT, q_full);
        }
        __syncwarp();
      };
      if (seg == 0) queries();
      bool on = true;
      for (uint32_t i = 0; on && i < o.take; ++i) {
        if (i + 1 < o.take) npg = page_of(i + 1, nat);
        const uint32_t mask = __ballot_sync(0xffffffffu, (uint32_t)lane < nb && pg >= 0);
        if (pg < 0) pg = (int)a.kv.num_pages;
        const int slot = (int)(unit_no % kPres);
        if (lane == 0) {
          pres[slot] = mask;
          mbar_arrive1(pres_full + slot);
        }
#pragma unroll 1
        for (int kv = 0; kv < 2; ++kv) {
          const uint32_t st = stage_use % S::kStages, round = stage_use / S::kStages;
          if (round) {
            wait(kv_empty + st, round - 1);
            on = !gave_up();
            if (!on) break;
          }
          if (lane == 0) mbar_arrive_expect_tx(kv_full + st, S::kTileB);
          __syncwarp();
          // one elected lane issues (a lane each takes the compiler's loop over
          // divergent operands, about 100 cycles a copy)
          uint8_t* dst = sm + S::OFF_KV + st * S::kTileB;
          const CUtensorMap* tm = kv ? &t.tmV : &t.tmK;
#pragma unroll 4
          for (uint32_t b = 0; b < nb; ++b, dst += t.box * 128) {
            const int bp = __shfl_sync(0xffffffffu, pg, (int)b), bo = (int)__shfl_sync(0xffffffffu, at, (int)b);
            if (elect_one())
#pragma unroll
              for (int h = 0; h < NH; ++h) tma_load_4d(dst + h * kHalfB, tm, h * 64, bo, (int)o.kvh, bp, kv_full + st);
          }
          __syncwarp();
          ++stage_use;
          if (kv == 0 && i == 0) {
            if (seg) queries();
            else publish();
          }
        }
        pg = npg;
        at = nat;
        ++unit_no;
      }
    }
    // (whoever gave up may not have waited for them)
#pragma unroll 1
    for (uint32_t n = stage_use > (uint32_t)S::kStages ? stage_use - S::kStages : 0; n < stage_use; ++n) landed(kv_full + n % S::kStages, n / S::kStages);
    if (q_use) landed(q_full, q_use - 1);
  } else if (warp == kWMma) {
    // ---------------- MMA ----------------
    constexpr uint32_t id_s = um_idesc<BF>(128, 128), id_o = um_idesc<BF>(128, HD) | (1u << 16);
    uint32_t stage_use = 0, np[2] = {0, 0}, unit_no = 0;
    uint32_t vphase = 0;      // bit s: parity of v_ready[s]
    // (descriptors are formed where they are used: hoisted out of the loop they
    // spill, and a word from local memory takes 400 cycles here)
    auto fresh_base = [&] {
      uint8_t* p = sm;
      asm volatile("" : "+l"(p));
      return p;
    };
    auto issue_s = [&](int x, uint32_t st) {
      if (elect_one()) {
        uint8_t* base = fresh_base();
#pragma unroll
        for (int h = 0; h < NH; ++h) {
          const uint64_t da = smem_desc_sw128(base + x * S::kTileB + h * kHalfB);
          const uint64_t db = smem_desc_sw128(base + S::OFF_KV + st * S::kTileB + h * kHalfB);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) umma_f16(tmem + x * 128, da + (uint64_t)(kk * 2), db + (uint64_t)(kk * 2), id_s, (h | kk) != 0);
        }
        umma_commit(s_full + x);
      }
      __syncwarp();
    };
    auto issue_o = [&](int x, uint32_t st, bool acc) {
      if (elect_one()) {
        const uint64_t db = smem_desc_sw128_mn(fresh_base() + S::OFF_KV + st * S::kTileB);
#pragma unroll
        for (int kk = 0; kk < kUmKeys / 16; ++kk)
          umma_ts(tmem + 256 + x * 128, tmem + x * 128 + (kk < 4 ? kk * 8 : 32 + kk * 8), db + (uint64_t)(kk * (16 * 128 >> 4)), id_o, acc || kk != 0);
        umma_commit(pv_done + x);
      }
      __syncwarp();
    };
    for (uint32_t seg = 0;; ++seg) {
      const Segment* g = segment(seg);
      if (!g) break;
      const uint32_t take = g->take, n0 = g->n[0], n1 = g->n[1];
      const int mixed0 = g->seen(0) - (int)(g->unit * kUmKeys);      // from this key of the part on, not all rows see all
      wait(q_full, seg);
      for (uint32_t i = 0; i <= take; ++i) {
        // K of unit i, V of unit i - 1 (the ring holds K0 V0 K1 V1 ...)
        const uint32_t ku = stage_use + 2 * i, vu = stage_use + 2 * i - 1;
        const uint32_t ks = ku % S::kStages, vs = vu % S::kStages;
        if (i < take) wait(kv_full + ks, ku / S::kStages);
        if (i > 0) {
          wait(kv_full + vs, vu / S::kStages);
          if ((int)(i * kUmKeys) > mixed0) {                    // (unit i - 1 ends there)
            const uint32_t slot = unit_no % kPres;
            wait(v_ready + slot, vphase >> slot);
            vphase ^= 1u << slot;
          }
          ++unit_no;
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          if (i > 0 && i - 1 < (x ? n1 : n0)) {
            wait(p_full + x, np[x]);
            ++np[x];
            tc_fence_after();
            issue_o(x, vs, i > 1);
          }
          if (i < (x ? n1 : n0)) {
            tc_fence_after();
            issue_s(x, ks);
          }
          if (x == 0 && i < take && (int)((i + 1) * kUmKeys) > mixed0) {     // V of unit i has to be cleaned
            wait(kv_full + (ku + 1) % S::kStages, (ku + 1) / S::kStages);
            if (elect_one()) mbar_arrive1(v_go + unit_no % kPres);
            __syncwarp();
          }
        }
        if (elect_one()) {
          if (i > 0 && tries) umma_commit(kv_empty + vs);
          if (i < take && tries) umma_commit(kv_empty + ks);
          if (i + 1 == take && tries) umma_commit(q_empty);
        }
        __syncwarp();
      }
      stage_use += 2 * take;
      segment_done(seg);
    }
    if (stage_use) wait(kv_empty + (stage_use - 1) % S::kStages, (stage_use - 1) / S::kStages);   // the last arrival of a commit
    if (gave_up()) {
      if (elect_one()) umma_commit(drained);
      __syncwarp();
      landed(drained, 0);
    }
  }
  } else {
    // ---------------- softmax and epilogue of row tile x ----------------
    const int x = warp >> 3, half = (warp >> 2) & 1, bar = 1 + 4 * x + (warp & 3);
    const uint32_t r = 32u * (warp & 3) + lane;
    const uint32_t tl = tmem + ((32u * (warp & 3)) << 16);
    const uint32_t tS = tl + x * 128 + half * 64, tO = tl + 256 + x * 128 + half * (HD / 2);
    volatile uint32_t* xr = xt + x * 128 + r;
    uint32_t ns = 0, unit_no = 0;       // units of this row tile, units of the run
    uint32_t vphase = 0;                // bit s: parity of v_go[s]
    if (threadIdx.x == 0) t.ws.head[blockIdx.x] = {0, 0, 0, 0};
    // Part k of the run; both warps of a pair enter it or neither does.  Who
    // comes first decides (2 k + 2: entered, 2 k + 3: not); the other may be at
    // an earlier part still.  (A vote at the pair's barrier: 0.7 us of 512 tokens'
    // 36.7.)
    uint32_t* agreed = tslot + 1 + kPres + 4 * x + (warp & 3);
    auto enter = [&](uint32_t k) -> const Segment* {
      wait(seg_full + k % kSegs, k / kSegs);
      const Segment* g = segs + k % kSegs;
      bool no = gave_up();
      if (!no && g->take == 0) return nullptr;
      uint32_t old = 0;
      if (lane == 0) old = atomicCAS(agreed, 2 * k, 2 * k + (no ? 3 : 2));
      old = __shfl_sync(0xffffffffu, old, 0);
      if (old > 2 * k) no = old == 2 * k + 3;
      __syncwarp();
      return no ? nullptr : g;
    };
    // (of a part only what its every unit needs is kept in registers: the
    // loop's spills are read back from L2)
    for (uint32_t seg = 0;; ++seg) {
      const Segment* g = enter(seg);
      if (!g) break;
      const uint32_t units = g->n[x];
      auto token = [&] { return x * PT + (int)(r / G); };               // of the task
      const bool live = r < (uint32_t)PT * G && token() < g->rows;
      // the first unit with a key that some row of the task does not see
      const uint32_t special = g->gaps ? 0u : (uint32_t)max(0, g->seen(0) / kUmKeys - (int)g->unit);
      // A V row past the length is zeroed (its box holds earlier keys), and so
      // is every non-finite element of a row that some rows see and others do
      // not, or 0 * V would reach the others; the epilogue adds it to those
      // that do.  The 16 warps share the tile: one alone, with 8 loads in
      // flight beside the products', would need longer than a unit takes.
      auto clean = [&](uint32_t i) {
        constexpr int CH = HD / 8, N = 16 * 32;           // 16-byte chunks of a row; threads
        const int key0 = (int)((g->unit + i) * kUmKeys), task_all = g->seen(0), task_any = g->seen(g->rows - 1);
        if (key0 + kUmKeys <= task_all) return;
        const uint32_t use = 2 * (unit_no + i) + 1, st = use % S::kStages;
        const int lo = max(0, task_all - key0) * CH, hi = min(kUmKeys, max(0, task_any - key0)) * CH;
        const int base = max(0, task_any - 256);          // key of the first mark
        auto chunk = [&](int e) {
          return reinterpret_cast<uint4*>(sm + S::OFF_KV + st * S::kTileB + (e % CH >> 3) * kHalfB + sw128_off((uint32_t)(e / CH), (uint32_t)(e % CH & 7)));
        };
        // (every warp comes to every such unit, in order, so a parity cannot be
        // mistaken for another phase's; of kv_full it could, which runs on
        // without the warps of a row tile that does not look at a unit)
        const uint32_t slot = (unit_no + i) % kPres;
        wait(v_go + slot, vphase >> slot);
        vphase ^= 1u << slot;
        wait(kv_full + st, use / S::kStages);
        for (int e = hi + (int)threadIdx.x; e < kUmKeys * CH; e += N) *chunk(e) = make_uint4(0u, 0u, 0u, 0u);
        uint4 v[kUmKeys * CH / N];
#pragma unroll
        for (int j = 0; j < kUmKeys * CH / N; ++j) {
          const int e = lo + (int)threadIdx.x + j * N;
          v[j] = e < hi ? *chunk(e) : make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int j = 0; j < kUmKeys * CH / N; ++j) {
          if (!(bad_any<BF>(v[j].x) | bad_any<BF>(v[j].y) | bad_any<BF>(v[j].z) | bad_any<BF>(v[j].w))) continue;
          const int e = lo + (int)threadIdx.x + j * N;
          *chunk(e) = make_uint4(v[j].x & ~bad_mask<BF>(v[j].x), v[j].y & ~bad_mask<BF>(v[j].y), v[j].z & ~bad_mask<BF>(v[j].z),
                                 v[j].w & ~bad_mask<BF>(v[j].w));
          const uint32_t bit = (uint32_t)(key0 + e / CH - base);
          atomicOr(segs[seg % kSegs].marks + (bit >> 5), 1u << (bit & 31));
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive1(v_ready + slot);
      };
      float m = -kLift<T>, l = 0.f;
      bool fresh = true;              // no visible key among this thread's yet
      for (uint32_t i = 0; i < units; ++i) {
        wait(s_full + x, ns);
        tc_fence_after();
        if (i >= special) {
          const int key0 = (int)((g->unit + i) * kUmKeys);
          uint32_t mask = 0xFFFFu;
          const uint32_t sh = 31 - __clz(t.box);
          if (g->gaps) {
            const uint32_t un = unit_no + i;
            wait(pres_full + un % kPres, un / kPres);
            mask = pres[un % kPres];
          }
          if (g->gaps || key0 + kUmKeys > g->seen(x * PT))
            um_mask(tS, (live ? g->seen(token()) : 0) - key0 - 64 * half, mask >> ((64 * half) >> sh), sh);
        }
        uint32_t w[32];
        float sum;
        for (bool first = true;; first = false) {
          sum = um_pass<T>(tS, t.sl2, m, w);
          // Out of range: a sum of 2^15 or more (or NaN), or of less than kLeast
          // among the first keys that the row sees.
          const bool off = live && (!(sum < kMost) || (fresh && sum < kLeast<T>));
          if (!first || !pair_any(bar, off)) break;
          // both threads of a row: the same m, from both halves' maxima
          const float top = um_top(tS) * t.sl2;
          const float to = fmaxf(pair_tell(bar, xr, half, 0, top), pair_tell(bar, xr, half, 1, top)) - kLift<T>;
          const float say = (off ? 2.f : 0.f) + (fresh ? 1.f : 0.f);
          const float s0 = pair_tell(bar, xr, half, 0, say), s1 = pair_tell(bar, xr, half, 1, say);
          const bool all_fresh = s0 != 0.f && s0 != 2.f && s1 != 0.f && s1 != 2.f;
          float scale = 1.f;
          if (live && (s0 >= 2.f || s1 >= 2.f) && (to > m || (all_fresh && to > -INFINITY))) {
            if (!all_fresh) scale = ex2(m - to);     // else there is nothing to rescale
            m = to;
            l *= scale;
          }
          if (i > 0) {
            wait(pv_done + x, ns - 1);
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < HD / 64; ++c) {
              uint32_t o[32];
              tm_ld32(tO + 32 * c, o);
              tm_wait_ld(o);
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * scale);
              tmem_st32(tO + 32 * c, o);
            }
          }
          if (top > -INFINITY) fresh = false;
        }
        if (sum > 0.f) fresh = false;
        l += sum;
        tmem_st32(tS, w);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive1(p_full + x);
        ++ns;
        if (i >= special) clean(i);
      }
      for (uint32_t i = max(units, special); i < g->take; ++i) clean(i);      // units that only the other row tile looks at
      unit_no += g->take;
      if (x * PT < g->rows) {
        // the row's sum: both halves', in one order
        l = pair_tell(bar, xr, half, 0, l) + pair_tell(bar, xr, half, 1, l);
        const bool whole = g->parts == 0, first = g->unit == 0;
        const int tok = token(), row0 = g->row0;
        const uint32_t kvh = g->kvh;
        const float il = whole ? (l == 0.f ? 0.f : 1.f / l) : 1.f;
        const uint32_t rr = (uint32_t)x * PT * G + r;
        uint16_t* op = a.out + (int64_t)(row0 + tok) * a.out_stride + (int64_t)(kvh * G + r % G) * HD + half * (HD / 2);
        float* slot = t.ws.slot(blockIdx.x, first ? 1 : 0, HD);
        float* part = slot + 2 * t.ws.R + (size_t)rr * 4 + (size_t)half * (HD / 2) * t.ws.R;   // [HD / 4][R][4]: lanes side by side
        if (first && !whole && threadIdx.x == 0) t.ws.head[blockIdx.x] = {(uint32_t)row0, kvh, (uint32_t)g->rows * G, g->parts};
        if (live && !whole && half == 0) {
          slot[rr] = l == 0.f ? -INFINITY : m;
          slot[t.ws.R + rr] = l;
        }
        if (units) {
          wait(pv_done + x, ns - 1);
          tc_fence_after();
        }
        const volatile uint32_t* mk = g->marks;
        uint32_t marks = 0;      // some key of the segment has a non-finite V
        if (units)
          for (int w = 0; w < 8; ++w) marks |= mk[w];
#pragma unroll 1
        for (int c = 0; c < HD / 64; ++c) {
          uint32_t w[32];
          float o[32];
          if (units) {
            tm_ld32(tO + 32 * c, w);
            tm_wait_ld(w);
          }
#pragma unroll
          for (int d = 0; d < 32; ++d) o[d] = units ? __uint_as_float(w[d]) * il : 0.f;
          if (marks) add_nonfinite<BF>(a, *g, mk, live ? g->seen(tok) : 0, half * (HD / 2) + 32 * c, o);
          if (live && whole) {
#pragma unroll
            for (int d = 0; d < 32; d += 8)
              *reinterpret_cast<uint4*>(op + 32 * c + d) = make_uint4(T16<T>::pack(o[d], o[d + 1]), T16<T>::pack(o[d + 2], o[d + 3]),
                                                                      T16<T>::pack(o[d + 4], o[d + 5]), T16<T>::pack(o[d + 6], o[d + 7]));
          } else if (live) {
#pragma unroll
            for (int d = 0; d < 32; d += 4)
              *reinterpret_cast<float4*>(part + (size_t)(32 * c + d) * t.ws.R) = make_float4(o[d], o[d + 1], o[d + 2], o[d + 3]);
          }
        }
        tc_fence_before();
      }
      segment_done(seg);
    }
  }
  if (gave_up() && lane == 0) atomicOr(a.err, ERR_MBAR_TIMEOUT);
  tc_fence_before();
  __syncthreads();
  if (warp == kWMma) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

template <typename T, int HD>
cudaError_t umma_go(const UmArgs& t, cudaStream_t st) {
  static std::atomic<uint64_t> ready{0};
  const cudaError_t e = raise_smem((const void*)&paged_umma_kernel<T, HD>, (int)UmShape<HD>::kSmem, ready);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(t.workers);
  cfg.blockDim = dim3(kUmThreads);
  cfg.dynamicSmemBytes = UmShape<HD>::kSmem;
  cfg.stream = st;
  return cudaLaunchKernelEx(&cfg, &paged_umma_kernel<T, HD>, t);
}

}  // namespace

size_t paged_umma_ws(int num_sms, int hd) { return part_ws_bytes((uint32_t)num_sms, kUmmaRows, (uint32_t)hd); }

cudaError_t paged_umma_launch(const PagedAttnArgs& a, int dtype, int hd, cudaStream_t st) {
  UmArgs t;
  t.a = a;
  t.workers = (uint32_t)a.num_sms;
  t.ws = part_ws(a.ws, t.workers, kUmmaRows);
  t.box = 8;
  while (t.box < (uint32_t)kUmKeys && a.kv.page_size % (2 * t.box) == 0) t.box *= 2;
  const uint32_t G = a.n_q / a.kv.n_kv;
  t.pt = 128 / G;
  t.sl2 = a.scale * 1.4426950408889634f;
  if (!paged_tensor_map(&t.tmK, a.kv, a.kv.k, hd, t.box) || !paged_tensor_map(&t.tmV, a.kv, a.kv.v, hd, t.box) ||
      !paged_q_map(&t.tmQ, a, hd, G, t.pt))
    return cudaErrorInvalidValue;
  cudaError_t e;
  if (dtype == RD_F16) e = hd == 128 ? umma_go<__half, 128>(t, st) : umma_go<__half, 64>(t, st);
  else e = hd == 128 ? umma_go<__nv_bfloat16, 128>(t, st) : umma_go<__nv_bfloat16, 64>(t, st);
  if (e != cudaSuccess) return e;
  return paged_merge_tile_launch(a, t.ws, t.workers, dtype, hd, st);
}

}  // namespace nnz
