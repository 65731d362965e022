// Attention of few query rows over paged K/V (at most 16 rows per sequence
// and kv head: single tokens, drafts of a few tokens): bound by the bytes of
// K and V.
//
// Every warp is a worker of the shared cut (paged_sched.cuh), 8 to a CTA and a
// CTA to an SM; the parts of a split task meet first within the CTA, then
// (where it spans CTAs) in the workspace, or, for one sequence, through the
// distributed shared memory of a cluster.  A warp streams its run of 16-key
// units through a private ring of shared memory, each unit four (or, with
// pages whose size is only a multiple of 8, eight) TMA copies of K and V
// halves with the 128-byte swizzle, so a unit's page may lie anywhere and
// ldmatrix reads without conflicts.  16 keys and 8 warps: a page of 16 is one
// unit, and 8 rings of 24 KB keep 190 KB of an SM's memory in flight.  S = Q K^T and
// O += P V are mma.m16n8k16 with the G heads of every new token as rows; the
// online softmax keeps its f32 maximum and sum in the score fragments' lanes.
// P enters the second product in the pool's type, the only one that the tensor
// cores multiply with V as it is stored (the sum is of P before it is rounded):
// half a unit in its last place in every weight, as much again as the result's
// own rounding at the most.  (The remainder of P as a second operand would take
// that away, and make NaN of an infinite V, by 0 times infinity.)
// The ring runs ahead across task boundaries.  Page numbers are read 32
// copies ahead, one per lane.
//
// Absent pages and keys past the length are not loaded or not trusted: their
// scores are masked, their V rows zeroed in shared memory.
//
// Measured (16 / 8 heads of 128, f16): 64 single tokens over 2017 .. 4032 keys
// 135 - 141 us by the board, 5.6 - 5.9 TB/s of K and V, 0.87 - 0.9 of a plain
// copy's rate; one token over 32767 keys (bf16) 30.7 us, 4.4 TB/s, and over 515
// keys 6.5 us, which is the launch, two dependent loads, four units and the merge
// over the cluster.  Farther from the bytes' time: 64 tokens with 8 / 2 heads of
// 64 35 us (15), 32 sequences of 4 or 8 new tokens over 1000 .. 4000 keys 74 and 86
// us (50).
#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include <math.h>

#include <atomic>

#include "paged_sched.cuh"
#include "paged_tma.cuh"

namespace cg = cooperative_groups;

namespace nnz {

namespace {

constexpr int kStWarps = 8;
constexpr int kStKeys = 16;

template <int HD>
struct StShape {
  static constexpr int kHalves = HD / 64;
  static constexpr int kBoxB = kStKeys * 128;                 // 16 keys x 64 dims
  static constexpr int kStageB = 2 * kHalves * kBoxB;          // K halves, V halves
  static constexpr int kStages = HD == 128 ? 3 : 6;
  static constexpr int kWarpB = kStages * kStageB + 1024;      // + barriers and flags, whole swizzle atoms
  static constexpr int kSmem = kStWarps * kWarpB + 1024;       // + alignment
};

// A warp's part of a task that it does not hold whole.
struct StPart {
  unsigned long long t0;   // the task's first unit
  const float* sums;       // a slot (paged_sched.cuh), shared or global memory
  uint32_t units;          // 0: no part
  uint32_t row0, kvh, rows;
};

struct StArgs {
  CUtensorMap tmK, tmV;
  PagedAttnArgs a;
  PartWs ws;
  float* park;         // a slot per warp
  uint32_t cluster;    // > 1: one sequence, CTAs in clusters
  uint32_t clusters;   // of a kv head (used as its length asks)
  uint32_t box;        // keys per copy: 16 or 8
  float sl2;           // scale * log2(e)
};

template <typename T>
__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (T16<T>::kBf16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr)
               : "memory");
}

// 16-byte chunk ch (dims 8 ch ..) of key row r of a tile of swizzled boxes.
__device__ __forceinline__ uint32_t st_off(int r, int ch) {
  return (uint32_t)((ch >> 3) * (kStKeys * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4));
}

// (m, l, o) of a row plus one more part of it; lane: HD / 32 dims.
template <int HD>
__device__ __forceinline__ void merge_part(float pm, float pl, const float* po, float& m, float& l, float (&o)[HD / 32]) {
  const float mn = fmaxf(m, pm), ms = mn == -INFINITY ? 0.f : mn;
  const float c = exp2f(m - ms), f = exp2f(pm - ms);
  m = mn;
  l = l * c + pl * f;
#pragma unroll
  for (int d = 0; d < HD / 32; ++d) o[d] = o[d] * c + po[d] * f;
}

template <typename T, int HD>
__device__ __forceinline__ void merge_out(const PagedAttnArgs& a, uint32_t row0, uint32_t kvh, uint32_t row, int G, int lane, float l,
                                          const float (&o)[HD / 32]) {
  const float il = l == 0.f ? 0.f : 1.f / l;
  uint16_t* op = a.out + ((int64_t)row0 + row / G) * a.out_stride + ((int64_t)kvh * G + row % G) * HD + lane * (HD / 32);
#pragma unroll
  for (int d = 0; d < HD / 32; d += 2) *reinterpret_cast<uint32_t*>(op + d) = T16<T>::pack(o[d] * il, o[d + 1] * il);
}

// ROWS8: at most 8 query rows (the lower half of every fragment is absent).
// CL: one sequence, CTAs in clusters.  (Asked for one CTA to an SM the compiler
// takes up to 255 registers, which one token over 32767 keys gains from, 30.2
// instead of 34.8 us, and 64 tokens lose from, 139 instead of 135.)
template <typename T, int HD, bool ROWS8, bool CL>
__global__ void __launch_bounds__(kStWarps * 32, CL ? 1 : 0) paged_stream_kernel(const __grid_constant__ StArgs t) {
  using S = StShape<HD>;
  constexpr int NR = ROWS8 ? 1 : 2;        // fragment row halves
  constexpr int KS = HD / 16;              // K steps of S
  constexpr int NT = HD / 8;               // n tiles of O
  extern __shared__ uint8_t smem_raw[];
  __shared__ StPart parts[kStWarps][2];     // that start before the warp's run or within it
  __shared__ StPart merge[2];                // split tasks whose last part is this CTA's
  __shared__ __align__(16) float gather[kStreamRows * (HD + 2)];     // a CTA's sums in a cluster; warps' in a merge
  float (*red)[HD + 2] = reinterpret_cast<float (*)[HD + 2]>(gather);
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const PagedAttnArgs& a = t.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q4 = lane & 3;
  uint8_t* ring = smem + warp * S::kWarpB;
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + S::kStages * S::kStageB);
  volatile uint32_t* there = reinterpret_cast<uint32_t*>(bars + S::kStages);   // copies present, one bit each
  if (lane == 0) {
    for (int s = 0; s < S::kStages; ++s) mbar_init(&bars[s], 1);
    fence_barrier_init();
  }
  __syncwarp();
  const int G = (int)(a.n_q / a.kv.n_kv);
  const int QT = (int)a.max_new;           // one tile holds all rows
  // The run of this warp.  One sequence: its part of the head that the cluster
  // has.  Few tasks: of a part of one task that the CTA has for itself, if that
  // makes no CTA's run longer than a quarter and 8 units (us, against the even
  // cut: 2 x 515 keys 11.3 / 16.9, 8 x 2048 22.6 / 29.5, 16 x 4000 50.3 / 74.8).
  // Else: of the even cut.  Positions of units: within the task, or (even cut)
  // in all tasks' concatenation.
  const uint32_t worker = blockIdx.x * kStWarps + warp;
  Cursor c;
  PartRun run{0, 0, 0};
  bool even = false;
  uint64_t mine = 0, u0 = 0, u1 = 0;
  uint32_t per = 1;
  if (CL) {
    const uint32_t id = blockIdx.x / t.cluster;
    c.s = 0;
    c.kvh = id / t.clusters;
    c.qt = 0;
    c.q = seq_info(a, 0);
    if (worker == 0 && lane == 0 && seq_bad(a, c.q)) atomicOr(a.err, ERR_BAD_PAGE);
    if (c.q.rows > 0) {
      c.units = tile_units(c.q, 0, QT, kStKeys);
      // as many clusters as get four units to a warp
      const uint32_t warps = t.cluster * kStWarps;
      run.parts = min(t.clusters, max(1u, c.units / (4 * warps)));
      run.part = id % t.clusters;
      if (run.part < run.parts) {
        const uint32_t n = run.parts * warps, w = run.part * warps + blockIdx.x % t.cluster * kStWarps + warp;
        u0 = (uint64_t)c.units * w / n;
        u1 = (uint64_t)c.units * (w + 1) / n;
        c.unit = (uint32_t)u0;
      }
    }
  } else {
    even = !warp_parts<1>(a, QT, kStKeys, lane, gridDim.x, [](uint32_t q) { return q / 4 + 8; }, worker == 0, blockIdx.x, nullptr, c, run);
    if (even) {
      const uint64_t total = warp_total(a, QT, kStKeys, lane, worker == 0, mine);
      per = (max(1u, (uint32_t)div_up(total, gridDim.x)) + kStWarps - 1) / kStWarps;
      u0 = (uint64_t)worker * per;
      u1 = min(u0 + per, total);
    } else if (run.parts) {
      const uint32_t n = run.end - c.unit;
      u0 = c.unit + n * warp / kStWarps;
      u1 = c.unit + n * (warp + 1) / kStWarps;
      c.unit = (uint32_t)u0;
    }
  }
  // CTAs that hold parts of the task that begins at unit t0
  const uint64_t cta_units = (uint64_t)per * kStWarps;
  auto first_cta = [&](uint64_t t0) -> uint32_t { return even ? (uint32_t)(t0 / cta_units) : blockIdx.x - run.part; };
  auto num_parts = [&](uint64_t t0, uint32_t units) -> uint32_t {
    return even ? (uint32_t)((t0 + units - 1) / cta_units - t0 / cta_units + 1) : run.parts;
  };
  if (lane < 2) parts[warp][lane].units = 0;
  __syncwarp();
  if (u0 < u1) {
  if (even) warp_find(a, QT, kStKeys, lane, u0, mine, c);

  // ---- producer: copies of one unit, one per lane ----
  Cursor pc = c;
  uint32_t left = (uint32_t)(u1 - u0);      // units still to be issued
  const uint32_t nb = kStKeys / t.box;       // copies along the keys of a unit
  uint32_t page0 = 0, npage = 0;             // key boxes whose page numbers the lanes hold
  int my_page = -1;
  uint32_t my_at = 0;
  auto issue = [&](int stg) {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the slot was read, and maybe zeroed, by this warp
    __syncwarp();
    const uint32_t b0 = pc.unit * nb;
    if (b0 < page0 || b0 + nb > page0 + npage) {
      page0 = b0;
      npage = 32;
      const uint32_t key = (page0 + lane) * t.box, pi = key / a.kv.page_size;
      my_at = key - pi * a.kv.page_size;
      my_page = -1;
      if ((int64_t)key < pc.q.seen(pc.q.rows - 1)) {
        my_page = __ldg(a.page_table + (size_t)pc.s * a.table_stride + pi);
        if (my_page >= (int64_t)a.kv.num_pages) {
          atomicOr(a.err, ERR_BAD_PAGE);
          my_page = -1;
        }
      }
    }
    // one elected lane issues (a lane each takes the compiler's loop over
    // divergent operands, about 100 cycles a copy)
    const int i0 = (int)(b0 - page0), i1 = (int)(i0 + nb - 1);
    const int p0 = __shfl_sync(0xffffffffu, my_page, i0), p1 = __shfl_sync(0xffffffffu, my_page, i1);
    const int a0 = (int)__shfl_sync(0xffffffffu, my_at, i0), a1 = (int)__shfl_sync(0xffffffffu, my_at, i1);
    uint8_t* dst = ring + stg * S::kStageB;
    if (elect_one()) {
      const uint32_t have = (p0 >= 0 ? 1u : 0u) | (nb == 2 && p1 >= 0 ? 2u : 0u);
      there[stg] = have;
      mbar_arrive_expect_tx(&bars[stg], (uint32_t)__popc(have) * 2 * S::kHalves * t.box * 128);
#pragma unroll
      for (int part = 0; part < 2 * S::kHalves; ++part) {
        const CUtensorMap* tm = part < S::kHalves ? &t.tmK : &t.tmV;
        if (p0 >= 0) tma_load_4d(dst + part * S::kBoxB, tm, part % S::kHalves * 64, a0, (int)pc.kvh, p0, &bars[stg]);
        if (nb == 2 && p1 >= 0) tma_load_4d(dst + part * S::kBoxB + 8 * 128, tm, part % S::kHalves * 64, a1, (int)pc.kvh, p1, &bars[stg]);
      }
    }
    __syncwarp();
    --left;
    if (++pc.unit == pc.units) {
      npage = 0;
      if (left) cursor_next_task(a, pc, QT, kStKeys);
    }
  };
  int pstg = 0;
  for (int s = 0; s < S::kStages && left; ++s) {
    issue(pstg);
    pstg = pstg + 1 == S::kStages ? 0 : pstg + 1;
  }

  uint32_t flying = (uint32_t)(u1 - u0) - left;      // units issued and not waited for yet
  int cstg = 0;
  uint32_t phase = 0;       // bit s: parity of stage s
  uint64_t u = u0;
  for (;;) {
    const uint32_t take = (uint32_t)min((uint64_t)(c.units - c.unit), u1 - u);   // units of this task here
    const int nrow = c.q.rows * G;
    // query fragments of row g (and g + 8): row = token * G + head
    uint32_t qa[KS][2 * NR];
    int limit[NR];           // keys that the row sees
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const int row = g + 8 * r;
      const bool ok = row < nrow;
      const int tok = ok ? row / G : 0;
      limit[r] = ok ? (int)c.q.seen(tok) : 0;
      const uint16_t* qp = a.q + (c.q.row0 + tok) * a.q_stride + (int64_t)(c.kvh * G + (ok ? row - tok * G : 0)) * HD + 2 * q4;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        qa[ks][r] = ok ? __ldg(reinterpret_cast<const uint32_t*>(qp + 16 * ks)) : 0u;
        qa[ks][NR + r] = ok ? __ldg(reinterpret_cast<const uint32_t*>(qp + 16 * ks + 8)) : 0u;
      }
    }
    const int seen_all = (int)c.q.seen(0), seen_any = (int)c.q.seen(c.q.rows - 1);
    float o[NT][2 * NR];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 2 * NR; ++e) o[j][e] = 0.f;
    float m[NR], l[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      m[r] = -INFINITY;
      l[r] = 0.f;
    }
    for (uint32_t i = 0; i < take; ++i) {
      // A wait that gives up ends the copies, and is tried once more: none may
      // be under way when the ring is used again or the CTA is left.  (The
      // units that are then not loaded are worked on as the ring is.)
      if (flying) {
        --flying;
        auto landed = [&] {        // the warp as one
          for (uint32_t n = 0; !__all_sync(0xffffffffu, mbar_try_wait(&bars[cstg], (phase >> cstg) & 1u));)
            if (++n == kSpinLimit) return false;
          return true;
        };
        if (!landed()) {
          left = 0;
          landed();
          if (lane == 0) atomicOr(a.err, ERR_MBAR_TIMEOUT);
        }
      }
      phase ^= 1u << cstg;
      const uint32_t kb = smem_u32(ring + cstg * S::kStageB), vb = kb + S::kHalves * S::kBoxB;
      const int key0 = (int)(c.unit + i) * kStKeys;
      const uint32_t have = there[cstg];
      const bool all_there = have == (1u << nb) - 1u;
      auto present = [&](int k) { return all_there || ((have >> (nb == 1 ? 0 : k >> 3)) & 1u); };   // k: key of the unit
      if (!all_there || key0 + kStKeys > seen_any) {
        // V rows that nothing may look at: zero, so that 0 * V stays 0
        for (int k = lane; k < kStKeys * HD / 8; k += 32) {
          const int r = k / (HD / 8);
          if (!present(r) || key0 + r >= seen_any)
            asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(vb + st_off(r, k % (HD / 8))), "r"(0u) : "memory");
        }
        __syncwarp();
      }
      // S = Q K^T: two n tiles of 8 keys
      float s[2][4];
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
        s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
        for (int kq = 0; kq < KS / 2; ++kq) {
          uint32_t r0, r1, r2, r3;
          ldsm4(kb + st_off(nt * 8 + (lane & 7), 4 * kq + (lane >> 3)), r0, r1, r2, r3);
          mma16<T>(s[nt], qa[2 * kq][0], ROWS8 ? 0u : qa[2 * kq][NR - 1], qa[2 * kq][NR], ROWS8 ? 0u : qa[2 * kq][2 * NR - 1], r0, r1);
          mma16<T>(s[nt], qa[2 * kq + 1][0], ROWS8 ? 0u : qa[2 * kq + 1][NR - 1], qa[2 * kq + 1][NR],
                   ROWS8 ? 0u : qa[2 * kq + 1][2 * NR - 1], r2, r3);
        }
      }
      uint32_t pa[2][2];       // [key half][row half]
      float pv[NR][4], mx[NR];
      const bool masked = !all_there || key0 + kStKeys > seen_all;
#pragma unroll
      for (int r = 0; r < NR; ++r) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int k = (e >> 1) * 8 + 2 * q4 + (e & 1);
          pv[r][e] = s[e >> 1][2 * r + (e & 1)] * t.sl2;
          if (masked && !(key0 + k < limit[r] && present(k))) pv[r][e] = -INFINITY;
        }
        mx[r] = fmaxf(fmaxf(pv[r][0], pv[r][1]), fmaxf(pv[r][2], pv[r][3]));
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
      }
      if (__any_sync(0xffffffffu, mx[0] > m[0] || mx[NR - 1] > m[NR - 1])) {
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          const float mn = fmaxf(m[r], mx[r]);
          const float al = m[r] == mn ? 1.f : ex2(m[r] - mn);     // 0 at the first key seen
          m[r] = mn;
          l[r] *= al;
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            o[j][2 * r] *= al;
            o[j][2 * r + 1] *= al;
          }
        }
      }
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        const float ms = m[r] == -INFINITY ? 0.f : m[r];      // nothing seen yet: every p is 2^-inf = 0
#pragma unroll
        for (int e = 0; e < 4; ++e) pv[r][e] = ex2(pv[r][e] - ms);
        l[r] += (pv[r][0] + pv[r][1]) + (pv[r][2] + pv[r][3]);
        pa[0][r] = T16<T>::pack(pv[r][0], pv[r][1]);
        pa[1][r] = T16<T>::pack(pv[r][2], pv[r][3]);
      }
      if (key0 + kStKeys > seen_all && nrow > G) {
        // Keys that some rows see and others do not: a non-finite V row would
        // reach the others as 0 * V.  Such a row (rare) is added in f32 to the
        // rows that see it and zeroed for the product.
        uint32_t bad = 0;      // lane r < 16: row r has a non-finite element
        if (lane < kStKeys)
          for (int ch = 0; ch < HD / 8; ++ch) {
            uint32_t w0, w1, w2, w3;
            asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(w0), "=r"(w1), "=r"(w2), "=r"(w3) : "r"(vb + st_off(lane, ch)) : "memory");
            constexpr bool bf = T16<T>::kBf16;
            bad |= bad_any<bf>(w0) | bad_any<bf>(w1) | bad_any<bf>(w2) | bad_any<bf>(w3);
          }
        uint32_t rows = __ballot_sync(0xffffffffu, bad != 0);
        while (rows) {
          const int k = __ffs(rows) - 1;
          rows &= rows - 1;
#pragma unroll
          for (int r = 0; r < NR; ++r) {
            float p = 0.f;     // p of (row g + 8 r, key k): held by lane 4 g + (k % 8) / 2
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float x = __shfl_sync(0xffffffffu, pv[r][e], (lane & ~3) | ((k & 7) >> 1));
              if (e == (k >> 3) * 2 + (k & 1)) p = x;
            }
            if (key0 + k < limit[r])
#pragma unroll
              for (int j = 0; j < NT; ++j) {
                uint32_t w;
                asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(vb + st_off(k, j) + 4 * q4) : "memory");
                const float2 f = T16<T>::to_f2(w);
                o[j][2 * r] = fmaf(p, f.x, o[j][2 * r]);
                o[j][2 * r + 1] = fmaf(p, f.y, o[j][2 * r + 1]);
              }
          }
          __syncwarp();
          if (lane < HD / 8)
            asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(vb + st_off(k, lane)), "r"(0u) : "memory");
          __syncwarp();
        }
      }
      // O += P V
#pragma unroll
      for (int jp = 0; jp < NT / 2; ++jp) {
        uint32_t r0, r1, r2, r3;
        ldsm4t(vb + st_off((lane & 7) + 8 * ((lane >> 3) & 1), 2 * jp + (lane >> 4)), r0, r1, r2, r3);
        if constexpr (ROWS8) {
          float d0[4] = {o[2 * jp][0], o[2 * jp][1], 0.f, 0.f}, d1[4] = {o[2 * jp + 1][0], o[2 * jp + 1][1], 0.f, 0.f};
          mma16<T>(d0, pa[0][0], 0u, pa[1][0], 0u, r0, r1);
          mma16<T>(d1, pa[0][0], 0u, pa[1][0], 0u, r2, r3);
          o[2 * jp][0] = d0[0];
          o[2 * jp][1] = d0[1];
          o[2 * jp + 1][0] = d1[0];
          o[2 * jp + 1][1] = d1[1];
        } else {
          mma16<T>(reinterpret_cast<float(&)[4]>(o[2 * jp]), pa[0][0], pa[0][NR - 1], pa[1][0], pa[1][NR - 1], r0, r1);
          mma16<T>(reinterpret_cast<float(&)[4]>(o[2 * jp + 1]), pa[0][0], pa[0][NR - 1], pa[1][0], pa[1][NR - 1], r2, r3);
        }
      }
      __syncwarp();
      if (left) {              // refill the slot just consumed
        issue(cstg);
        ++flying;
      }
      cstg = cstg + 1 == S::kStages ? 0 : cstg + 1;
    }
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    }
    if (take == c.units && !CL) {
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        const int row = g + 8 * r;
        if (row >= nrow) continue;
        const float il = l[r] == 0.f ? 0.f : 1.f / l[r];
        uint16_t* op = a.out + (c.q.row0 + row / G) * a.out_stride + (int64_t)(c.kvh * G + row % G) * HD + 2 * q4;
#pragma unroll
        for (int j = 0; j < NT; ++j) *reinterpret_cast<uint32_t*>(op + 8 * j) = T16<T>::pack(o[j][2 * r] * il, o[j][2 * r + 1] * il);
      }
    } else {
      // the last part of the run goes to the ring, which nothing fills any
      // more; one before it, with copies under way, to global memory
      const int which = c.unit == 0 ? 1 : 0;
      float* slot = u + take == u1 ? reinterpret_cast<float*>(ring) : t.park + (size_t)worker * slot_floats(kStreamRows, HD);
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        const int row = g + 8 * r;
        if (row >= nrow) continue;
        if (q4 == 0) {
          slot[row] = m[r];
          slot[kStreamRows + row] = l[r];
        }
        float* op = slot + 2 * kStreamRows + row * HD + 2 * q4;
#pragma unroll
        for (int j = 0; j < NT; ++j) *reinterpret_cast<float2*>(op + 8 * j) = make_float2(o[j][2 * r], o[j][2 * r + 1]);
      }
      if (lane == 0) parts[warp][which] = {u - c.unit, slot, c.units, (uint32_t)c.q.row0, c.kvh, (uint32_t)nrow};
    }
    u += take;
    c.unit += take;
    if (u >= u1) break;
    cursor_next_task(a, c, QT, kStKeys);
  }
  }

  if (CL) {
    // ---- one task: the CTA's parts, then the cluster's in its first CTA ----
    cg::cluster_group cl = cg::this_cluster();
    if (run.part >= run.parts) return;                    // the whole cluster
    __syncthreads();
    const uint32_t rows = (uint32_t)(c.q.rows * G), rank = blockIdx.x % t.cluster, id = blockIdx.x / t.cluster;
    for (uint32_t row = warp; row < rows; row += kStWarps) {
      float m = -INFINITY, l = 0.f, o[HD / 32];
#pragma unroll
      for (int d = 0; d < HD / 32; ++d) o[d] = 0.f;
      for (int k = 0; k < 2 * kStWarps; ++k) {
        const StPart& p = parts[k >> 1][k & 1];
        if (!p.units) continue;
        merge_part<HD>(p.sums[row], p.sums[kStreamRows + row], p.sums + 2 * kStreamRows + row * HD + lane * (HD / 32), m, l, o);
      }
      float* q = gather + row * (HD + 2);
      if (lane == 0) {
        q[HD] = m;
        q[HD + 1] = l;
      }
#pragma unroll
      for (int d = 0; d < HD / 32; ++d) q[lane * (HD / 32) + d] = o[d];
    }
    cl.sync();
    // CTA r of the cluster sums rows r, r + cluster, ..
    for (uint32_t row = rank + t.cluster * warp; row < rows; row += t.cluster * kStWarps) {
      float m = -INFINITY, l = 0.f, o[HD / 32];
#pragma unroll
      for (int d = 0; d < HD / 32; ++d) o[d] = 0.f;
#pragma unroll 4
      for (uint32_t k = 0; k < t.cluster; ++k) {
        const float* q = cl.map_shared_rank(gather, k) + row * (HD + 2);
        float po[HD / 32];
#pragma unroll
        for (int d = 0; d < HD / 32; ++d) po[d] = q[lane * (HD / 32) + d];
        merge_part<HD>(q[HD], q[HD + 1], po, m, l, o);
      }
      if (run.parts == 1) {
        merge_out<T, HD>(a, (uint32_t)c.q.row0, c.kvh, row, G, lane, l, o);
      } else {
        float* slot = t.ws.slot(id, 0, HD);
        if (lane == 0) {
          slot[row] = m;
          slot[kStreamRows + row] = l;
        }
#pragma unroll
        for (int d = 0; d < HD / 32; ++d) slot[2 * kStreamRows + row * HD + lane * (HD / 32) + d] = o[d];
      }
    }
    if (run.parts > 1) __threadfence();
    cl.sync();      // the CTAs' sums have been read, the cluster's are stored
    if (run.parts == 1 || rank != 0) return;
    if (threadIdx.x == 0) merge[0].units = part_done(t.ws, id - run.part, run.parts) ? 1u : 0u;
    __syncthreads();
    if (!merge[0].units) return;
    for (uint32_t row = warp; row < rows; row += kStWarps) {
      float m = -INFINITY, l = 0.f, o[HD / 32];
#pragma unroll
      for (int d = 0; d < HD / 32; ++d) o[d] = 0.f;
#pragma unroll 4
      for (uint32_t k = 0; k < run.parts; ++k) {
        const float* q = t.ws.slot(id - run.part + k, 0, HD);
        float po[HD / 32];
#pragma unroll
        for (int d = 0; d < HD / 32; ++d) po[d] = __ldcg(q + 2 * kStreamRows + row * HD + lane * (HD / 32) + d);
        merge_part<HD>(__ldcg(q + row), __ldcg(q + kStreamRows + row), po, m, l, o);
      }
      merge_out<T, HD>(a, (uint32_t)c.q.row0, c.kvh, row, G, lane, l, o);
    }
    return;
  }

  // ---- the CTA's parts: groups of one task each, a warp per group ----
  if (threadIdx.x < 2) merge[threadIdx.x].units = 0;
  __syncthreads();
  {
    // lane i < 16: part i, in order; a group starts where the task changes
    const StPart* all = &parts[0][0];
    const bool have = lane < 2 * kStWarps && all[lane].units != 0;
    const unsigned long long t0 = have ? all[lane].t0 : 0;
    const uint32_t valid = __ballot_sync(0xffffffffu, have), below = valid & ((1u << lane) - 1u);
    const unsigned long long prev = __shfl_sync(0xffffffffu, t0, below ? 31 - __clz(below) : 0);
    uint32_t starts = __ballot_sync(0xffffffffu, have && (!below || prev != t0));
    for (int n = 0; n < warp && starts; ++n) starts &= starts - 1;      // the group of this warp ..
    while (starts) {
      const int i = __ffs(starts) - 1;
      const uint32_t later = starts & (starts - 1);
      const uint32_t members = valid & ~((1u << i) - 1u) & (later ? (1u << (__ffs(later) - 1)) - 1u : 0xFFFFFFFFu);
      const StPart p = all[i];
      const uint32_t c0 = first_cta(p.t0), np = num_parts(p.t0, p.units);
      float* slot = t.ws.slot(blockIdx.x, c0 == blockIdx.x ? 1 : 0, HD);
      for (uint32_t row = 0; row < p.rows; ++row) {
        float m = -INFINITY, l = 0.f, o[HD / 32];
#pragma unroll
        for (int d = 0; d < HD / 32; ++d) o[d] = 0.f;
        for (uint32_t k = members; k; k &= k - 1) {
          const float* q = all[__ffs(k) - 1].sums;
          merge_part<HD>(q[row], q[kStreamRows + row], q + 2 * kStreamRows + row * HD + lane * (HD / 32), m, l, o);
        }
        if (np == 1) {
          merge_out<T, HD>(a, p.row0, p.kvh, row, G, lane, l, o);
        } else {
          if (lane == 0) {
            slot[row] = m;
            slot[kStreamRows + row] = l;
          }
#pragma unroll
          for (int d = 0; d < HD / 32; ++d) slot[2 * kStreamRows + row * HD + lane * (HD / 32) + d] = o[d];
        }
      }
      if (np > 1) {
        __threadfence();
        __syncwarp();
        if (lane == 0 && part_done(t.ws, c0, np)) merge[c0 == blockIdx.x ? 1 : 0] = p;
      }
      for (int n = 0; n < kStWarps && starts; ++n) starts &= starts - 1;   // .. and every eighth after it
    }
  }
  __syncthreads();
  // ---- split tasks that this CTA completed ----
#pragma unroll 1
  for (int i = 0; i < 2; ++i) {
    const StPart p = merge[i];
    if (!p.units) continue;
    const uint32_t c0 = first_cta(p.t0), n = num_parts(p.t0, p.units);
    const int sw = p.rows > 4 ? 1 : p.rows > 2 ? 2 : p.rows > 1 ? 4 : 8;   // warps to a row
    const int split = warp % sw;
    for (uint32_t r0 = 0; r0 < p.rows; r0 += kStWarps / sw) {
      const uint32_t row = r0 + warp / sw;
      const bool live = row < p.rows;
      float m = -INFINITY, l = 0.f, o[HD / 32];
#pragma unroll
      for (int d = 0; d < HD / 32; ++d) o[d] = 0.f;
      if (live) {
#pragma unroll 4
        for (uint32_t k = split; k < n; k += sw) {
          const float* q = t.ws.slot(c0 + k, k == 0 ? 1 : 0, HD);
          float po[HD / 32];      // another SM's stores: from L2
#pragma unroll
          for (int d = 0; d < HD / 32; ++d) po[d] = __ldcg(q + 2 * kStreamRows + row * HD + lane * (HD / 32) + d);
          merge_part<HD>(__ldcg(q + row), __ldcg(q + kStreamRows + row), po, m, l, o);
        }
      }
      if (sw > 1) {
        if (lane == 0) {
          red[warp][HD] = m;
          red[warp][HD + 1] = l;
        }
#pragma unroll
        for (int d = 0; d < HD / 32; ++d) red[warp][lane * (HD / 32) + d] = o[d];
        __syncthreads();
        if (split == 0)
          for (int k = 1; k < sw; ++k)
            merge_part<HD>(red[warp + k][HD], red[warp + k][HD + 1], &red[warp + k][lane * (HD / 32)], m, l, o);
        __syncthreads();
      }
      if (live && split == 0) merge_out<T, HD>(a, p.row0, p.kvh, row, G, lane, l, o);
    }
  }
}

// Clusters for one sequence (its parts then meet through distributed shared
// memory; through the workspace they take 5 us longer): 8 CTAs to a head where
// the page table holds at most 4096 keys, else as many clusters of 4 as the
// device runs at once.  One row, 16 / 8 heads of 128, us by length:
//   keys       515   2048   8192   32767
//   8 x 1      6.7    8.7   18.1    51.5
//   4 x 4      8.2   11.5   16.4    32.8
//   even cut  11.5   12.8   20.9    36.1
template <typename K>
void stream_clusters(K* fn, StArgs& t, cudaLaunchConfig_t cfg, PerDevice (&fits)[9]) {
  const uint64_t keys = (uint64_t)t.a.table_stride * t.a.kv.page_size;
  for (uint32_t C = keys <= 4096 ? 8 : 4; C >= 4; C /= 2) {
    // clusters of C that the device runs at once (asked once; -1: none)
    const int n = fits[C].get([&] {
      cudaLaunchAttribute at[1];
      at[0].id = cudaLaunchAttributeClusterDimension;
      at[0].val.clusterDim.x = C;
      at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
      cfg.gridDim = dim3(C);
      cfg.attrs = at;
      cfg.numAttrs = 1;
      int most = 0;
      if (cudaOccupancyMaxActiveClusters(&most, fn, &cfg) == cudaSuccess && most > 0) return most;
      cudaGetLastError();
      return -1;
    });
    const uint32_t n_kv = t.a.kv.n_kv;
    if (n >= (int)n_kv) {
      t.cluster = C;
      t.clusters = C == 8 ? 1u : (uint32_t)n / n_kv;
      return;
    }
  }
}

template <typename T, int HD, bool ROWS8>
cudaError_t stream_go(StArgs t, cudaStream_t st) {
  static std::atomic<uint64_t> ready[2] = {};
  static PerDevice fits[9];
  const auto fn = &paged_stream_kernel<T, HD, ROWS8, false>;
  const auto fc = &paged_stream_kernel<T, HD, ROWS8, true>;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kStWarps * 32);
  cfg.dynamicSmemBytes = StShape<HD>::kSmem;
  cfg.stream = st;
  t.cluster = t.clusters = 1;
  if (t.a.num_seqs == 1) {
    const cudaError_t e = raise_smem((const void*)fc, StShape<HD>::kSmem, ready[1]);
    if (e != cudaSuccess) return e;
    stream_clusters(fc, t, cfg, fits);
  }
  if (t.cluster == 1) {
    const cudaError_t e = raise_smem((const void*)fn, StShape<HD>::kSmem, ready[0]);
    if (e != cudaSuccess) return e;
    cfg.gridDim = dim3((uint32_t)t.a.num_sms);
    cfg.numAttrs = 0;
    return cudaLaunchKernelEx(&cfg, fn, t);
  }
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = t.cluster;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(t.cluster * t.clusters * t.a.kv.n_kv);
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, fc, t);
}

template <typename T>
cudaError_t stream_t(const StArgs& t, int hd, cudaStream_t st) {
  const bool r8 = (uint64_t)t.a.max_new * (t.a.n_q / t.a.kv.n_kv) <= 8;
  if (hd == 128) return r8 ? stream_go<T, 128, true>(t, st) : stream_go<T, 128, false>(t, st);
  return r8 ? stream_go<T, 64, true>(t, st) : stream_go<T, 64, false>(t, st);
}

}  // namespace

size_t paged_stream_ws(int num_sms, int hd) {
  return part_ws_bytes((uint32_t)num_sms, kStreamRows, (uint32_t)hd) +
         (size_t)num_sms * kStWarps * slot_floats(kStreamRows, (uint32_t)hd) * 4;
}

cudaError_t paged_stream_launch(const PagedAttnArgs& a, int dtype, int hd, cudaStream_t st) {
  StArgs t;
  t.a = a;
  t.ws = part_ws(a.ws, (uint32_t)a.num_sms, kStreamRows);
  t.park = reinterpret_cast<float*>(static_cast<uint8_t*>(a.ws) + part_ws_bytes((uint32_t)a.num_sms, kStreamRows, (uint32_t)hd));
  t.box = a.kv.page_size % 16 ? 8 : 16;
  t.sl2 = a.scale * 1.4426950408889634f;
  if (!paged_tensor_map(&t.tmK, a.kv, a.kv.k, hd, t.box) || !paged_tensor_map(&t.tmV, a.kv, a.kv.v, hd, t.box))
    return cudaErrorInvalidValue;
  return dtype == RD_F16 ? stream_t<__half>(t, hd, st) : stream_t<__nv_bfloat16>(t, hd, st);
}

}  // namespace nnz
