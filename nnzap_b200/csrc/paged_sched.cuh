// How the paged attention kernels share their work: the key units of all
// tasks, one after the other, cut into equal runs, one run per worker.
//
// A task is one (sequence, kv head, tile of query rows); its units are tiles
// of KT keys (one unit at least, so that rows without keys get their zeros).
// Worker w takes units [w per, (w + 1) per) of the concatenation in task
// order: whatever the mix of lengths, all workers finish together, and a
// worker splits at most two tasks (its first and its last).  Where there are
// few tasks, a worker may take one part of one task instead (warp_parts).  A worker that
// holds a whole task writes its output; the parts of a split task (max, sum,
// sum p v) meet in the workspace and are merged by whoever finishes last.  The
// cut and the order of the merge depend on the lengths alone, so results do
// not change from call to call.
#pragma once
#include "paged.cuh"

namespace nnz {

struct SeqInfo {
  int64_t row0;   // first row of q / out
  int64_t n;      // new tokens as given (positions go by it)
  int rows;       // new tokens computed
  int64_t len;    // keys as given
  int64_t cap;    // keys that the table can name

  // keys [0, seen(i)) are visible to new token i
  __device__ __forceinline__ int64_t seen(int64_t i) const {
    const int64_t e = len < len - n + i + 1 ? len : len - n + i + 1;
    return e < 0 ? 0 : e < cap ? e : cap;
  }
};

__device__ __forceinline__ SeqInfo seq_info(const PagedAttnArgs& a, uint32_t s) {
  SeqInfo q;
  const int64_t qs = __ldg(a.q_start + s), qe = __ldg(a.q_start + s + 1);
  q.row0 = qs;
  q.n = qe - qs;
  q.len = __ldg(a.kv_len + s);
  q.cap = (int64_t)a.table_stride * a.kv.page_size;
  int64_t r = (qe < (int64_t)a.tokens ? qe : (int64_t)a.tokens) - qs;
  if (r > (int64_t)a.max_new) r = a.max_new;
  q.rows = qs < 0 || r < 0 ? 0 : (int)r;
  return q;
}

__device__ __forceinline__ bool seq_bad(const PagedAttnArgs& a, const SeqInfo& q) {
  return q.row0 < 0 || q.n < 0 || q.rows != q.n || q.len < 0 || q.len > q.cap;
}

// Units of tile `qt` (rows [qt QT, ...)) of one sequence and kv head.
__device__ __forceinline__ uint32_t tile_units(const SeqInfo& q, int qt, int QT, int KT) {
  const int last = min((qt + 1) * QT, q.rows) - 1;
  const int64_t k = q.seen(last);
  return k <= KT ? 1u : (uint32_t)((k + KT - 1) / KT);
}

// sum of floor((x i + y) / m) over i < n (Euclid on the lattice points).
__device__ __forceinline__ uint64_t floor_sum(uint32_t n, uint32_t m, uint32_t x, uint32_t y) {
  uint64_t sum = 0;
  for (;;) {
    if (x >= m) {
      sum += (uint64_t)n * (n - 1) / 2 * (x / m);
      x %= m;
    }
    if (y >= m) {
      sum += (uint64_t)n * (y / m);
      y %= m;
    }
    const uint64_t last = (uint64_t)x * n + y;
    if (last < m) return sum;
    if (last >> 32) {
      n = (uint32_t)(last / m);
      y = (uint32_t)(last % m);
    } else {                       // 32-bit division
      n = (uint32_t)last / m;
      y = (uint32_t)last % m;
    }
    const uint32_t t = m;
    m = x;
    x = t;
  }
}

// Units of one kv head of one sequence.
__device__ __forceinline__ uint64_t head_units(const SeqInfo& q, int QT, int KT) {
  const int tiles = (q.rows + QT - 1) / QT;
  if (tiles <= 1) return tiles ? tile_units(q, 0, QT, KT) : 0;
  const int64_t a0 = q.len - q.n + QT;       // keys that the first tile's last row sees
  if (a0 >= 1 && q.len - q.n + q.rows <= q.cap && a0 + (int64_t)tiles * QT < (1ll << 31))
    return floor_sum((uint32_t)tiles - 1, (uint32_t)KT, (uint32_t)QT, (uint32_t)a0 + KT - 1) + tile_units(q, tiles - 1, QT, KT);
  uint64_t u = 0;                             // rows without keys, or keys past the table
  for (int qt = 0; qt < tiles; ++qt) u += tile_units(q, qt, QT, KT);
  return u;
}

// A worker's place in the task order.
struct Cursor {
  uint32_t s, kvh;
  int qt;
  uint32_t unit, units;   // unit within the task, units of the task
  SeqInfo q;
};

// First task of sequence s or later; false past the last.
__device__ __forceinline__ bool cursor_seq(const PagedAttnArgs& a, Cursor& c, int QT, int KT) {
  for (; c.s < a.num_seqs; ++c.s) {
    c.q = seq_info(a, c.s);
    if (c.q.rows > 0) {
      c.kvh = 0;
      c.qt = 0;
      c.unit = 0;
      c.units = tile_units(c.q, 0, QT, KT);
      return true;
    }
  }
  return false;
}

__device__ __forceinline__ bool cursor_next_task(const PagedAttnArgs& a, Cursor& c, int QT, int KT) {
  c.unit = 0;
  if ((c.qt + 1) * QT < c.q.rows) {
    ++c.qt;
  } else {
    c.qt = 0;
    if (++c.kvh == a.kv.n_kv) {
      ++c.s;
      return cursor_seq(a, c, QT, KT);
    }
  }
  c.units = tile_units(c.q, c.qt, QT, KT);
  return true;
}

__device__ __forceinline__ uint64_t warp_sum64(uint64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Inclusive sum over the lanes up to this one.
template <typename V>
__device__ __forceinline__ V warp_scan(V v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V t = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += t;
  }
  return v;
}

// All units, a lane per sequence; `mine`: the lane's units in the
// last 32 sequences.  One lane of one warp of the grid reports lengths that
// are out of range.
__device__ __forceinline__ uint64_t warp_total(const PagedAttnArgs& a, int QT, int KT, int lane, bool report, uint64_t& mine) {
  uint64_t total = 0;
  for (uint32_t s0 = 0; s0 < a.num_seqs; s0 += 32) {
    mine = 0;
    if (s0 + lane < a.num_seqs) {
      const SeqInfo q = seq_info(a, s0 + lane);
      if (report && seq_bad(a, q)) atomicOr(a.err, ERR_BAD_PAGE);
      mine = head_units(q, QT, KT) * a.kv.n_kv;
    }
    total += mine;
  }
  return warp_sum64(total);
}

// The place of unit `want` (below the total) of the concatenated tasks.
__device__ __forceinline__ void warp_find(const PagedAttnArgs& a, int QT, int KT, int lane, uint64_t want, uint64_t mine, Cursor& c) {
  uint64_t before = 0;
  for (uint32_t s0 = 0;; s0 += 32) {
    if (a.num_seqs > 32) {
      mine = 0;
      if (s0 + lane < a.num_seqs) mine = head_units(seq_info(a, s0 + lane), QT, KT) * a.kv.n_kv;
    }
    const uint64_t inc = before + warp_scan(mine, lane);
    const uint32_t hit = __ballot_sync(0xffffffffu, want < inc);
    if (hit || s0 + 32 >= a.num_seqs) {
      const int l = hit ? __ffs(hit) - 1 : 0;
      c.s = s0 + l;
      want -= __shfl_sync(0xffffffffu, inc - mine, l);
      break;
    }
    before = __shfl_sync(0xffffffffu, inc, 31);
  }
  c.q = seq_info(a, c.s);
  const uint64_t hu = head_units(c.q, QT, KT);
  uint32_t rel;
  if (want < 0xFFFFFFFFull && hu < 0xFFFFFFFFull) {   // 32-bit division
    c.kvh = (uint32_t)want / (uint32_t)hu;
    rel = (uint32_t)want % (uint32_t)hu;
  } else {
    c.kvh = (uint32_t)(want / hu);
    rel = (uint32_t)(want % hu);
  }
  // the tile: 32 at a time
  for (int q0 = 0;; q0 += 32) {
    const uint32_t tu = (int64_t)(q0 + lane) * QT < c.q.rows ? tile_units(c.q, q0 + lane, QT, KT) : 0;
    const uint32_t inc = warp_scan(tu, lane);
    const uint32_t hit = __ballot_sync(0xffffffffu, rel < inc);
    if (hit || (int64_t)(q0 + 32) * QT >= c.q.rows) {
      const int l = hit ? __ffs(hit) - 1 : 0;
      c.qt = q0 + l;
      c.units = __shfl_sync(0xffffffffu, tu, l);
      c.unit = rel - __shfl_sync(0xffffffffu, inc - tu, l);
      break;
    }
    rel -= __shfl_sync(0xffffffffu, inc, 31);
  }
}

__device__ __forceinline__ uint64_t div_up(uint64_t x, uint32_t y) {
  return x >> 32 ? (x + y - 1) / y : ((uint32_t)x + (y - 1)) >= y - 1 ? ((uint32_t)x + (y - 1)) / y : (x + y - 1) / y;
}

// One part of one task per CTA, for few tasks: parts of at most q units, the
// smallest q of the even cut's .. slack more (in steps of 1/16) that makes at
// most `ctas` of them; false if there is none.  Lanes hold the (sequence, tile)
// pairs 32 i + lane, i < N (N > 1: in `sm`, 32 N words, and in loops that are
// not unrolled: every CTA starts with this, once, and waits for instructions).
struct PartRun {
  uint32_t part, parts;    // 0 parts: none for this CTA
  uint32_t end;            // of the part within the task (its start: c.unit)
};

template <int N, typename Slack>
__device__ __forceinline__ bool warp_parts(const PagedAttnArgs& a, int QT, int KT, int lane, uint32_t ctas, Slack slack, bool report,
                                           uint32_t cta, uint32_t* sm, Cursor& c, PartRun& run) {
  if (a.num_seqs > 32) return false;
  SeqInfo mine{0, 0, 0, 0, 0};
  if ((uint32_t)lane < a.num_seqs) {
    mine = seq_info(a, (uint32_t)lane);
    if (report && seq_bad(a, mine)) atomicOr(a.err, ERR_BAD_PAGE);
  }
  const int nt = (mine.rows + QT - 1) / QT, inc = warp_scan(nt, lane), D = __shfl_sync(0xffffffffu, inc, 31);
  if (D > 32 * N || (uint32_t)D * a.kv.n_kv > ctas) return false;
  uint32_t reg = 0, sum = 0;                  // sequence << 27 | units (of 16 keys or more, and keys are below 2^31)
#pragma unroll 1
  for (int j0 = 0; j0 < D; j0 += 32) {
    const int j = j0 + lane;
    int s = 0;        // its sequence: those before it end at or before j
    for (uint32_t l = 0; l < a.num_seqs; ++l) s += __shfl_sync(0xffffffffu, inc, (int)l) <= j ? 1 : 0;
    const int first = __shfl_sync(0xffffffffu, inc - nt, s & 31);
    uint32_t v = 0;
    if (j < D) {
      const uint32_t u = tile_units(seq_info(a, (uint32_t)s), j - first, QT, KT);
      sum += u;
      v = (uint32_t)s << 27 | u;
    }
    if constexpr (N > 1) sm[j] = v;
    else reg = v;
  }
  if (__any_sync(0xffffffffu, sum >> 26)) return false;      // (the sum over the lanes is 32-bit)
  auto pair = [&](int j0) { return N > 1 ? sm[j0 + lane] : reg; };
  constexpr uint32_t kUnits = (1u << 27) - 1;
  const uint32_t per = max(1u, (uint32_t)div_up((uint64_t)__reduce_add_sync(0xffffffffu, sum) * a.kv.n_kv, ctas));
  const uint32_t cap = ctas / a.kv.n_kv;      // parts of all pairs, per kv head
  const uint32_t q1 = per + slack(per);
#pragma unroll 1
  for (uint32_t q = per; q <= q1; q += max(1u, q / 16)) {
    uint32_t n = 0;
#pragma unroll 1
    for (int j0 = 0; j0 < D; j0 += 32) n += ((pair(j0) & kUnits) + q - 1) / q;
    if (__reduce_add_sync(0xffffffffu, n) > cap) continue;
    run = {0, 0, 0};
    uint32_t before = 0;                      // parts in order of pair, kv head, part
#pragma unroll 1
    for (int j0 = 0; j0 < D; j0 += 32) {
      const uint32_t v = pair(j0), np = ((v & kUnits) + q - 1) / q, all = np * a.kv.n_kv;
      const uint32_t incl = before + warp_scan(all, lane);
      const uint32_t hit = __ballot_sync(0xffffffffu, cta < incl && cta >= incl - all);
      if (hit) {
        const int l = __ffs(hit) - 1;
        const uint32_t rel = cta - __shfl_sync(0xffffffffu, incl - all, l), w = __shfl_sync(0xffffffffu, v, l);
        run.parts = __shfl_sync(0xffffffffu, np, l);
        c.units = w & kUnits;
        c.s = w >> 27;
        c.kvh = rel / run.parts;
        run.part = rel - c.kvh * run.parts;
        c.qt = l + j0 - (int)__shfl_sync(0xffffffffu, inc - nt, (int)c.s);
        const uint32_t each = c.units / run.parts, more = c.units - each * run.parts;     // the first `more` have one unit more
        c.unit = each * run.part + min(run.part, more);
        run.end = c.unit + each + (run.part < more ? 1u : 0u);
        c.q = seq_info(a, c.s);
        break;
      }
      before = __shfl_sync(0xffffffffu, incl, 31);
    }
    return true;
  }
  return false;
}

// ---- workspace: a header, a counter and two slots of partials per CTA ----
// A CTA's part of a split task goes to slot 1 of the CTA if it is the task's
// first, else to slot 0.
// Streaming kernel: the counter of the first part's CTA counts the parts that
// are there, and the CTA that completes it merges them, in order, and sets it
// back to 0: the workspace is zeroed once by its owner and every call leaves
// it as it found it.  Tiled kernel: the first part's CTA leaves a header, which
// a merge kernel goes by.
//
// One slot: R maxima (log2 domain), R sums, R x HD sums of p v (row by row
// from the streaming kernel, [HD / 4][R][4] from the tiled one).
__host__ __device__ constexpr size_t slot_floats(uint32_t R, uint32_t hd) { return (size_t)R * (hd + 2); }

struct PartHeader {
  uint32_t row0;    // first q / out row of the task
  uint32_t kvh;
  uint32_t rows;    // (token, head) rows, head fastest
  uint32_t parts;   // 0: the CTA holds no first part of a split task
};

struct PartWs {
  PartHeader* head;
  uint32_t* count;
  float* slots;
  uint32_t R;
  __device__ __forceinline__ float* slot(uint32_t cta, int which, uint32_t hd) const {
    return slots + ((size_t)cta * 2 + which) * slot_floats(R, hd);
  }
};

inline size_t part_ws_bytes(uint32_t ctas, uint32_t R, uint32_t hd) {
  return (((size_t)ctas * 20 + 255) & ~(size_t)255) + (size_t)ctas * 2 * slot_floats(R, hd) * 4;
}
inline PartWs part_ws(void* ws, uint32_t ctas, uint32_t R) {
  uint8_t* b = static_cast<uint8_t*>(ws);     // counters first: both kernels' workspaces begin with them
  return {reinterpret_cast<PartHeader*>(b + (size_t)ctas * 4), reinterpret_cast<uint32_t*>(b),
          reinterpret_cast<float*>(b + (((size_t)ctas * 20 + 255) & ~(size_t)255)), R};
}

// One thread, after its CTA's (or warp's) stores to a slot have been made
// visible: counts the part; true for the last one.
__device__ __forceinline__ bool part_done(const PartWs& ws, uint32_t first_cta, uint32_t parts) {
  __threadfence();
  if (atomicAdd(ws.count + first_cta, 1u) != parts - 1) return false;
  ws.count[first_cta] = 0;
  __threadfence();
  return true;
}

cudaError_t paged_merge_tile_launch(const PagedAttnArgs& a, const PartWs& ws, uint32_t workers, int dtype, int hd, cudaStream_t st);

// Few query rows per kv head and sequence (at most 16): keys streamed by
// independent warps (paged_stream.cu).
constexpr uint32_t kStreamRows = 16;
size_t paged_stream_ws(int num_sms, int hd);      // bytes of workspace
cudaError_t paged_stream_launch(const PagedAttnArgs& a, int dtype, int hd, cudaStream_t st);
// Many query rows: 2 x 128 to a CTA, tcgen05 (paged_umma.cu).
constexpr uint32_t kUmmaRows = 256;
size_t paged_umma_ws(int num_sms, int hd);
cudaError_t paged_umma_launch(const PagedAttnArgs& a, int dtype, int hd, cudaStream_t st);

}  // namespace nnz
