// How the paged attention kernels share their work: the key units of all
// tasks, one after the other, cut into equal runs, one run per worker.
//
// A task is one (sequence, kv head, tile of query rows); its units are tiles
// of KT keys (one unit at least, so that rows without keys get their zeros).
// Worker w takes units [w per, (w + 1) per) of the concatenation in task
// order: whatever the mix of lengths, all workers finish together, and a
// worker splits at most two tasks (its first and its last).  A worker that
// holds a whole task writes its output; of a split task every worker leaves a
// partial (max, sum, sum p v) in the workspace, the task's first part in slot
// 1 of its worker, the others in slot 0 of theirs, and the first part's
// worker leaves a header that the merge kernel goes by.  The cut depends on
// the lengths alone, so results do not change from call to call.
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

// Units of one kv head of one sequence.
__device__ __forceinline__ uint64_t head_units(const SeqInfo& q, int QT, int KT) {
  uint64_t u = 0;
  for (int qt = 0; qt * QT < q.rows; ++qt) u += tile_units(q, qt, QT, KT);
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

// Moves to the unit `skip` units on.
__device__ __forceinline__ bool cursor_skip(const PagedAttnArgs& a, Cursor& c, uint64_t skip, int QT, int KT) {
  for (;;) {
    if (c.unit == 0 && c.qt == 0) {   // whole heads first
      const uint64_t hu = head_units(c.q, QT, KT);
      const uint64_t heads = a.kv.n_kv - c.kvh;
      if (skip >= hu * heads) {
        skip -= hu * heads;
        ++c.s;
        if (!cursor_seq(a, c, QT, KT)) return false;
        continue;
      }
      c.kvh += (uint32_t)(skip / hu);
      skip %= hu;
      c.units = tile_units(c.q, 0, QT, KT);
      while (skip >= c.units) {
        skip -= c.units;
        ++c.qt;
        c.units = tile_units(c.q, c.qt, QT, KT);
      }
      c.unit = (uint32_t)skip;
      return true;
    }
    const uint64_t rest = c.units - c.unit;
    if (skip < rest) {
      c.unit += (uint32_t)skip;
      return true;
    }
    skip -= rest;
    if (!cursor_next_task(a, c, QT, KT)) return false;
  }
}

// All units, and the sequence that holds unit `want(total)` with the units
// before it: every thread of the block calls this (NT threads, a multiple of
// 32).  `want` maps the total to the block's first unit.  Lengths that are
// out of range are reported by the thread that reads them.
struct BlockStart {
  uint64_t total, first, before;
  uint32_t seq;
};

template <int NT, typename Want>
__device__ __forceinline__ BlockStart block_start(const PagedAttnArgs& a, int QT, int KT, Want want) {
  __shared__ unsigned long long wsum[NT / 32];
  __shared__ unsigned long long found_before;
  __shared__ uint32_t found_seq;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  auto units_of = [&](uint32_t s, bool report) -> unsigned long long {
    if (s >= a.num_seqs) return 0ull;
    const SeqInfo q = seq_info(a, s);
    if (report && seq_bad(a, q)) atomicOr(a.err, ERR_BAD_PAGE);
    return q.rows > 0 ? head_units(q, QT, KT) * a.kv.n_kv : 0ull;
  };
  BlockStart b;
  b.total = 0;
  unsigned long long mine = 0;   // of the last chunk that this thread looked at
  for (uint32_t s0 = 0; s0 < a.num_seqs; s0 += NT) {
    mine = units_of(s0 + tid, blockIdx.x == 0);
    unsigned long long v = mine;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane == 0) wsum[warp] = v;
    __syncthreads();
    for (int w = 0; w < NT / 32; ++w) b.total += wsum[w];
    __syncthreads();
  }
  b.first = want(b.total);
  b.seq = 0;
  b.before = 0;
  if (b.first >= b.total) return b;
  unsigned long long base = 0;
  for (uint32_t s0 = 0; s0 < a.num_seqs; s0 += NT) {
    if (a.num_seqs > NT) mine = units_of(s0 + tid, false);
    unsigned long long inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long t = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += t;
    }
    if (lane == 31) wsum[warp] = inc;
    __syncthreads();
    unsigned long long off = base, all = base;
    for (int w = 0; w < NT / 32; ++w) {
      if (w < warp) off += wsum[w];
      all += wsum[w];
    }
    if (b.first >= off + inc - mine && b.first < off + inc) {
      found_seq = s0 + tid;
      found_before = off + inc - mine;
    }
    __syncthreads();
    if (b.first < all) break;
    base = all;
  }
  b.seq = found_seq;
  b.before = found_before;
  return b;
}

// ---- workspace: headers, then two slots of partials per worker ----------
struct PartHeader {
  uint32_t row0;    // first q / out row of the task
  uint32_t kvh;
  uint32_t rows;    // (token, head) rows, head fastest
  uint32_t parts;   // 0: the worker holds no first part of a split task
};

// One slot: R maxima (log2 domain), R sums, R x HD sums of p v (row by row
// from the streaming kernel, [HD / 4][R][4] from the tiled one).
__host__ __device__ constexpr size_t slot_floats(uint32_t R, uint32_t hd) { return (size_t)R * (hd + 2); }

struct PartWs {
  PartHeader* head;
  float* slots;
  uint32_t R;
  __device__ __forceinline__ float* slot(uint64_t worker, int which, uint32_t hd) const {
    return slots + (worker * 2 + which) * slot_floats(R, hd);
  }
};

inline size_t part_ws_bytes(uint32_t workers, uint32_t R, uint32_t hd) {
  return (((size_t)workers * sizeof(PartHeader) + 255) & ~(size_t)255) + (size_t)workers * 2 * slot_floats(R, hd) * 4;
}
inline PartWs part_ws(void* ws, uint32_t workers, uint32_t R) {
  return {static_cast<PartHeader*>(ws),
          reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + (((size_t)workers * sizeof(PartHeader) + 255) & ~(size_t)255)), R};
}

// Merges the parts of split tasks into the output (paged.cu); launched with
// programmatic dependent launch behind the kernel that left them.
cudaError_t paged_merge_launch(const PagedAttnArgs& a, const PartWs& ws, uint32_t workers, int dtype, int hd, cudaStream_t st);
cudaError_t paged_merge_tile_launch(const PagedAttnArgs& a, const PartWs& ws, uint32_t workers, int dtype, int hd, cudaStream_t st);

// Few query rows per kv head and sequence (at most 16): keys streamed by
// independent warps (paged_stream.cu).
constexpr uint32_t kStreamRows = 16;
uint32_t paged_stream_workers(int num_sms);
cudaError_t paged_stream_launch(const PagedAttnArgs& a, int dtype, int hd, cudaStream_t st);
// Many query rows: 2 x 128 to a CTA, tcgen05 (paged_umma.cu).
constexpr uint32_t kUmmaRows = 256;
cudaError_t paged_umma_launch(const PagedAttnArgs& a, int dtype, int hd, cudaStream_t st);

}  // namespace nnz
