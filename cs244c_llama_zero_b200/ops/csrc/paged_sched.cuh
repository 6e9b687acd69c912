// How the attention kernels over a paged cache divide their work.
//
// An ITEM is the product of one kv head with one tile of a sequence's new tokens (tile_tokens tokens times
// the heads that share the kv head).  It reads item_units() UNITS of cached tokens.  All units of all items
// lie on one axis (sequences, in each the kv heads, in each the tiles, in each the units), which is cut into
// as many equal ranges as there are blocks: every block streams the same number of units whatever the lengths
// of the sequences are.  A block's range covers some items whole, whose rows it finishes itself, and at most
// two in part (its first and its last one): those go to the workspace as unnormalised sums with their maxima
// and sums of exponentials, and a second kernel joins them in the order of the blocks, so that results do
// not depend on timing.
#pragma once

#include "paged.h"

namespace b200 {

struct PagedShape {
  int tile_tokens;  // new tokens of an item
  int unit_log2;    // cached tokens of a unit
  int kv_heads;
};

__host__ __device__ inline int ceil_div(int a, int b) { return (a + b - 1) / b; }

// Cached tokens that the last row of tile rt sees (0 or less: none).
__host__ __device__ inline int item_visible(const SeqInfo& s, int rt, int tile_tokens) {
  const long long end = (long long)(rt + 1) * tile_tokens;
  return s.len - s.qn + (int)(end < s.qn ? end : s.qn);
}

// An item of rows that see nothing has one unit all the same: somebody has to write its zeros.
__host__ __device__ inline int item_units(const SeqInfo& s, int rt, const PagedShape& sh) {
  const int vis = item_visible(s, rt, sh.tile_tokens);
  return vis > 0 ? ((vis - 1) >> sh.unit_log2) + 1 : 1;
}

__host__ __device__ inline long long head_units(const SeqInfo& s, const PagedShape& sh) {
  long long n = 0;
  const int tiles = ceil_div(s.qn, sh.tile_tokens);
  for (int rt = 0; rt < tiles; ++rt) n += item_units(s, rt, sh);
  return n;
}

// First unit of block c's range among g blocks, and the block whose range holds unit u.  Every range is
// non-empty (g <= total).
__host__ __device__ inline long long range_begin(long long c, long long total, long long g) { return c * total / g; }
__host__ __device__ inline int block_of_unit(long long u, long long total, long long g) {
  long long c = u * g / total;
  while (range_begin(c + 1, total, g) <= u) ++c;
  return (int)c;
}

struct PagedItem {
  int b, kvh, rt;
  int n_units;
  long long start;  // its first unit
  SeqInfo seq;
};

// The item that holds unit u, given a sequence b that holds it and that sequence's first unit.
__host__ __device__ inline PagedItem item_at(const PagedSeqs& s, const PagedShape& sh, int b, long long base,
                                             long long u) {
  PagedItem it;
  it.b = b;
  it.seq = seq_info(s, b);
  const long long per_head = head_units(it.seq, sh);
  it.kvh = (int)((u - base) / per_head);
  it.start = base + it.kvh * per_head;
  it.rt = 0;
  it.n_units = item_units(it.seq, 0, sh);
  while (u >= it.start + it.n_units) {
    it.start += it.n_units;
    it.n_units = item_units(it.seq, ++it.rt, sh);
  }
  return it;
}

// The item after `it`; only called when there is one.
__host__ __device__ inline void next_item(PagedItem& it, const PagedSeqs& s, const PagedShape& sh) {
  it.start += it.n_units;
  if ((it.rt + 1) * (long long)sh.tile_tokens < it.seq.qn) {
    ++it.rt;
  } else {
    it.rt = 0;
    if (++it.kvh == sh.kv_heads) {
      it.kvh = 0;
      do {
        it.seq = seq_info(s, ++it.b);
      } while (it.seq.qn == 0 && it.b + 1 < s.batch);
    }
  }
  it.n_units = item_units(it.seq, it.rt, sh);
}

// What block c (c < blocks) leaves for the joining kernel: its first item.
struct PagedRecord {
  long long start;
  int n_units;
  int b, kvh, rt;
};

// Workspace of one call: header, records, (max, sum) and sums of the two part items of every block.
struct PagedWorkspace {
  long long* total;  // [2]: units, blocks with work
  PagedRecord* records;
  float2* ml;  // [2 * blocks][rows]
  float* o;    // [2 * blocks][rows][head_dim]
};
__host__ inline size_t paged_workspace_bytes(int blocks, int rows, int head_dim) {
  return 256 + (size_t)blocks * ((sizeof(PagedRecord) + 15) / 16 * 16) + 256 +
         (size_t)2 * blocks * rows * (sizeof(float2) + sizeof(float) * (size_t)head_dim) + 256;
}
__host__ inline PagedWorkspace paged_workspace(void* base, int blocks, int rows) {
  PagedWorkspace w;
  uint8_t* p = reinterpret_cast<uint8_t*>(base);
  w.total = reinterpret_cast<long long*>(p);
  p += 256;
  w.records = reinterpret_cast<PagedRecord*>(p);
  p += ((size_t)blocks * ((sizeof(PagedRecord) + 15) / 16 * 16) + 255) / 256 * 256;
  w.ml = reinterpret_cast<float2*>(p);
  w.o = reinterpret_cast<float*>(p + (size_t)2 * blocks * rows * sizeof(float2));
  return w;
}

#if defined(__CUDACC__)

struct PagedRange {
  long long total;  // all units
  int blocks;       // blocks with work: min(grid, total)
  int b;            // sequence that holds the block's first unit ...
  long long base;   // ... and that sequence's first unit
};

// Finds this block's part, by all THREADS threads (a multiple of 32, at most 1024).  Each thread sums the
// units of a run of sequences; the sums are scanned.  Sequences with bad metadata count nothing.
template <int THREADS>
__device__ inline PagedRange find_range(const PagedSeqs& s, const PagedShape& sh, DeviceErrors* errs) {
  __shared__ long long warp_sums[THREADS / 32];
  __shared__ long long found[2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = ceil_div(s.batch, THREADS);
  const int b0 = min(tid * per, s.batch), b1 = min(b0 + per, s.batch);
  long long mine = 0;
  for (int b = b0; b < b1; ++b) {
    const SeqInfo q = seq_info(s, b);
    if (!q.ok && blockIdx.x == 0) report_error(errs, kErrBadIndex, b);
    mine += head_units(q, sh) * sh.kv_heads;
  }
  long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) warp_sums[warp] = incl;
  if (tid == 0) found[0] = -1;
  __syncthreads();
  long long before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) before += warp_sums[w];
    total += warp_sums[w];
  }
  PagedRange r;
  r.total = total;
  r.blocks = (int)min((long long)gridDim.x, total);
  if ((int)blockIdx.x < r.blocks) {
    const long long u = range_begin(blockIdx.x, total, r.blocks);
    long long at = before + incl - mine;
    if (u >= at && u < at + mine) {
      for (int b = b0; b < b1; ++b) {
        const long long n = b1 - b0 == 1 ? mine : head_units(seq_info(s, b), sh) * sh.kv_heads;
        if (u < at + n) {
          found[0] = b;
          found[1] = at;
          break;
        }
        at += n;
      }
    }
  }
  __syncthreads();
  r.b = (int)found[0];
  r.base = found[1];
  return r;
}

#endif

}  // namespace b200
