// How the attention kernels over a paged cache divide their work.
//
// An ITEM is the product of one kv head with one tile of a sequence's new tokens (tile_tokens tokens times
// the heads that share the kv head).  It reads item_units() UNITS of cached tokens.  All units of all items
// lie on one axis (sequences, in each the kv heads, in each the tiles, in each the units), which is cut into
// as many equal ranges as there are blocks, so that every block has the same to do whatever the lengths of the
// sequences are.  Each item takes kItemCost more places on the axis than it has units, ahead of them: changing
// items costs a block about as much as that many units (a batch of 256 ragged sequences of up to 2048 tokens
// took 60 us without, 52 us with it).  A cut that falls into these places moves to the item's start.
// A block's range covers some items whole, whose rows it finishes itself, and at most two in part (its first
// and its last one): those go to the workspace as unnormalised sums with their maxima and sums of
// exponentials, and a second kernel joins them in the order of the blocks, so that results do not depend on
// timing.
#pragma once

#include "paged.h"

namespace b200 {

constexpr int kItemCost = 2;

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

// Places of the items of one kv head on the axis.
__host__ __device__ inline long long head_places(const SeqInfo& s, const PagedShape& sh) {
  long long n = 0;
  const int tiles = ceil_div(s.qn, sh.tile_tokens);
  for (int rt = 0; rt < tiles; ++rt) n += item_units(s, rt, sh) + kItemCost;
  return n;
}

// Where block c's range would begin if cuts did not move (g <= total: all different).
__host__ __device__ inline long long raw_begin(long long c, long long total, long long g) { return c * total / g; }

struct PagedItem {
  int b, kvh, rt;
  int n_units;
  long long start;  // its first place
  SeqInfo seq;
};
__host__ __device__ inline long long item_end(const PagedItem& it) { return it.start + kItemCost + it.n_units; }
// A cut at place v inside the item, moved to the item's start if it falls ahead of its second unit.
__host__ __device__ inline long long moved_cut(const PagedItem& it, long long v) {
  return v <= it.start + kItemCost ? it.start : v;
}
// The item's unit at which a moved cut falls, or its number of units for a cut at or behind its end.
__host__ __device__ inline int unit_of_cut(const PagedItem& it, long long cut) {
  if (cut <= it.start) return 0;
  return cut >= item_end(it) ? it.n_units : (int)(cut - it.start - kItemCost);
}

// The item that holds place v, given a sequence b that holds it and that sequence's first place.
__host__ __device__ inline PagedItem item_at(const PagedSeqs& s, const PagedShape& sh, int b, long long base,
                                             long long v) {
  PagedItem it;
  it.b = b;
  it.seq = seq_info(s, b);
  const long long per_head = head_places(it.seq, sh);
  it.kvh = (int)((v - base) / per_head);
  it.start = base + it.kvh * per_head;
  it.rt = 0;
  it.n_units = item_units(it.seq, 0, sh);
  while (v >= item_end(it)) {
    it.start = item_end(it);
    it.n_units = item_units(it.seq, ++it.rt, sh);
  }
  return it;
}

// The item after `it`; only called when there is one.
__host__ __device__ inline void next_item(PagedItem& it, const PagedSeqs& s, const PagedShape& sh) {
  it.start = item_end(it);
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

// What block c (c < blocks) leaves for the joining kernel: where its range begins, and the item there.
struct PagedRecord {
  long long begin, start;
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
  long long total;   // all places
  int blocks;        // blocks with a range: min(grid, total)
  long long begin, end;  // this block's (empty if both cuts have moved to one item's start)
  PagedItem item;    // at `begin`
};

// Finds this block's part, by all THREADS threads (a multiple of 32, at most 1024).  Each thread sums the
// places of a run of sequences; the sums are scanned.  Sequences with bad metadata take none.
template <int THREADS>
__device__ inline PagedRange find_range(const PagedSeqs& s, const PagedShape& sh, DeviceErrors* errs) {
  __shared__ long long warp_sums[THREADS / 32];
  __shared__ long long found_base[2];
  __shared__ int found_seq[2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = ceil_div(s.batch, THREADS);
  const int b0 = min(tid * per, s.batch), b1 = min(b0 + per, s.batch);
  long long mine = 0;
  for (int b = b0; b < b1; ++b) {
    const SeqInfo q = seq_info(s, b);
    if (!q.ok && blockIdx.x == 0) report_error(errs, kErrBadIndex, b);
    mine += head_places(q, sh) * sh.kv_heads;
  }
  long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) warp_sums[warp] = incl;
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
  r.begin = r.end = 0;
  if ((int)blockIdx.x >= r.blocks) return r;  // the whole block
  const long long first = before + incl - mine;
  const bool last_block = (int)blockIdx.x + 1 == r.blocks;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if (k == 1 && last_block) continue;
    const long long v = raw_begin(blockIdx.x + k, total, r.blocks);
    long long at = first;
    if (v >= at && v < at + mine) {
      for (int b = b0; b < b1; ++b) {
        const long long n = b1 - b0 == 1 ? mine : head_places(seq_info(s, b), sh) * sh.kv_heads;
        if (v < at + n) {
          found_seq[k] = b;
          found_base[k] = at;
          break;
        }
        at += n;
      }
    }
  }
  __syncthreads();
  const long long v0 = raw_begin(blockIdx.x, total, r.blocks), v1 = raw_begin(blockIdx.x + 1, total, r.blocks);
  r.item = item_at(s, sh, found_seq[0], found_base[0], v0);
  r.begin = moved_cut(r.item, v0);
  if (last_block)
    r.end = total;
  else if (v1 < item_end(r.item))
    r.end = moved_cut(r.item, v1);
  else
    r.end = moved_cut(item_at(s, sh, found_seq[1], found_base[1], v1), v1);
  return r;
}

// What a joining block has to do: the parts of the item that block c of the attention kernel is the first to
// cut, `parts` of them (0: nothing), part i in workspace slot(i).  By whole warps.
struct PagedJoin {
  PagedRecord rec;
  int c, parts, first_slot;
  __device__ int slot(int i) const { return i == 0 ? first_slot : 2 * (c - 1 + i); }
};
__device__ inline PagedJoin find_join(const PagedWorkspace& ws, int c) {
  PagedJoin j;
  j.c = c;
  j.parts = 0;
  // all asked for at once: there for every block, written by those with a range
  const int blocks = (int)ws.total[1];
  j.rec = ws.records[c];
  const long long before = ws.records[c - 1].begin;
  if (c >= blocks || j.rec.begin == j.rec.start || before > j.rec.start) return j;  // no cut, or not the first
  const long long end = j.rec.start + kItemCost + j.rec.n_units;
  int last = c;
  for (int base = c + 1;; base += 32) {
    const int i = base + (int)(threadIdx.x & 31);
    const unsigned in = __ballot_sync(0xffffffffu, i < blocks && ws.records[min(i, blocks - 1)].begin < end);
    last += __popc(in);
    if (in != 0xffffffffu) break;
  }
  j.parts = last - c + 2;
  j.first_slot = 2 * (c - 1) + (before == j.rec.start ? 0 : 1);
  return j;
}

#endif

}  // namespace b200
