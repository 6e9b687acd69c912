// Attention of chunks of new tokens over a paged key/value cache, on the 5th-generation tensor cores.
//
// The heads that share a kv head are packed with the tokens: a tile's 128 rows are 128 / group consecutive
// tokens times the group's heads, so K and V are staged once for the whole group.  An item is two such tiles
// (A and B) of one sequence and kv head; units are 128 cached tokens; a block per SM streams an equal share of
// all units (paged_sched.cuh), so that one long sequence fills the device as well as many short ones.
//
// Warpgroups (the first hands registers to the others with setmaxnreg):
//   0: warp 0 loads Q (TMA: box of 64 columns x group heads x tokens) and, for bf16 pages, K and V (TMA: one box
//      per page and 64 columns); warp 1 issues the MMAs; warps 2 and 3 go through V of the units that not all rows
//      see whole.
//   1, 2: softmax of tile A and B, one thread per row, as in the training forward kernel: scores from tensor
//      memory, probabilities back into the same columns as the A operand of the PV product, lazy rescaling of O.
//   3 (8-bit pages only): loads Q, and expands codes into the shared-memory tiles; see below.
// With 8-bit pages the products are taken in fp16, whose 11 bits lose nothing next to the result's 8: a row of q is
// scaled by a power of two to a maximum in [1, 2), and code * scale of K and of V by one for each unit of 128
// tokens (to a maximum in (2^14, 2^15]); a token's factor and its product with a code are rounded there (2^-11
// relative each, for scales down to 2^-19 of the unit's largest).  K's power multiplies the unit's scores.  V's,
// 2^e, goes into the exponent: the weights are 2^(s_j + e - m), with the running maximum m taken over s_j + e and
// 2^6 of headroom, and the normaliser sums them times 2^-e.  Rounding code * scale to bf16 instead cost two bits of
// the result.
// That is for few tiles of a sequence.  With many (a long prompt), every tile would expand the same codes again:
// then one kernel expands all visible units once, to fp16 [sequence, unit, kv head, 128, head_dim] with their
// powers of two beside them, and Q's rows, and the attention kernel loads both by TMA (KV_EXPANDED).
// MMA order: S_A(0) S_B(0) | PV_A(j) S_A(j+1) PV_B(j) S_B(j+1) | ...
//
// Masking is by selection (a masked score becomes -inf whatever K holds).  A probability of 0 times an infinity or a
// NaN is NaN, so V must hold none where some row of an item does not see it.  V's rows behind the last visible token
// are zeroed in shared memory: what lies in a page behind a sequence's end has no influence.  Infinities and NaN ahead
// of it, in units that not all rows see whole, are zeroed too (bf16); a block that met some looks them up in the cache
// once more in its epilogue, and writes NaN into the columns that held them for the rows that see them (long chunk
// 574 -> 580 us, ragged prompts 47 -> 49 us).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "gemm.h"
#include "kernels.h"
#include "paged.h"
#include "paged_sched.cuh"

namespace b200 {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRescaleThreshold = 8.0f;  // log2 units
constexpr float kHeadroom = 6.0f;          // 8-bit: log2 of the largest weight (before lazy raises)
constexpr int kItemRows = 256;

// 8-bit pages that have been expanded to fp16 units.
constexpr int KV_EXPANDED = 3;
struct ExpandedUnits {
  __half* k;  // [batch, units, kv_heads, 128, head_dim]
  __half* v;
  float2* power;    // [batch, units, kv_heads]: 2^e of K, e of V
  __half* q;        // [total_q, heads, head_dim]
  float* q_power;   // [total_q, heads]
  int units;        // of a sequence (by the block table's width)
};

template <int FMT, int HD>
struct ChunkCfg {
  static constexpr bool EXPANDED = FMT == KV_EXPANDED;
  static constexpr bool QUANT = FMT == KV_E4M3 || FMT == KV_INT8;
  static constexpr bool F16 = EXPANDED || QUANT;
  static constexpr int THREADS = QUANT ? 512 : 384;
  static constexpr int LAUNCH_REGS = QUANT ? 128 : 168;
  static constexpr int KB = HD / 64;
  static constexpr int TILE_BYTES = 128 * HD * 2;
  static constexpr int STAGES = (HD == 64) ? 3 : 2;
  static constexpr int Q_BUFS = (HD == 64) ? 2 : 1;
  // bf16: a softmax thread keeps its row's 128 scores in registers, for which the first warpgroup hands over
  // some of its own.  8-bit expanded here: the fourth warpgroup leaves 128 registers per thread, and the scores are
  // read from tensor memory twice, 32 at a time (holding them spilled: 7.2 us a unit instead of 4.7 at head_dim 128).
  static constexpr int REGS_LOW = 88;
  static constexpr int REGS_HIGH = 208;
  static constexpr int REGS_NEEDED = QUANT ? 0 : 128 * REGS_LOW + 256 * REGS_HIGH;
  static_assert(REGS_NEEDED <= THREADS * LAUNCH_REGS, "register split over budget");
  // hd 64: row sums from the tensor cores, by a block of ones behind V (see the training forward kernel)
  static constexpr bool ONES = (HD == 64) && !F16;  // (8-bit: the sums are weighted for each unit)
  static constexpr int O_COLS = ONES ? HD + 16 : HD;
  static constexpr int STAGE_BYTES = (ONES ? 3 : 2) * TILE_BYTES;
  static constexpr int Q_OFF = 0;
  static constexpr int KV_OFF = Q_BUFS * 2 * TILE_BYTES;
  static constexpr int BAR_OFF = KV_OFF + STAGES * STAGE_BYTES;
  static constexpr int UNIT_OFF = BAR_OFF + 256;  // 8-bit: powers of two of Q's rows, K's and V's units
  static constexpr int SMEM_BYTES = UNIT_OFF + (QUANT ? Q_BUFS * 1024 + 128 : 0) + 1024;
  static_assert(SMEM_BYTES + 4096 <= 232448, "shared memory exceeds 227 KB");
  static constexpr int TMEM_COLS = 512;
  static constexpr int T_S = 0;
  static constexpr int T_O = 256;
  static_assert(T_O + 2 * O_COLS <= TMEM_COLS, "tensor memory");
};

// A role's walk over its block's items.  Kept in shared memory, one for each warp and advanced by its lane 0:
// in registers it would spill inside the hot loops of the softmax.
struct ChunkWalk {
  PagedItem it;
  long long end;   // of the block's range
  int j0, j1;      // units of the item in it
  int n_tiles;     // 1: the item has rows in tile A only
  int visible;     // cached tokens that its last row sees
  int all_see;     // and its first row (may be negative)
};
__device__ __forceinline__ void enter_item(ChunkWalk& w, const PagedShape& sh, int j0) {
  w.j0 = j0;
  w.j1 = unit_of_cut(w.it, w.end);
  w.n_tiles = w.it.seq.qn - w.it.rt * sh.tile_tokens > sh.tile_tokens / 2 ? 2 : 1;
  w.visible = item_visible(w.it.seq, w.it.rt, sh.tile_tokens);
  w.all_see = w.it.seq.len - w.it.seq.qn + w.it.rt * sh.tile_tokens + 1;
}
// The unit from which on some row of the item does not see all 128 tokens.
__device__ __forceinline__ int first_hidden_unit(const ChunkWalk& w) { return max(w.all_see, 0) >> 7; }
// By one thread.  False at the end of the range.
__device__ __forceinline__ bool next_part(ChunkWalk& w, const PagedSeqs& s, const PagedShape& sh) {
  if (w.end <= item_end(w.it)) return false;
  PagedItem it = w.it;
  next_item(it, s, sh);
  w.it = it;
  enter_item(w, sh, 0);
  return true;
}
// By a whole warp.
__device__ __forceinline__ bool next_part_warp(ChunkWalk& w, const PagedSeqs& s, const PagedShape& sh, int lane) {
  __syncwarp();
  bool more = false;
  if (lane == 0) more = next_part(w, s, sh);
  more = __shfl_sync(0xffffffffu, (int)more, 0) != 0;
  __syncwarp();
  return more;
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
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
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// 2^e, and the exponent e that brings max_code * scale into (2^14, 2^15] (the lowest one for a scale of 0).
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }
__device__ __forceinline__ int unit_exponent(uint32_t top, float max_code) {
  if (top == 0u) return kLowestExponent;
  const int e = (int)(__float_as_uint(__uint_as_float(top) * max_code) >> 23) - 127;  // floor(log2)
  return max(e - 14, kLowestExponent);  // (113 for the largest bf16 values)
}

// A token whose V has no finite scale is lost to the rows that see it, and has to be nothing to the others, although
// a probability of 0 times a NaN is NaN: its V becomes zeros and its K NaN, since masked scores are replaced.
__device__ __forceinline__ void settle_scales(float& k, float& v) {
  if (v - v != 0.f) {
    k = __int_as_float(0x7FC00000);
    v = 0.f;
  }
}
// What a scale counts as in its unit's maximum, which compares bits: infinities, NaN and -0 do not count.
__device__ __forceinline__ uint32_t scale_bits(float x) { return x > 0.f && x - x == 0.f ? __float_as_uint(x) : 0u; }

// 16 codes times a factor as 16 fp16.
template <int FMT>
__device__ __forceinline__ void expand16(const uint4& q, float factor, uint4 (&out)[2]) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
  uint32_t r[8];
  const __half2 f = __float2half2_rn(factor);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t p[2];  // the codes as fp16, exactly
    if constexpr (FMT == KV_E4M3) {
      asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t"
          "cvt.rn.f16x2.e4m3x2 %1, hi;\n\t}"
          : "=r"(p[0]), "=r"(p[1])
          : "r"(w[i]));
    } else {
      // code + 128 as the low bits of 1024; then 1152 is taken off
      const uint32_t b = w[i] ^ 0x80808080u, bias = 0x64806480u;
      p[0] = __byte_perm(b, 0x64646464u, 0x4140);
      p[1] = __byte_perm(b, 0x64646464u, 0x4342);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&p[h]), *reinterpret_cast<const __half2*>(&bias));
        p[h] = *reinterpret_cast<const uint32_t*>(&x);
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const __half2 x = __hmul2(*reinterpret_cast<const __half2*>(&p[h]), f);
      r[2 * i + h] = *reinterpret_cast<const uint32_t*>(&x);
    }
  }
  out[0] = make_uint4(r[0], r[1], r[2], r[3]);
  out[1] = make_uint4(r[4], r[5], r[6], r[7]);
}

// Waits for the tensor-memory loads in flight, and ties the registers of one of them to the wait: another
// load is issued right behind it, and nothing else keeps the uses of these from moving before the wait.
__device__ __forceinline__ void tmem_arrived(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                 "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}

// Scores from column `seen` on become -inf.
__device__ __forceinline__ void mask32(uint32_t (&s)[32], int seen) {
  if (seen < 32) {
#pragma unroll
    for (int e = 0; e < 32; ++e)
      if (e >= seen) s[e] = 0xFF800000u;
  }
}

// By two warps (`half` 0 and 1), each on its half of the 16-byte pieces: takes infinities and NaN out of the first
// `live` rows of a V tile (128 rows, 64 columns per 16 KB block); true if there were any.  x * 0 is NaN for those and
// for nothing else: one instruction for two values finds whether there are any, and most tiles have none.
template <int HD>
__device__ __forceinline__ bool take_out_non_finite(uint8_t* vs, int live, int half, int lane) {
  const int first = half * 32 + lane;
  uint32_t acc[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int kb = 0; kb < HD / 64; ++kb)
#pragma unroll 8
    for (int i = first; i < live * 8; i += 64) {
      const uint4 x = *reinterpret_cast<const uint4*>(vs + kb * 16384 + i * 16);
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(acc[e]) : "r"(w[e]), "r"(0u));
    }
  if (!__any_sync(0xffffffffu, ((acc[0] | acc[1] | acc[2] | acc[3]) & 0x7FFF7FFFu) != 0u)) return false;
  for (int kb = 0; kb < HD / 64; ++kb)
    for (int i = first; i < live * 8; i += 64) {
      uint16_t* piece = reinterpret_cast<uint16_t*>(vs + kb * 16384 + i * 16);
      for (int e = 0; e < 8; ++e)
        if ((piece[e] & 0x7F80) == 0x7F80) piece[e] = 0;
    }
  return true;
}
// By a row's thread, in the rare block that took some out: NaN into the columns in which the tokens t0 to t1 that the
// row sees hold one, behind what the thread has written there.  put(d) writes column d.
template <typename Put>
__device__ __forceinline__ void put_back_nan(const PagedAttnParams& p, int b, int kvh, int t0, int t1, const Put& put) {
  const int page_log2 = p.seqs.page_log2, hd = p.pool.head_dim;
  for (int t = t0; t < t1; ++t) {
    const int page = p.seqs.table[(long long)b * p.seqs.table_stride + (t >> page_log2)];
    if (page < 0 || page >= p.seqs.n_pages) continue;
    const long long cell = (((long long)page * p.pool.kv_heads + kvh) << page_log2) + (t & ((1 << page_log2) - 1));
    const uint16_t* v = reinterpret_cast<const uint16_t*>(p.pool.v) + cell * hd;
    for (int d = 0; d < hd; ++d)
      if ((v[d] & 0x7F80) == 0x7F80) put(d);
  }
}

template <int FMT, int HD>
__global__ void __launch_bounds__(ChunkCfg<FMT, HD>::THREADS, 1)
    paged_chunk_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                       const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ PagedAttnParams p,
                       PagedShape shape, PagedWorkspace ws, ExpandedUnits ex) {
  using C = ChunkCfg<FMT, HD>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align_smem_1024(smem_raw);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::BAR_OFF);
  uint64_t* q_full = bars;
  uint64_t* q_empty = q_full + C::Q_BUFS;
  uint64_t* kv_full = q_empty + C::Q_BUFS;
  uint64_t* kv_empty = kv_full + C::STAGES;
  uint64_t* s_full = kv_empty + C::STAGES;
  uint64_t* p_full = s_full + 2;
  uint64_t* o_done = p_full + 2;
  uint64_t* o_free = o_done + 2;
  // bf16, per stage, of units that some row does not see whole: V has arrived (v_raw), is fit for the product (v_clean)
  uint64_t* v_clean = o_free + 2;
  uint64_t* v_raw = v_clean + C::STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(v_raw + C::STAGES);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* taken_out = abort_flag + 1;  // bf16: some V of this block held an infinity or a NaN

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::Q_BUFS; ++i) {
      mbar_init(&q_full[i], C::QUANT ? 4 : 1);
      mbar_init(&q_empty[i], 1);
    }
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&kv_full[s], C::QUANT ? 4 : 1);
      mbar_init(&kv_empty[s], 1);
      mbar_init(&v_clean[s], 2);
      mbar_init(&v_raw[s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[t], 4);
      mbar_init(&o_done[t], 1);
      mbar_init(&o_free[t], 4);
    }
    *abort_flag = 0;
    *taken_out = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::TMEM_COLS);
    tmem_relinquish();
  }
  if constexpr (C::ONES) {
    for (int st = 0; st < C::STAGES; ++st) {
      uint4* ones = reinterpret_cast<uint4*>(smem + C::KV_OFF + st * C::STAGE_BYTES + 2 * C::TILE_BYTES);
      for (int i = threadIdx.x; i < C::TILE_BYTES / 16; i += C::THREADS)
        ones[i] = make_uint4(0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u);
    }
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait_and_release();

  const PagedRange range = find_range<C::THREADS>(p.seqs, shape, p.errs);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    ws.total[0] = range.total;
    ws.total[1] = range.blocks;
  }
  const bool busy = range.begin != range.end;
  __shared__ ChunkWalk walks[C::THREADS / 32];
  ChunkWalk& w = walks[warp];
  if (busy && lane == 0) {
    w.it = range.item;
    w.end = range.end;
    enter_item(w, shape, unit_of_cut(range.item, range.begin));
  }
  if ((int)blockIdx.x < range.blocks && threadIdx.x == 0)
    ws.records[blockIdx.x] = {range.begin, range.item.start, range.item.n_units, range.item.b, range.item.kvh,
                              range.item.rt};
  __syncwarp();
  const int tile_tokens = shape.tile_tokens / 2;  // of one tile
  const int page_log2 = p.seqs.page_log2;

  if (warp < 4) {
    if constexpr (!C::QUANT) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::REGS_LOW));
    if (!C::QUANT && busy && warp == 0 && lane == 0) {
      tma_prefetch_desc(&tm_q);
      int g = 0;
      bool ok = true;
      for (int k = 0; ok; ++k) {
        const int qs = k % C::Q_BUFS;
        if (k >= C::Q_BUFS &&
            !mbar_wait_bounded(&q_empty[qs], ((k / C::Q_BUFS) - 1) & 1, abort_flag, p.errs, kErrAttnWait, 10))
          break;
        uint8_t* qbase = smem + C::Q_OFF + qs * 2 * C::TILE_BYTES;
        mbar_expect_tx(&q_full[qs], w.n_tiles * C::KB * tile_tokens * p.group * 128);
        for (int t = 0; t < w.n_tiles; ++t)
#pragma unroll
          for (int kb = 0; kb < C::KB; ++kb)
            tma_load_3d(qbase + t * C::TILE_BYTES + kb * 16384, &tm_q, &q_full[qs], 64 * kb, w.it.kvh * p.group,
                        w.it.seq.q0 + w.it.rt * shape.tile_tokens + t * tile_tokens);
        {
          const int* table = p.seqs.table + (long long)w.it.b * p.seqs.table_stride;
          const int page_size = 1 << page_log2, kvh = w.it.kvh, visible = w.visible, j1 = w.j1;
          const int hidden = first_hidden_unit(w);
          for (int j = w.j0; j < j1; ++j, ++g) {
            const int st = g % C::STAGES;
            if (!mbar_wait_bounded(&kv_empty[st], ((g / C::STAGES) & 1) ^ 1u, abort_flag, p.errs, kErrAttnWait, 0)) {
              ok = false;
              break;
            }
            uint8_t* ks = smem + C::KV_OFF + st * C::STAGE_BYTES;
            uint8_t* vs = ks + C::TILE_BYTES;
            if constexpr (C::EXPANDED) {
              const int row = ((w.it.b * ex.units + j) * shape.kv_heads + kvh) * 128;
              mbar_expect_tx(&kv_full[st], 2 * C::TILE_BYTES);
#pragma unroll
              for (int kb = 0; kb < C::KB; ++kb) {
                tma_load_2d(ks + kb * 16384, &tm_k, &kv_full[st], 64 * kb, row);
                tma_load_2d(vs + kb * 16384, &tm_v, &kv_full[st], 64 * kb, row);
              }
              continue;
            }
            const int n_pages = min(128 >> page_log2, max(0, (visible - j * 128 + page_size - 1) >> page_log2));
            // a unit that is not seen whole gets V on a barrier of its own: warps 2 and 3 go through it first
            uint64_t* v_bar = j >= hidden ? &v_raw[st] : &kv_full[st];
            const int bytes = n_pages * page_size * HD * 2;
            mbar_expect_tx(&kv_full[st], j >= hidden ? bytes : 2 * bytes);
            if (j >= hidden) mbar_expect_tx(&v_raw[st], bytes);
            for (int i = 0; i < n_pages; ++i) {
              int page = table[((j * 128) >> page_log2) + i];
              if (page < 0 || page >= p.seqs.n_pages) {
                report_error(p.errs, kErrBadIndex, w.it.b);
                page = p.seqs.n_pages;  // behind the tensor: the copy fills zeros
              }
              const int row = (int)(min((long long)page * shape.kv_heads + kvh,
                                        (long long)p.seqs.n_pages * shape.kv_heads)
                                    << page_log2);
              const int at = i * page_size * 128;
#pragma unroll
              for (int kb = 0; kb < C::KB; ++kb) {
                tma_load_2d(ks + kb * 16384 + at, &tm_k, &kv_full[st], 64 * kb, row);
                tma_load_2d(vs + kb * 16384 + at, &tm_v, v_bar, 64 * kb, row);
              }
            }
          }
        }
        if (!ok || !next_part(w, p.seqs, shape)) break;
      }
    } else if (busy && warp == 1 && lane == 0) {
      constexpr uint32_t F16 = C::F16 ? (1u << 7) | (1u << 10) : 0u;  // A and B format: bf16 -> fp16
      constexpr uint32_t IDESC_S = idesc_bf16_f32(128, 128, false, false) ^ F16;
      constexpr uint32_t IDESC_O = idesc_bf16_f32(128, C::O_COLS, false, true) ^ F16;
      int g = 0;
      uint32_t clean_parity = 0;  // bit per stage
      int pn[2] = {0, 0}, on[2] = {0, 0};
      bool ok = true;
      for (int k = 0; ok; ++k) {
        const int qs = k % C::Q_BUFS;
        const uint32_t q_addr = smem_u32(smem + C::Q_OFF + qs * 2 * C::TILE_BYTES);
        if (!mbar_wait_bounded(&q_full[qs], (k / C::Q_BUFS) & 1, abort_flag, p.errs, kErrAttnWait, 2)) break;
        auto issue_s = [&](int t, int st) {
          const uint64_t dq = smem_desc_sw128(q_addr + t * C::TILE_BYTES, 16, 1024);
          const uint64_t dk = smem_desc_sw128(smem_u32(smem + C::KV_OFF + st * C::STAGE_BYTES), 16, 1024);
#pragma unroll
          for (int ks = 0; ks < HD / 16; ++ks) {
            const uint64_t off = ((ks >> 2) * 16384 + (ks & 3) * 32) >> 4;
            tc_mma_f16(tmem + C::T_S + t * 128, dq + off, dk + off, IDESC_S, ks > 0 ? 1u : 0u);
          }
          tc_commit(&s_full[t]);
        };
        const int j0 = w.j0, n = w.j1 - j0, n_tiles = w.n_tiles, hidden = first_hidden_unit(w);
        int st = g % C::STAGES;
        if (!mbar_wait_bounded(&kv_full[st], (g / C::STAGES) & 1, abort_flag, p.errs, kErrAttnWait, 1)) break;
        tc_fence_after();
        for (int t = 0; t < n_tiles; ++t) issue_s(t, st);
        for (int j = 0; ok && j < n; ++j) {
          st = (g + j) % C::STAGES;
          const int st1 = (g + j + 1) % C::STAGES;
          if constexpr (!C::F16) {
            if (j0 + j >= hidden) {
              if (!mbar_wait_bounded(&v_clean[st], (clean_parity >> st) & 1, abort_flag, p.errs, kErrAttnWait, 7)) {
                ok = false;
                break;
              }
              clean_parity ^= 1u << st;
            }
          }
          bool next_loaded = false;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (!ok || t >= n_tiles) break;
            if (!mbar_wait_bounded(&p_full[t], pn[t] & 1, abort_flag, p.errs, kErrAttnWait, 3 + t)) {
              ok = false;
              break;
            }
            ++pn[t];
            if (j == 0 && on[t] > 0 &&
                !mbar_wait_bounded(&o_free[t], (on[t] - 1) & 1, abort_flag, p.errs, kErrAttnWait, 5 + t)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint64_t dv =
                smem_desc_sw128(smem_u32(smem + C::KV_OFF + st * C::STAGE_BYTES + C::TILE_BYTES), 16384, 1024);
#pragma unroll
            for (int ks = 0; ks < 8; ++ks)
              tc_mma_f16_ts(tmem + C::T_O + t * C::O_COLS, tmem + C::T_S + t * 128 + ks * 8, dv + ks * (2048 >> 4),
                            IDESC_O, (j == 0 && ks == 0) ? 0u : 1u);
            if (j + 1 == n) {
              tc_commit(&o_done[t]);
              ++on[t];
            } else {
              if (!next_loaded) {
                if (!mbar_wait_bounded(&kv_full[st1], ((g + j + 1) / C::STAGES) & 1, abort_flag, p.errs, kErrAttnWait,
                                       1)) {
                  ok = false;
                  break;
                }
                next_loaded = true;
                tc_fence_after();
              }
              issue_s(t, st1);
            }
          }
          if (!ok) break;
          tc_commit(&kv_empty[st]);
        }
        g += n;
        tc_commit(&q_empty[qs]);
        if (!ok || !next_part(w, p.seqs, shape)) break;
      }
    } else if (!C::F16 && busy && warp >= 2) {
      const int half = warp - 2;
      int g = 0;
      uint32_t raw_parity = 0;  // bit per stage
      while (true) {
        bool ok = true;
        for (int j = max(w.j0, first_hidden_unit(w)); j < w.j1; ++j) {
          const int st = (g + j - w.j0) % C::STAGES;
          ok = mbar_wait_bounded(&v_raw[st], (raw_parity >> st) & 1, abort_flag, p.errs, kErrAttnWait, 8);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          raw_parity ^= 1u << st;
          uint8_t* vs = smem + C::KV_OFF + st * C::STAGE_BYTES + C::TILE_BYTES;
          const int live = min(max(w.visible - j * 128, 0), 128);
#pragma unroll
          for (int kb = 0; kb < C::KB; ++kb)
            for (int i = live * 8 + half * 32 + lane; i < 1024; i += 64)
              *reinterpret_cast<uint4*>(vs + kb * 16384 + i * 16) = make_uint4(0u, 0u, 0u, 0u);
          if (w.all_see < w.visible)  // (else all rows are of one token and see the same)
            if (take_out_non_finite<HD>(vs, live, half, lane) && lane == 0) *taken_out = 1;
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&v_clean[st]);
        }
        if (!ok) break;
        g += w.j1 - w.j0;
        if (!next_part_warp(w, p.seqs, shape, lane)) break;
      }
    }
  } else if (C::QUANT && warp >= 12) {
    if constexpr (C::QUANT) {
      // K and V of a tile in turn: the next one's codes are in flight while one is expanded, page ids are read
      // a tile ahead.
      const int tid = threadIdx.x - 384;
      constexpr int PER_ROW = HD / 16;        // pieces of 16 codes per token
      constexpr int PIECES = PER_ROW;         // per thread and tile: tokens tid / PER_ROW + i * 128 / PER_ROW
      const int piece = tid % PER_ROW, tok0 = tid / PER_ROW;
      // scales of the unit's tokens and their maxima per warp, double-buffered: one barrier of the warpgroup a unit
      __shared__ float scales[2][2][128];
      __shared__ uint2 maxima[2][4];
      int cell[PIECES], next_page[PIECES];    // cell: (page, head, offset) index, -1 if nothing is visible there
      uint4 q[2][PIECES];
      int next_scale_page;
      float k_scale, v_scale;                 // of token tid
      int j = busy ? w.j0 : 0;
      auto read_pages = [&]() {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
          const int t = j * 128 + tok0 + i * (128 / PER_ROW);
          next_page[i] = t < w.visible ? p.seqs.table[(long long)w.it.b * p.seqs.table_stride + (t >> page_log2)] : -1;
        }
        const int t = j * 128 + tid;
        next_scale_page = t < w.visible ? p.seqs.table[(long long)w.it.b * p.seqs.table_stride + (t >> page_log2)] : -1;
      };
      auto resolve = [&]() {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
          const int t = j * 128 + tok0 + i * (128 / PER_ROW);
          const int page = next_page[i];
          cell[i] = -1;
          if (page >= 0 && page < p.seqs.n_pages)
            cell[i] = ((page * shape.kv_heads + w.it.kvh) << page_log2) + (t & ((1 << page_log2) - 1));
          else if (t < w.visible)
            report_error(p.errs, kErrBadIndex, w.it.b);
        }
      };
      auto load_codes = [&](int v) {
        const uint8_t* src = reinterpret_cast<const uint8_t*>(v ? p.pool.v : p.pool.k) + piece * 16;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
          q[v][i] = make_uint4(0u, 0u, 0u, 0u);
          if (cell[i] >= 0 && B200_IN_BOUNDS(p.errs, cell[i], 1, pool_cells(p.seqs, shape.kv_heads), 141))
            q[v][i] = *reinterpret_cast<const uint4*>(src + (long long)cell[i] * HD);
        }
      };
      auto load_scales = [&]() {
        k_scale = v_scale = 0.f;
        if (next_scale_page >= 0 && next_scale_page < p.seqs.n_pages) {
          const int c = ((next_scale_page * shape.kv_heads + w.it.kvh) << page_log2) +
                        ((j * 128 + tid) & ((1 << page_log2) - 1));
          if (B200_IN_BOUNDS(p.errs, c, 1, pool_cells(p.seqs, shape.kv_heads), 142)) {
            k_scale = p.pool.k_scale[c];
            v_scale = p.pool.v_scale[c];
          }
          settle_scales(k_scale, v_scale);
        }
      };
      // Q: a thread takes a row of each tile
      auto load_q = [&](int k) {
        const int qs = k % C::Q_BUFS;
        const bool free = k < C::Q_BUFS || mbar_wait_bounded(&q_empty[qs], ((k / C::Q_BUFS) - 1) & 1, abort_flag,
                                                             p.errs, kErrAttnWait, 10);
        if (!__all_sync(0xffffffffu, free)) return false;
        const int tok_in_tile = tid / p.group, head = tid % p.group;
        for (int t = 0; t < w.n_tiles; ++t) {
          const int tok = w.it.rt * shape.tile_tokens + t * tile_tokens + tok_in_tile;
          const bool live = tok_in_tile < tile_tokens && tok < w.it.seq.qn &&
                            B200_IN_BOUNDS(p.errs, w.it.seq.q0 + tok, 1, p.seqs.total_q, 140);
          const __nv_bfloat16* src = p.q + (long long)(w.it.seq.q0 + tok) * p.q_stride_t +
                                     (long long)(w.it.kvh * p.group + head) * p.q_stride_h;
          uint4 x[HD / 8];
          uint32_t top = 0u;
#pragma unroll
          for (int i = 0; i < HD / 8; ++i) {
            x[i] = live ? *reinterpret_cast<const uint4*>(src + 8 * i) : make_uint4(0u, 0u, 0u, 0u);
            top = __vmaxu2(top, __vmaxu2(__vmaxu2(x[i].x & 0x7FFF7FFFu, x[i].y & 0x7FFF7FFFu),
                                         __vmaxu2(x[i].z & 0x7FFF7FFFu, x[i].w & 0x7FFF7FFFu)));
          }
          const int e = q_row_exponent(max(top & 0xFFFFu, top >> 16));
          const float down = __uint_as_float((uint32_t)(254 - e) << 23);
          reinterpret_cast<float*>(smem + C::UNIT_OFF)[(qs * 2 + t) * 128 + tid] = __uint_as_float((uint32_t)e << 23);
          uint8_t* row = smem + C::Q_OFF + qs * 2 * C::TILE_BYTES + t * C::TILE_BYTES + tid * 128;
#pragma unroll
          for (int i = 0; i < HD / 8; ++i) {
            uint4 y;
            y.x = pack_f16(bf16lo(x[i].x) * down, bf16hi(x[i].x) * down);
            y.y = pack_f16(bf16lo(x[i].y) * down, bf16hi(x[i].y) * down);
            y.z = pack_f16(bf16lo(x[i].z) * down, bf16hi(x[i].z) * down);
            y.w = pack_f16(bf16lo(x[i].w) * down, bf16hi(x[i].w) * down);
            *reinterpret_cast<uint4*>(row + (i >> 3) * 16384 + (((i ^ tid) & 7) << 4)) = y;
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full[qs]);
        return true;
      };
      // Once a wait has run out, `ok` stays false: nothing more is waited for or handed over, but the warps go
      // through the rest of the range together, since they meet at a barrier for every unit.
      bool ok = busy;
      int k = 0;
      if (busy) {
        read_pages();
        ok = load_q(0);
        resolve();
        load_codes(0);
        load_scales();
      }
      bool more = busy;
      for (int g = 0; more; ++g) {
        const int st = g % C::STAGES;
        bool new_item = false;
        // the unit's powers of two
        scales[g & 1][0][tid] = k_scale;
        scales[g & 1][1][tid] = v_scale;
        uint32_t km = __reduce_max_sync(0xffffffffu, scale_bits(k_scale));
        uint32_t vm = __reduce_max_sync(0xffffffffu, scale_bits(v_scale));
        if (lane == 0) maxima[g & 1][warp & 3] = make_uint2(km, vm);
        named_bar(1, 128);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          km = max(km, maxima[g & 1][i].x);
          vm = max(vm, maxima[g & 1][i].y);
        }
        const int ke = unit_exponent(km, kv_code_max(FMT)), ve = unit_exponent(vm, kv_code_max(FMT));
        const float kf = pow2i(-ke), vf = pow2i(-ve);
        if (++j == w.j1) {
          more = new_item = next_part_warp(w, p.seqs, shape, lane);
          j = 0;
        }
        if (more) read_pages();
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          if (v == 0) {
            load_codes(1);
            ok = ok && mbar_wait_bounded(&kv_empty[st], ((g / C::STAGES) & 1) ^ 1u, abort_flag, p.errs, kErrAttnWait, 0);
            ok = __all_sync(0xffffffffu, ok);
            if (tid == 0 && ok)
              reinterpret_cast<float2*>(smem + C::UNIT_OFF + C::Q_BUFS * 1024)[st] = make_float2(pow2i(ke), (float)ve);
          } else if (more) {
            resolve();
            load_codes(0);
            load_scales();
          }
          uint8_t* dst = smem + C::KV_OFF + st * C::STAGE_BYTES + v * C::TILE_BYTES + (piece >> 2) * 16384;
          if (ok) {
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
              const int tok = tok0 + i * (128 / PER_ROW);
              uint4 x[2];
              expand16<FMT>(q[v][i], scales[g & 1][v][tok] * (v ? vf : kf), x);
#pragma unroll
              for (int h = 0; h < 2; ++h)
                *reinterpret_cast<uint4*>(dst + tok * 128 + ((((piece & 3) * 2 + h) ^ (tok & 7)) << 4)) = x[h];
            }
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (ok && lane == 0) mbar_arrive(&kv_full[st]);
        if (new_item) ok = ok && load_q(++k);
      }
    }
  } else {
    if constexpr (!C::QUANT) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::REGS_HIGH));
    const int t = (warp - 4) >> 2;
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const uint32_t s_cols = tmem + lane_off + C::T_S + t * 128;
    const uint32_t o_cols = tmem + lane_off + C::T_O + t * C::O_COLS;
    const float scale2 = p.scale * kLog2e;
    const int tok_in_tile = r / p.group, head = r % p.group;
    int sn = 0, on = 0, g = 0;
    for (int part_no = 0; busy; ++part_no) {
      const int j0 = w.j0, j1 = w.j1;
      if (t < w.n_tiles) {
        const int tok = w.it.rt * shape.tile_tokens + t * tile_tokens + tok_in_tile;
        const bool live = tok_in_tile < tile_tokens && tok < w.it.seq.qn &&
                          B200_IN_BOUNDS(p.errs, w.it.seq.q0 + tok, 1, p.seqs.total_q, 143);
        const int lim = live ? w.it.seq.len - w.it.seq.qn + tok + 1 : 0;  // tokens that this row sees
        float m_used = -INFINITY, l = 0.f;
        float q_power = 1.f;
        float2 power = make_float2(1.f, 0.f);
        const float2* powers = nullptr;
        if constexpr (C::EXPANDED) {
          powers = ex.power + (long long)w.it.b * ex.units * shape.kv_heads + w.it.kvh;
          power = powers[(long long)j0 * shape.kv_heads];
          if (live) q_power = ex.q_power[(long long)(w.it.seq.q0 + tok) * p.heads + w.it.kvh * p.group + head];
        }
        bool ok = true;
        for (int j = j0; j < j1; ++j) {
          if (!mbar_wait_bounded(&s_full[t], sn & 1, abort_flag, p.errs, kErrAttnWait, 11 + t)) {
            ok = false;
            break;
          }
          ++sn;
          tc_fence_after();
          const int seen = lim - j * 128;
          // scores to log2 units; 8-bit: plus V's exponent
          float to_log2 = scale2, v_exp = 0.f;
          if constexpr (C::EXPANDED) {
            to_log2 = score_factor(scale2, q_power, power.x);
            v_exp = power.y;
            if (j + 1 < j1) power = powers[(long long)(j + 1) * shape.kv_heads];  // for the next unit
          }
          if constexpr (C::QUANT) {
            const float* units = reinterpret_cast<const float*>(smem + C::UNIT_OFF);
            const float2 u = reinterpret_cast<const float2*>(units + C::Q_BUFS * 256)[(g + j - j0) % C::STAGES];
            to_log2 = score_factor(scale2, units[((part_no % C::Q_BUFS) * 2 + t) * 128 + r], u.x);
            v_exp = u.y;
          }
          uint32_t s[C::QUANT ? 2 : 4][32];  // 8-bit: two buffers of 32 scores, else the row's 128
          float mx8[8];
          if constexpr (C::QUANT) {
#pragma unroll
            for (int e = 0; e < 8; ++e) mx8[e] = -INFINITY;
            tmem_ld_32x32b_x32(s_cols, s[0]);
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4) {
              tmem_arrived(s[q4 & 1]);
              if (q4 < 3) tmem_ld_32x32b_x32(s_cols + 32 * (q4 + 1), s[(q4 + 1) & 1]);
              mask32(s[q4 & 1], seen - 32 * q4);
#pragma unroll
              for (int e = 0; e < 32; e += 2)
                mx8[(e >> 1) & 7] = fmax3f(mx8[(e >> 1) & 7], __uint_as_float(s[q4 & 1][e]),
                                           __uint_as_float(s[q4 & 1][e + 1]));
            }
          } else {
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4) tmem_ld_32x32b_x32(s_cols + 32 * q4, s[q4]);
            tc_wait_ld();
            if (seen < 128) {
#pragma unroll
              for (int q4 = 0; q4 < 4; ++q4) mask32(s[q4], seen - 32 * q4);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) mx8[e] = __uint_as_float(s[0][e]);
#pragma unroll
            for (int e = 8; e < 128; e += 2)
              mx8[(e >> 1) & 7] = fmax3f(mx8[(e >> 1) & 7], __uint_as_float(s[e >> 5][e & 31]),
                                         __uint_as_float(s[e >> 5][(e + 1) & 31]));
          }
          const float mx = fmax3f(fmax3f(mx8[0], mx8[1], mx8[2]), fmax3f(mx8[3], mx8[4], mx8[5]), fmaxf(mx8[6], mx8[7]));
          const float m_row = C::F16 ? fmaf(mx, to_log2, v_exp) : mx * scale2;
          if (j == j0) {
            m_used = m_row;
          } else if (__any_sync(0xffffffffu, m_row > m_used + kRescaleThreshold)) {
            // taken by the whole warp: tcgen05.ld / st are warp-collective
            const float m_new = (m_row > m_used + kRescaleThreshold) ? m_row : m_used;
            const float alpha = m_new == m_used ? 1.f : ex2_approx(m_used - m_new);
            l *= alpha;
#pragma unroll
            for (int cc = 0; cc < HD; cc += 32) {
              uint32_t ov[32];
              tmem_ld_32x32b_x32(o_cols + cc, ov);
              tc_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * alpha);
              tmem_st_32x32b_x32(o_cols + cc, ov);
            }
            if constexpr (C::ONES) {
              uint32_t lv[16];
              tmem_ld_32x32b_x16(o_cols + HD, lv);
              tc_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) lv[e] = __float_as_uint(__uint_as_float(lv[e]) * alpha);
              tmem_st_32x32b_x16(o_cols + HD, lv);
            }
            m_used = m_new;
          }
          // nothing seen yet: all probabilities 0
          const float m_sub = m_used == -INFINITY ? 0.f : m_used - (C::F16 ? kHeadroom + v_exp : 0.f);
          uint64_t sums[4] = {0ull, 0ull, 0ull, 0ull};  // pairs of fp32 zeros
          const uint64_t scale_pair = pair(to_log2, to_log2), m_pair = pair(-m_sub, -m_sub);
          // the probabilities of two columns, in their sums and packed for the product with V
          auto weigh = [&](uint32_t s0, uint32_t s1, int e) {
            float p0, p1;
            unpair(fma2(pair(__uint_as_float(s0), __uint_as_float(s1)), scale_pair, m_pair), p0, p1);
            p0 = ex2_approx(p0);
            p1 = ex2_approx(p1);
            if constexpr (!C::ONES) sums[(e >> 1) & 3] = add2(sums[(e >> 1) & 3], pair(p0, p1));
            return C::F16 ? pack_f16(p0, p1) : pack_bf16(p0, p1);
          };
          if constexpr (C::QUANT) {
            tmem_ld_32x32b_x32(s_cols, s[0]);
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4) {
              tmem_arrived(s[q4 & 1]);
              if (q4 < 3) tmem_ld_32x32b_x32(s_cols + 32 * (q4 + 1), s[(q4 + 1) & 1]);
              uint32_t pr[16];
              mask32(s[q4 & 1], seen - 32 * q4);
#pragma unroll
              for (int e = 0; e < 32; e += 2) pr[e >> 1] = weigh(s[q4 & 1][e], s[q4 & 1][e + 1], e);
              tmem_st_32x32b_x16(s_cols + 16 * q4, pr);  // over scores that have been read
            }
          } else {
#pragma unroll
            for (int e = 0; e < 128; e += 2)
              s[e >> 6][(e >> 1) & 31] = weigh(s[e >> 5][e & 31], s[e >> 5][(e + 1) & 31], e);
            tmem_st_32x32b_x32(s_cols + 0, s[0]);
            tmem_st_32x32b_x32(s_cols + 32, s[1]);
          }
          if constexpr (!C::ONES) {
            float lo, hi;
            unpair(add2(add2(sums[0], sums[1]), add2(sums[2], sums[3])), lo, hi);
            l += C::F16 ? (lo + hi) * ex2_approx(-v_exp) : lo + hi;
          }
          tc_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[t]);
        }
        if (!ok) break;
        if (!mbar_wait_bounded(&o_done[t], on & 1, abort_flag, p.errs, kErrAttnWait, 13 + t)) break;
        ++on;
        tc_fence_after();
        if constexpr (C::ONES) {
          uint32_t lv[16];
          tmem_ld_32x32b_x16(o_cols + HD, lv);
          tc_wait_ld();
          l = __uint_as_float(lv[0]);
        }
        const float inv_l = l == 0.f ? 0.f : 1.0f / l;
        __nv_bfloat16* dst = p.out + (long long)(w.it.seq.q0 + tok) * p.o_stride_t +
                             (long long)(w.it.kvh * p.group + head) * p.o_stride_h;
        // parts go to the workspace as [slot][column / 4][row]: a warp writes 512 contiguous bytes
        const int slot = 2 * blockIdx.x + (part_no == 0 ? 0 : 1);
        const bool whole = j1 - j0 == w.it.n_units;
        const int row = t * 128 + r;
        float4* part = reinterpret_cast<float4*>(ws.o) + (size_t)slot * (HD / 4) * kItemRows + row;
#pragma unroll
        for (int cc = 0; cc < HD; cc += 32) {
          uint32_t ov[32];
          tmem_ld_32x32b_x32(o_cols + cc, ov);
          tc_wait_ld();
          if (cc + 32 >= HD) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&o_free[t]);
          }
          if (whole) {
#pragma unroll
            for (int e = 0; e < 32; e += 8) {
              uint4 x;
              x.x = pack_bf16(__uint_as_float(ov[e]) * inv_l, __uint_as_float(ov[e + 1]) * inv_l);
              x.y = pack_bf16(__uint_as_float(ov[e + 2]) * inv_l, __uint_as_float(ov[e + 3]) * inv_l);
              x.z = pack_bf16(__uint_as_float(ov[e + 4]) * inv_l, __uint_as_float(ov[e + 5]) * inv_l);
              x.w = pack_bf16(__uint_as_float(ov[e + 6]) * inv_l, __uint_as_float(ov[e + 7]) * inv_l);
              if (live) *reinterpret_cast<uint4*>(dst + cc + e) = x;
            }
          } else if (live) {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              part[(size_t)((cc + e) / 4) * kItemRows] =
                  make_float4(__uint_as_float(ov[e]), __uint_as_float(ov[e + 1]), __uint_as_float(ov[e + 2]),
                              __uint_as_float(ov[e + 3]));
          }
        }
        if (!whole && live) ws.ml[(size_t)slot * kItemRows + row] = make_float2(m_used, l);
        if constexpr (!C::F16) {
          if (*taken_out != 0 && live && w.all_see < w.visible)
            put_back_nan(p, w.it.b, w.it.kvh, max(j0, first_hidden_unit(w)) * 128, min(lim, j1 * 128), [&](int d) {
              if (whole)
                reinterpret_cast<uint16_t*>(dst)[d] = 0x7FC0;
              else
                reinterpret_cast<float*>(part + (size_t)(d / 4) * kItemRows)[d % 4] = __int_as_float(0x7FC00000);
            });
        }
      }
      g += j1 - j0;
      if (!next_part_warp(w, p.seqs, shape, lane)) break;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::TMEM_COLS);
  }
}

// Joins the parts of items that lie in more than one block's range (see paged_join_kernel): a thread per
// row, 16 columns per block in y.
template <int HD>
__global__ void __launch_bounds__(kItemRows)
    paged_chunk_join_kernel(const __grid_constant__ PagedAttnParams p, PagedShape shape, PagedWorkspace ws) {
  pdl_wait_and_release();
  const PagedJoin join = find_join(ws, blockIdx.x + 1);
  if (join.parts == 0) return;
  const PagedRecord& rec = join.rec;
  const int parts = join.parts;
  const SeqInfo seq = seq_info(p.seqs, rec.b);
  const int tile_tokens = shape.tile_tokens / 2;
  const int row = threadIdx.x;
  const int tok_in_tile = (row & 127) / p.group, head = (row & 127) % p.group;
  const int tok = rec.rt * shape.tile_tokens + (row >> 7) * tile_tokens + tok_in_tile;
  if (tok_in_tile >= tile_tokens || tok >= seq.qn) return;
  if (!B200_IN_BOUNDS(p.errs, seq.q0 + tok, 1, p.seqs.total_q, 144)) return;
  float mx = -INFINITY;
  for (int i = 0; i < parts; ++i) {
    const int slot = join.slot(i);
    mx = fmaxf(mx, ws.ml[(size_t)slot * kItemRows + row].x);
  }
  float4 acc[4];
#pragma unroll
  for (int d = 0; d < 4; ++d) acc[d] = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f;
  for (int i = 0; i < parts; ++i) {
    const int slot = join.slot(i);
    const float2 q = ws.ml[(size_t)slot * kItemRows + row];
    const float f = q.x == mx ? 1.f : ex2_approx(q.x - mx);
    l += q.y * f;
    const float4* src = reinterpret_cast<const float4*>(ws.o) + ((size_t)slot * (HD / 4) + blockIdx.y * 4) * kItemRows + row;
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      const float4 v = src[d * kItemRows];
      acc[d].x += v.x * f;
      acc[d].y += v.y * f;
      acc[d].z += v.z * f;
      acc[d].w += v.w * f;
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  __nv_bfloat16* dst = p.out + (long long)(seq.q0 + tok) * p.o_stride_t +
                       (long long)(rec.kvh * p.group + head) * p.o_stride_h + blockIdx.y * 16;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint4 x;
    x.x = pack_bf16(acc[2 * h].x * inv, acc[2 * h].y * inv);
    x.y = pack_bf16(acc[2 * h].z * inv, acc[2 * h].w * inv);
    x.z = pack_bf16(acc[2 * h + 1].x * inv, acc[2 * h + 1].y * inv);
    x.w = pack_bf16(acc[2 * h + 1].z * inv, acc[2 * h + 1].w * inv);
    *reinterpret_cast<uint4*>(dst + 8 * h) = x;
  }
}

// Blocks below `unit_blocks` expand one unit of one kv head each, the others a run of Q's rows.  Reads each
// code once and writes it as fp16; bound by memory.
template <int FMT, int HD>
__global__ void __launch_bounds__(128) paged_expand_kernel(PagedAttnParams p, ExpandedUnits ex, int unit_blocks) {
  pdl_wait_and_release();
  constexpr int LANES = HD / 8;  // per row of Q
  const int tid = threadIdx.x, lane = tid & 31;
  if ((int)blockIdx.x >= unit_blocks) {
    const long long row = (long long)((int)blockIdx.x - unit_blocks) * (128 / LANES) + tid / LANES;
    const int sub = tid % LANES;
    if (row >= (long long)p.seqs.total_q * p.heads) return;  // whole groups of LANES lanes
    const __nv_bfloat16* src = p.q + row / p.heads * p.q_stride_t + row % p.heads * p.q_stride_h + sub * 8;
    const uint4 x = *reinterpret_cast<const uint4*>(src);
    const uint32_t top = __vmaxu2(__vmaxu2(x.x & 0x7FFF7FFFu, x.y & 0x7FFF7FFFu),
                                  __vmaxu2(x.z & 0x7FFF7FFFu, x.w & 0x7FFF7FFFu));
    uint32_t m = max(top & 0xFFFFu, top >> 16);
    const uint32_t group = LANES == 32 ? 0xFFFFFFFFu : ((1u << LANES) - 1u) << (lane / LANES * LANES);
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(group, m, o));
    const int e = q_row_exponent(m);
    const float down = __uint_as_float((uint32_t)(254 - e) << 23);
    uint4 y;
    y.x = pack_f16(bf16lo(x.x) * down, bf16hi(x.x) * down);
    y.y = pack_f16(bf16lo(x.y) * down, bf16hi(x.y) * down);
    y.z = pack_f16(bf16lo(x.z) * down, bf16hi(x.z) * down);
    y.w = pack_f16(bf16lo(x.w) * down, bf16hi(x.w) * down);
    *reinterpret_cast<uint4*>(ex.q + row * HD + sub * 8) = y;
    if (sub == 0) ex.q_power[row] = __uint_as_float((uint32_t)e << 23);
    return;
  }
  const int kvh = (int)blockIdx.x % p.pool.kv_heads, u = (int)blockIdx.x / p.pool.kv_heads;
  const int b = u / ex.units, j = u % ex.units;
  const SeqInfo seq = seq_info(p.seqs, b);
  if (seq.qn == 0 || j * 128 >= max(seq.len, 1)) return;  // (an empty sequence still has one unit, of zeros)
  __shared__ float scales[2][128];
  __shared__ int cells[128];
  __shared__ uint2 maxima[4];
  int cell = -1;
  const int t = j * 128 + tid;
  if (t < seq.len) {
    const int page = p.seqs.table[(long long)b * p.seqs.table_stride + (t >> p.seqs.page_log2)];
    if (page >= 0 && page < p.seqs.n_pages)
      cell = ((page * p.pool.kv_heads + kvh) << p.seqs.page_log2) + (t & ((1 << p.seqs.page_log2) - 1));
    else
      report_error(p.errs, kErrBadIndex, b);
    if (cell >= 0 && !B200_IN_BOUNDS(p.errs, cell, 1, pool_cells(p.seqs, p.pool.kv_heads), 145)) cell = -1;
  }
  float ks = cell >= 0 ? p.pool.k_scale[cell] : 0.f, vs = cell >= 0 ? p.pool.v_scale[cell] : 0.f;
  settle_scales(ks, vs);
  cells[tid] = cell;
  scales[0][tid] = ks;
  scales[1][tid] = vs;
  uint32_t km = __reduce_max_sync(0xffffffffu, scale_bits(ks));
  uint32_t vm = __reduce_max_sync(0xffffffffu, scale_bits(vs));
  if (lane == 0) maxima[tid >> 5] = make_uint2(km, vm);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    km = max(km, maxima[i].x);
    vm = max(vm, maxima[i].y);
  }
  const int ke = unit_exponent(km, kv_code_max(FMT)), ve = unit_exponent(vm, kv_code_max(FMT));
  const float kf = pow2i(-ke), vf = pow2i(-ve);
  if (tid == 0) ex.power[blockIdx.x] = make_float2(pow2i(ke), (float)ve);
  constexpr int PER_ROW = HD / 16;
  const int piece = tid % PER_ROW;
#pragma unroll
  for (int i = 0; i < PER_ROW; ++i) {
    const int tok = tid / PER_ROW + i * (128 / PER_ROW);
    const int c = cells[tok];
    uint4 q[2] = {make_uint4(0u, 0u, 0u, 0u), make_uint4(0u, 0u, 0u, 0u)};
    if (c >= 0) {
      q[0] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(p.pool.k) + (long long)c * HD + piece * 16);
      q[1] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(p.pool.v) + (long long)c * HD + piece * 16);
    }
    const size_t at = ((size_t)blockIdx.x * 128 + tok) * HD + piece * 16;
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      uint4 x[2];
      // nothing there: zeros, and not the NaN that 0 * a NaN code would give
      expand16<FMT>(q[v], scales[v][tok] * (v ? vf : kf), x);
      uint4* dst = reinterpret_cast<uint4*>((v ? ex.v : ex.k) + at);
      dst[0] = x[0];
      dst[1] = x[1];
    }
  }
}

template <int FMT, int HD>
void launch_attention(const PagedAttnParams& p, const CUtensorMap& tm_q, const CUtensorMap& tm_k,
                      const CUtensorMap& tm_v, const PagedShape& shape, const PagedWorkspace& ws,
                      const ExpandedUnits& ex, cudaStream_t s) {
  using C = ChunkCfg<FMT, HD>;
  auto* kernel = paged_chunk_kernel<FMT, HD>;
  static std::atomic<unsigned long long> configured{0};
  once_per_device(configured, [&] {
    cudaFuncAttributes attr;
    B200_CUDA_CHECK(cudaFuncGetAttributes(&attr, kernel));
    // the register split draws on what the launch gives: with fewer, setmaxnreg would wait for ever
    B200_CHECK(attr.numRegs * C::THREADS >= C::REGS_NEEDED, "paged attention: built with too few registers");
    B200_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM_BYTES));
  });
  const int blocks = num_sms_cached();
  launch_k(kernel, dim3(blocks), dim3(C::THREADS), C::SMEM_BYTES, s, 1, tm_q, tm_k, tm_v, p, shape, ws, ex);
  launch_k(paged_chunk_join_kernel<HD>, dim3(blocks - 1, HD / 16), dim3(kItemRows), 0, s, 1, p, shape, ws);
  B200_CUDA_CHECK(cudaGetLastError());
  count_launch(2);
}

// Expanding once pays when rows per kv head and sequence x head_dim reach this (8 int8 caches of 8192 tokens with
// 8 kv heads, expanded in each tile against once: head_dim 64, 256 rows 73 / 79 us, 512 rows 125 / 117;
// head_dim 128, 128 rows 104 / 110, 256 rows 151 / 126, 512 rows 250 / 177; 8192 rows over one e4m3 cache of 16384
// tokens 987 / 560), as long as the units by the block table's width fit this much scratch memory and the allocator
// has it.
constexpr long long kExpandRowColumns = 32768;
constexpr size_t kExpandBytes = 512u << 20;

template <int FMT, int HD>
void launch_chunk(const PagedAttnParams& p, const PagedAlloc& alloc, cudaStream_t s) {
  const int blocks = num_sms_cached();
  const int tile_tokens = 128 / p.group;
  const PagedShape shape{2 * tile_tokens, 7, p.pool.kv_heads};
  const size_t ws_bytes = (paged_workspace_bytes(blocks, kItemRows, HD) + 255) / 256 * 256;
  auto q_map = [&](const void* q, long long stride_h, long long stride_t) {
    return make_tmap_bf16_3d(q, HD, p.heads, p.seqs.total_q, stride_h, stride_t, 64, p.group, tile_tokens);
  };
  ExpandedUnits ex{};
  if constexpr (FMT == KV_BF16) {
    const PagedWorkspace ws = paged_workspace(alloc(ws_bytes, false), blocks, kItemRows);
    const uint64_t rows = (uint64_t)p.seqs.n_pages * p.pool.kv_heads << p.seqs.page_log2;
    launch_attention<FMT, HD>(p, q_map(p.q, p.q_stride_h, p.q_stride_t),
                              make_tmap_bf16_2d(p.pool.k, HD, rows, HD, 64, 1u << p.seqs.page_log2),
                              make_tmap_bf16_2d(p.pool.v, HD, rows, HD, 64, 1u << p.seqs.page_log2), shape, ws, ex, s);
  } else {
    ex.units = (int)((((long long)p.seqs.max_pages << p.seqs.page_log2) + 127) / 128);
    const long long unit_blocks = (long long)p.seqs.batch * ex.units * p.pool.kv_heads;
    const size_t kv_bytes = (size_t)unit_blocks * 128 * HD * 2;
    const long long q_rows = (long long)p.seqs.total_q * p.heads;
    const size_t q_bytes = (size_t)q_rows * HD * 2;
    const size_t power_bytes = ((size_t)unit_blocks * 8 + 255) / 256 * 256;
    uint8_t* base = nullptr;
    if ((long long)p.seqs.max_q * p.group * HD >= kExpandRowColumns && unit_blocks > 0 && 2 * kv_bytes <= kExpandBytes)
      base = reinterpret_cast<uint8_t*>(
          alloc(ws_bytes + 2 * kv_bytes + power_bytes + (q_bytes + 255) / 256 * 256 + (size_t)q_rows * 4, true));
    if (base != nullptr) {
      const PagedWorkspace ws = paged_workspace(base, blocks, kItemRows);
      ex.k = reinterpret_cast<__half*>(base + ws_bytes);
      ex.v = ex.k + kv_bytes / 2;
      ex.power = reinterpret_cast<float2*>(base + ws_bytes + 2 * kv_bytes);
      ex.q = reinterpret_cast<__half*>(base + ws_bytes + 2 * kv_bytes + power_bytes);
      ex.q_power = reinterpret_cast<float*>(base + ws_bytes + 2 * kv_bytes + power_bytes + (q_bytes + 255) / 256 * 256);
      const long long q_blocks = (q_rows + 128 / (HD / 8) - 1) / (128 / (HD / 8));
      launch_k(paged_expand_kernel<FMT, HD>, dim3((unsigned)(unit_blocks + q_blocks)), dim3(128), 0, s, 1, p, ex,
               (int)unit_blocks);
      count_launch(1);
      const uint64_t rows = (uint64_t)unit_blocks * 128;
      // (fp16 moves like bf16: the maps only copy)
      launch_attention<KV_EXPANDED, HD>(p, q_map(ex.q, HD, (long long)p.heads * HD),
                                        make_tmap_bf16_2d(ex.k, HD, rows, HD, 64, 128),
                                        make_tmap_bf16_2d(ex.v, HD, rows, HD, 64, 128), shape, ws, ex, s);
    } else {
      const PagedWorkspace ws = paged_workspace(alloc(ws_bytes, false), blocks, kItemRows);
      const CUtensorMap none = q_map(p.q, p.q_stride_h, p.q_stride_t);  // nothing is read by TMA
      launch_attention<FMT, HD>(p, none, none, none, shape, ws, ex, s);
    }
  }
}

}  // namespace

void paged_attention_chunk(const PagedAttnParams& p, const PagedAlloc& alloc, cudaStream_t s) {
  const bool hd64 = p.pool.head_dim == 64;
  switch (p.pool.fmt) {
    case KV_E4M3: hd64 ? launch_chunk<KV_E4M3, 64>(p, alloc, s) : launch_chunk<KV_E4M3, 128>(p, alloc, s); break;
    case KV_INT8: hd64 ? launch_chunk<KV_INT8, 64>(p, alloc, s) : launch_chunk<KV_INT8, 128>(p, alloc, s); break;
    default: hd64 ? launch_chunk<KV_BF16, 64>(p, alloc, s) : launch_chunk<KV_BF16, 128>(p, alloc, s); break;
  }
}

}  // namespace b200
