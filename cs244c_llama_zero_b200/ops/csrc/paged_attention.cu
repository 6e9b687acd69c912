// Attention of new tokens over a paged key/value cache (causal, grouped heads, ragged batch): the form for
// few rows, the joining kernel of both forms, and the choice between them.
//
// Row i of a sequence with q_len new of kv_len cached tokens stands at position p = kv_len - q_len + i:
//   o = sum_{j <= p} softmax_j(scale * q . k_j) v_j      (p < 0: zeros)
//
// Few rows (one new token, or a handful): every cached byte is used for a handful of products, and the
// cache's bandwidth is the bound.  The work is cut into equal runs of 64-token units over all sequences and
// heads (paged_sched.cuh).  Four warps per block, each on its own 16 tokens of the unit with its own ring of
// cp.async stages, so that nothing synchronises the warps until a run ends.  A page holds a multiple of 16
// tokens: the 16 tokens of a warp are one contiguous piece of memory.
//
// Products on the warp matrix instructions with the TOKENS along M and the rows along N (S^T = K Q^T,
// O^T = V^T P^T): with 8 rows along N no part of the instruction is padding for groups of up to 8 heads.
//   bf16: K by ldmatrix, V^T by ldmatrix.trans, probabilities rounded to bf16.
//   8-bit: 16-byte shared loads; the codes become fp16 in registers, exactly (e4m3: one conversion per pair;
//   int8: the code + 128 as the low bits of 1024, less 1152), with the order of head_dim inside a product and
//   of O's rows chosen such that a lane's 16 bytes feed its own fragments.  A row of q is scaled by a power of
//   two to a maximum in [1, 2) before it is rounded to fp16, which its 8 bits survive down to 2^-17 of the
//   maximum.  k_scale multiplies the scores in fp32.  v_scale goes into the exponent: with
//   x_j = s_j + log2 v_scale_j the weights 2^(x_j - m) that meet the codes have their maximum near 1 whatever
//   the scales are, so fp16 holds them (the largest at 2^6, errors below 2^-30 of it), and the normaliser
//   sums 2^(x_j - m) / v_scale_j in fp32.
// Up to 16 rows each warp takes 16 of a unit's 64 tokens for all rows, and the four are joined at the end of
// an item.  Above, up to 64, each warp takes a quarter of the rows for all tokens: it expands every code
// itself, but holds a quarter of O (for all rows it spills), and nothing is joined.  64 rows of head_dim 64
// over 8 int8 caches of 40000 tokens in all: 50 us, against 79 us split by tokens.
// The running maximum is raised only when a score exceeds it by more than 2^8 (one vote per 16 tokens).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "paged.h"
#include "paged_sched.cuh"

namespace b200 {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRaise = 8.0f;  // log2 units
// The running maximum of a row that has seen nothing: finite, so that differences with it are numbers, and below
// every score.
constexpr float kNothing = -3.0e38f;
constexpr float kZeroScale = 8.2718061e-25f;  // 2^kLowestExponent
static_assert(kLowestExponent == -80, "kZeroScale");
constexpr int kDecodeWarps = 4;
constexpr int kDecodeThreads = 32 * kDecodeWarps;
constexpr int kUnitLog2 = 6;  // 16 tokens per warp

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <bool F16>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (F16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ void lds128(uint32_t addr, uint32_t (&w)[4]) {
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void lds64(uint32_t addr, uint32_t& w0, uint32_t& w1) {
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w0), "=r"(w1) : "r"(addr) : "memory");
}
__device__ __forceinline__ float lg2_approx(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lds32f(uint32_t addr) {
  float f;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(f) : "r"(addr) : "memory");
  return f;
}

template <bool F16>
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
  if constexpr (!F16) return pack_bf16(lo, hi);
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// The 8-bit codes (b0, b1) and (b2, b3) of a word as two fp16 pairs, exactly.  int8 codes come with their
// sign bit flipped (code + 128).
template <int FMT>
__device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t& p0, uint32_t& p1) {
  if constexpr (FMT == KV_INT8) {
    const uint32_t bias = 0x64806480u;  // 1152
    const uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
    const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&bias));
    const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&b), *reinterpret_cast<const __half2*>(&bias));
    p0 = *reinterpret_cast<const uint32_t*>(&x);
    p1 = *reinterpret_cast<const uint32_t*>(&y);
  } else {
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, hi;\n\t}"
        : "=r"(p0), "=r"(p1)
        : "r"(w));
  }
}
template <int FMT>
__device__ __forceinline__ uint32_t code_word(uint32_t w) {
  return FMT == KV_INT8 ? w ^ 0x80808080u : w;
}

// NT: 8-row tiles per warp.  BY_ROWS: the warps split the rows, not the tokens.
template <int FMT, int HD, int NT, bool BY_ROWS>
struct DecodeCfg {
  static constexpr int ROWS = 8 * NT * (BY_ROWS ? kDecodeWarps : 1);
  static constexpr int COPIES = BY_ROWS ? 1 : kDecodeWarps;  // of O, to be joined
  static constexpr int ELEM = FMT == KV_BF16 ? 2 : 1;
  static constexpr int ROW_BYTES = HD * ELEM;
  static constexpr int TILE = 16 * ROW_BYTES;                  // one warp's K (or V) of a unit
  static constexpr int SCALES = FMT == KV_BF16 ? 0 : 128;      // 16 fp32 scales of K, 16 of V
  static constexpr int STAGE = 2 * TILE + SCALES;
  static constexpr int STAGES = 3;
  static constexpr float HEADROOM = FMT == KV_BF16 ? 0.f : 6.f;  // log2 of the largest weight (before lazy raises)
  static constexpr int RING = STAGES * STAGE;                  // per warp
  static constexpr int O_LD = HD + 4;                          // row stride of the merge buffer, in floats
  static constexpr int MERGE = COPIES * ROWS * O_LD * 4;
  static constexpr int ML_OFF = kDecodeWarps * RING + MERGE;
  static constexpr int SMEM = ML_OFF + COPIES * ROWS * 8;
};

// Byte offset of 16-byte chunk c of token row `tok` in a tile of 16 rows, arranged such that the fragment
// loads of a quarter warp touch all banks once.
template <int FMT, int HD, bool IS_V>
__device__ __forceinline__ uint32_t chunk_offset(int tok, int c) {
  if constexpr (FMT == KV_BF16) {  // rows of 128 or 256 bytes; 8 rows of one chunk are read together
    return tok * (HD * 2) + (((c & 8) | ((c ^ tok) & 7)) << 4);
  } else if constexpr (HD == 128) {  // rows of 128 bytes
    return tok * 128 + ((c ^ (IS_V ? ((tok >> 1) & 3) << 1 : (tok & 1) << 2)) << 4);
  } else {  // two rows per 128 bytes
    const int line = tok >> 1, p = ((tok & 1) << 2) | c;
    return line * 128 + ((IS_V ? p ^ ((line & 3) << 1) : p) << 4);
  }
}
// Pass i of a tile's copy moves 512 bytes, 16 per lane.  Its lanes' offsets are those of pass 0 with these
// bits flipped, plus 512 i (the row bits that i and the lane contribute are disjoint).
template <int FMT, int HD, bool IS_V>
__device__ __forceinline__ constexpr uint32_t pass_flip(int i) {
  if (FMT == KV_BF16) return (HD == 64 ? (4 * i) & 7 : (2 * i) & 7) << 4;
  return HD == 128 && IS_V ? ((2 * i) & 3) << 5 : 0;
}

template <int FMT, int HD, int NT, bool BY_ROWS>
__global__ void __launch_bounds__(kDecodeThreads)
    paged_decode_kernel(const __grid_constant__ PagedAttnParams p, PagedShape shape, PagedWorkspace ws) {
  using C = DecodeCfg<FMT, HD, NT, BY_ROWS>;
  constexpr bool QUANT = FMT != KV_BF16;
  constexpr int KS = HD / 16;  // k-steps of the scores, and 16-column tiles of O
  extern __shared__ __align__(128) uint8_t smem[];
  pdl_wait_and_release();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = lane >> 2, j = lane & 3;  // the lane's place in a fragment
  const PagedRange range = find_range<kDecodeThreads>(p.seqs, shape, p.errs);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    ws.total[0] = range.total;
    ws.total[1] = range.blocks;
  }
  if ((int)blockIdx.x >= range.blocks) return;
  PagedItem it = range.item;
  if (threadIdx.x == 0) ws.records[blockIdx.x] = {range.begin, it.start, it.n_units, it.b, it.kvh, it.rt};
  if (range.begin == range.end) return;

  const uint32_t ring = smem_u32(smem) + warp * C::RING;
  float* merge = reinterpret_cast<float*>(smem + kDecodeWarps * C::RING);
  float2* ml_smem = reinterpret_cast<float2*>(smem + C::ML_OFF);
  const int page_log2 = p.seqs.page_log2, page_mask = (1 << page_log2) - 1;

  // ---- loads: a second walk over the same units, STAGES ahead
  PagedItem li = it;
  int l_unit = unit_of_cut(li, range.begin), l_stop = unit_of_cut(li, range.end);  // of this item
  bool loading = true;
  int l_visible = item_visible(li.seq, li.rt, shape.tile_tokens);
  uint32_t slot_in = ring;
  constexpr int PER_ROW = C::ROW_BYTES / 16;
  const uint32_t k_off0 = chunk_offset<FMT, HD, false>(lane / PER_ROW, lane % PER_ROW);
  const uint32_t v_off0 = chunk_offset<FMT, HD, true>(lane / PER_ROW, lane % PER_ROW) + C::TILE;
  // Page of this warp's tokens of the unit to load (-1: it sees none of them).  Read one unit ahead and
  // looked at only when the unit is loaded, so that nobody waits for it.
  auto page_of = [&]() {
    const int t = l_unit * 64 + 16 * warp;
    return t < l_visible ? p.seqs.table[(long long)li.b * p.seqs.table_stride + (t >> page_log2)] : -1;
  };
  int page = page_of();
  auto load_unit = [&]() {
    if (loading) {
      const int t0 = l_unit * 64 + 16 * warp;
      int live = min(16, l_visible - t0);
      if (live > 0 && (page < 0 || page >= p.seqs.n_pages)) {
        if (lane == 0) report_error(p.errs, kErrBadIndex, li.b);
        live = 0;
      }
      long long cell = live > 0 ? (((long long)page * shape.kv_heads + li.kvh) << page_log2) + (t0 & page_mask) : 0;
      if (!B200_IN_BOUNDS(p.errs, cell, max(live, 1), pool_cells(p.seqs, shape.kv_heads), 135)) cell = live = 0;
      const uint8_t* k_src = reinterpret_cast<const uint8_t*>(p.pool.k) + cell * C::ROW_BYTES + lane * 16;
      const uint8_t* v_src = reinterpret_cast<const uint8_t*>(p.pool.v) + cell * C::ROW_BYTES + lane * 16;
      const uint32_t k_dst = slot_in + k_off0, v_dst = slot_in + v_off0;
      if (live == 16) {
#pragma unroll
        for (int i = 0; i < C::TILE / 512; ++i) {
          cp_async16((k_dst ^ pass_flip<FMT, HD, false>(i)) + i * 512, k_src + i * 512, 16);
          cp_async16((v_dst ^ pass_flip<FMT, HD, true>(i)) + i * 512, v_src + i * 512, 16);
        }
      } else {  // rows behind the last visible token become zeros
#pragma unroll
        for (int i = 0; i < C::TILE / 512; ++i) {
          const int bytes = i * (32 / PER_ROW) + lane / PER_ROW < live ? 16 : 0;
          const int at = bytes ? i * 512 : -lane * 16;  // a copy of no bytes still names a valid address
          cp_async16((k_dst ^ pass_flip<FMT, HD, false>(i)) + i * 512, k_src + at, bytes);
          cp_async16((v_dst ^ pass_flip<FMT, HD, true>(i)) + i * 512, v_src + at, bytes);
        }
      }
      if constexpr (QUANT) {
        if (lane < 8) {
          const int i = lane & 3;
          const int bytes = max(0, min(16, (live - 4 * i) * 4));
          const float* src = (lane < 4 ? p.pool.k_scale : p.pool.v_scale) + cell + (bytes ? 4 * i : 0);
          cp_async16(slot_in + 2 * C::TILE + lane * 16, src, bytes);
        }
      }
      slot_in = slot_in + C::STAGE == ring + C::RING ? ring : slot_in + C::STAGE;
      if (++l_unit == l_stop) {
        loading = range.end > item_end(li);
        if (loading) {
          next_item(li, p.seqs, shape);
          l_unit = 0;
          l_stop = unit_of_cut(li, range.end);
          l_visible = item_visible(li.seq, li.rt, shape.tile_tokens);
        }
      }
      if (loading) page = page_of();
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < C::STAGES - (BY_ROWS ? 1 : 0); ++i) load_unit();

  // fragment addresses inside a stage (a stage starts on a multiple of 128 bytes: flipping bits 4 to 6 of the
  // sum flips them in the offset)
  uint32_t k_frag, v_frag;
  if constexpr (!QUANT) {
    k_frag = chunk_offset<FMT, HD, false>(lane & 15, lane >> 4);
    v_frag = C::TILE + chunk_offset<FMT, HD, true>((lane & 7) + ((lane >> 4) << 3), (lane >> 3) & 1);
  } else {
    k_frag = chunk_offset<FMT, HD, false>(n, j);
    v_frag = C::TILE + (HD == 128 ? chunk_offset<FMT, HD, true>(2 * j, n)
                                  : chunk_offset<FMT, HD, true>(2 * j, n >> 1) + ((n & 1) << 3));
  }

  const float scale2 = p.scale * kLog2e;
  // Row tile t of this warp starts at row row0 + t * row_step: split by rows, the tiles go round the warps.
  const int row0 = BY_ROWS ? warp * 8 : 0;
  constexpr int row_step = BY_ROWS ? 8 * kDecodeWarps : 8;
  const int copy0 = BY_ROWS ? 0 : warp * C::ROWS;
  // Q^T fragments of an item as bf16; rows that do not exist are zeros.  Asked for before the item ahead of it
  // is joined and written, so that the two latencies overlap.
  uint32_t qf[NT][KS][2];
  float q_unit[NT][2];  // 8-bit: what the scores of rows 2 j and 2 j + 1 are multiplied by
  auto load_q = [&](const PagedItem& x) {
    const int tok0 = x.rt * shape.tile_tokens;
    const int rows = min(shape.tile_tokens, x.seq.qn - tok0) * p.group;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int r = row0 + t * row_step + n;
      const bool ok = r < rows && B200_IN_BOUNDS(p.errs, x.seq.q0 + tok0 + r / p.group, 1, p.seqs.total_q, 134);
      const __nv_bfloat16* src = p.q + (long long)(x.seq.q0 + tok0 + r / p.group) * p.q_stride_t +
                                 (long long)(x.kvh * p.group + r % p.group) * p.q_stride_h;
      if constexpr (!QUANT) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          qf[t][ks][0] = ok ? *reinterpret_cast<const uint32_t*>(src + 16 * ks + 2 * j) : 0u;
          qf[t][ks][1] = ok ? *reinterpret_cast<const uint32_t*>(src + 16 * ks + 2 * j + 8) : 0u;
        }
      } else {  // product 4 g + x takes columns 64 g + 16 j + 4 x + {0, 1} and {2, 3}
#pragma unroll
        for (int g = 0; g < HD / 64; ++g) {
          uint4 w[2] = {make_uint4(0u, 0u, 0u, 0u), make_uint4(0u, 0u, 0u, 0u)};
          if (ok) {
            w[0] = *reinterpret_cast<const uint4*>(src + 64 * g + 16 * j);
            w[1] = *reinterpret_cast<const uint4*>(src + 64 * g + 16 * j + 8);
          }
          const uint32_t x8[8] = {w[0].x, w[0].y, w[0].z, w[0].w, w[1].x, w[1].y, w[1].z, w[1].w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            qf[t][4 * g + k][0] = x8[2 * k];
            qf[t][4 * g + k][1] = x8[2 * k + 1];
          }
        }
      }
    }
  };
  load_q(it);
  uint32_t slot_out = BY_ROWS ? smem_u32(smem) : ring;
  int stage = 0;
  bool first = true;
  int unit = unit_of_cut(it, range.begin);
  while (true) {  // one item, or the part of it in this block's range
    const int seg = unit_of_cut(it, range.end) - unit;
    const bool whole = seg == it.n_units;
    const int tok0 = it.rt * shape.tile_tokens;
    const int rows = min(shape.tile_tokens, it.seq.qn - tok0) * p.group;
    const int base_pos = it.seq.len - it.seq.qn + tok0;  // position of the item's first row
    const int visible = item_visible(it.seq, it.rt, shape.tile_tokens);
    if constexpr (QUANT) {  // to fp16, the row scaled by a power of two to a maximum in [1, 2)
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        uint32_t top = 0u;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          top = __vmaxu2(top, __vmaxu2(qf[t][ks][0] & 0x7FFF7FFFu, qf[t][ks][1] & 0x7FFF7FFFu));
        uint32_t m = max(top & 0xFFFFu, top >> 16);
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
        const int e = q_row_exponent(m);
        const float down = __uint_as_float((uint32_t)(254 - e) << 23), up = __uint_as_float((uint32_t)e << 23);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            qf[t][ks][h] = pack_pair<true>(bf16lo(qf[t][ks][h]) * down, bf16hi(qf[t][ks][h]) * down);
        q_unit[t][0] = scale2 * __shfl_sync(0xffffffffu, up, 8 * j);
        q_unit[t][1] = scale2 * __shfl_sync(0xffffffffu, up, 8 * j + 4);
      }
    }
    const int all_see = base_pos + 1;  // fewest visible tokens of any row

    float o[KS][NT][4];
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][t][e] = 0.f;
    float m_sub[NT][2], l[NT][2];  // the maximum in use less the headroom
#pragma unroll
    for (int t = 0; t < NT; ++t) m_sub[t][0] = m_sub[t][1] = kNothing, l[t][0] = l[t][1] = 0.f;

    // 16 tokens from t0 on, at `tile` in shared memory, against the first N row tiles
    auto step = [&](auto n_tiles, uint32_t tile, int t0) {
      constexpr int N = decltype(n_tiles)::value;
      const uint32_t ka = tile + k_frag, va = tile + v_frag;
      float s[N][4];
#pragma unroll
      for (int t = 0; t < N; ++t) s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.f;
      if constexpr (!QUANT) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          uint32_t a[4];
          ldsm_x4((ka ^ (((2 * ks) & 7) << 4)) + (ks >> 2) * 128, a);
#pragma unroll
          for (int t = 0; t < N; ++t) mma_16816<false>(s[t], a, qf[t][ks][0], qf[t][ks][1]);
        }
      } else {
#pragma unroll
        for (int g = 0; g < HD / 64; ++g) {
          uint32_t lo[4], hi[4];
          lds128(ka ^ (g << 6), lo);
          lds128((ka ^ (g << 6)) + 8 * HD, hi);
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            uint32_t a[4];
            codes_to_f16<FMT>(code_word<FMT>(lo[x]), a[0], a[2]);
            codes_to_f16<FMT>(code_word<FMT>(hi[x]), a[1], a[3]);
#pragma unroll
            for (int t = 0; t < N; ++t) mma_16816<true>(s[t], a, qf[t][4 * g + x][0], qf[t][4 * g + x][1]);
          }
        }
      }
      // scores in log2 units; 8-bit: plus log2 of v_scale, with w = 1 / v_scale for the normaliser
      float w0 = 1.f, w1 = 1.f;
      if constexpr (QUANT) {
        const uint32_t sa = tile + 2 * C::TILE + n * 4;
        const float k0 = lds32f(sa), k1 = lds32f(sa + 32), v0 = lds32f(sa + 64), v1 = lds32f(sa + 96);
        // a scale of 0 (all codes 0) counts as 2^kLowestExponent, one below 2^-100 as that; one that is no number
        // goes into the scores alone: rows that do not see the token add 0 * w
        float x0 = lg2_approx(v0 == 0.f ? kZeroScale : fmaxf(v0, 7.888609e-31f));
        float x1 = lg2_approx(v1 == 0.f ? kZeroScale : fmaxf(v1, 7.888609e-31f));
        w0 = ex2_approx(-x0);
        w1 = ex2_approx(-x1);
        x0 += v0 - v0;
        x1 += v1 - v1;
#pragma unroll
        for (int t = 0; t < N; ++t) {
          s[t][0] = fmaf(s[t][0], k0 * q_unit[t][0], x0);
          s[t][1] = fmaf(s[t][1], k0 * q_unit[t][1], x0);
          s[t][2] = fmaf(s[t][2], k1 * q_unit[t][0], x1);
          s[t][3] = fmaf(s[t][3], k1 * q_unit[t][1], x1);
        }
      } else {
#pragma unroll
        for (int t = 0; t < N; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[t][e] *= scale2;
      }
      if (t0 + 16 > all_see) {  // a row that does not exist is masked like the last one
#pragma unroll
        for (int t = 0; t < N; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int lim = min(base_pos + (row0 + t * row_step + 2 * j + e) / p.group + 1, visible);
            if (t0 + n >= lim) s[t][e] = -INFINITY;
            if (t0 + n + 8 >= lim) s[t][2 + e] = -INFINITY;
          }
      }
      // weights: 2^d with d = score - m + headroom
      float d[N][4], top = kNothing;
#pragma unroll
      for (int t = 0; t < N; ++t) {
#pragma unroll
        for (int e = 0; e < 4; ++e) d[t][e] = s[t][e] - m_sub[t][e & 1];
        top = fmax3f(fmax3f(top, d[t][0], d[t][1]), d[t][2], d[t][3]);
      }
      if (__any_sync(0xffffffffu, top > kRaise + C::HEADROOM)) {
#pragma unroll
        for (int t = 0; t < N; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float mx = fmaxf(s[t][e], s[t][2 + e]);
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            const float m_new = fmaxf(m_sub[t][e], mx - C::HEADROOM);
            const float alpha = ex2_approx(m_sub[t][e] - m_new);
            m_sub[t][e] = m_new;
            l[t][e] *= alpha;
#pragma unroll
            for (int i = 0; i < KS; ++i) {
              o[i][t][e] *= alpha;
              o[i][t][2 + e] *= alpha;
            }
            d[t][e] = s[t][e] - m_new;
            d[t][2 + e] = s[t][2 + e] - m_new;
          }
      }
      uint32_t pf[N][2];
#pragma unroll
      for (int t = 0; t < N; ++t) {
        const float p0 = ex2_approx(d[t][0]), p1 = ex2_approx(d[t][1]);
        const float p2 = ex2_approx(d[t][2]), p3 = ex2_approx(d[t][3]);
        l[t][0] += QUANT ? fmaf(p0, w0, p2 * w1) : p0 + p2;
        l[t][1] += QUANT ? fmaf(p1, w0, p3 * w1) : p1 + p3;
        // rounded for the product with V (bf16: half a step of 2^-8 relative for each probability)
        pf[t][0] = transpose_8x8(pack_pair<QUANT>(p0, p1));
        pf[t][1] = transpose_8x8(pack_pair<QUANT>(p2, p3));
      }
      if constexpr (!QUANT) {
        // Where some rows do not see all tokens, infinities and NaN are taken out of V (0 times them would be NaN)
        // and put back as NaN into the columns of the rows that do see them.
        if (t0 + 16 > all_see && rows > p.group) {
#pragma unroll
          for (int i = 0; i < KS; ++i) {
            uint32_t a[4], bad[4];
            ldsm_x4_t((va ^ (((2 * i) & 7) << 4)) + (i >> 2) * 128, a);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              bad[x] = __vcmpeq2(a[x] & 0x7F807F80u, 0x7F807F80u);
              a[x] &= ~bad[x];
            }
#pragma unroll
            for (int t = 0; t < N; ++t) mma_16816<false>(o[i][t], a, pf[t][0], pf[t][1]);
            if (!__any_sync(0xffffffffu, (bad[0] | bad[1] | bad[2] | bad[3]) != 0u)) continue;
            // columns 16 i + n (a[0], a[2]) and 8 more (a[1], a[3]); tokens 2 j, 2 j + 1 and 8 more
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              int lowest = 16;  // token that holds one
#pragma unroll
              for (int x = 3; x >= 0; --x)
                if ((bad[h + (x & 2)] >> (16 * (x & 1))) & 1u) lowest = 2 * j + 4 * (x & 2) + (x & 1);
              lowest = min(lowest, __shfl_xor_sync(0xffffffffu, lowest, 1));
              lowest = min(lowest, __shfl_xor_sync(0xffffffffu, lowest, 2));
#pragma unroll
              for (int t = 0; t < N; ++t)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const int lim = min(base_pos + (row0 + t * row_step + 2 * j + e) / p.group + 1, visible);
                  if (lowest < 16 && t0 + lowest < lim) o[i][t][2 * h + e] = __int_as_float(0x7FC00000);
                }
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < KS; ++i) {
            uint32_t a[4];
            ldsm_x4_t((va ^ (((2 * i) & 7) << 4)) + (i >> 2) * 128, a);
#pragma unroll
            for (int t = 0; t < N; ++t) mma_16816<false>(o[i][t], a, pf[t][0], pf[t][1]);
          }
        }
      } else {
        // tile i: O's rows n and n + 8 are columns n * HD / 8 + 2 i and + 1 of V; words of tokens
        // 2 j, 2 j + 1, 2 j + 8, 2 j + 9
        constexpr int W = HD / 32;
        uint32_t w[4][W];
        if constexpr (HD == 128) {
          lds128(va, w[0]);
          lds128(va + 128, w[1]);
          lds128(va + 1024, w[2]);
          lds128(va + 1152, w[3]);
        } else {
          lds64(va, w[0][0], w[0][1]);
          lds64(va ^ 64, w[1][0], w[1][1]);
          lds64(va + 512, w[2][0], w[2][1]);
          lds64((va ^ 64) + 512, w[3][0], w[3][1]);
        }
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          const int k = i >> 1;
          const uint32_t sel = (i & 1) ? 0x7362u : 0x5140u;
          uint32_t a[4];
          codes_to_f16<FMT>(code_word<FMT>(__byte_perm(w[0][k], w[1][k], sel)), a[0], a[1]);
          codes_to_f16<FMT>(code_word<FMT>(__byte_perm(w[2][k], w[3][k], sel)), a[2], a[3]);
#pragma unroll
          for (int t = 0; t < N; ++t) mma_16816<true>(o[i][t], a, pf[t][0], pf[t][1]);
        }
      }
    };
    const int live_tiles = min(NT, max(0, (rows - row0 + row_step - 1) / row_step));

    for (int c = 0; c < seg; ++c, ++unit) {
      if constexpr (BY_ROWS) {
        cp_async_wait<C::STAGES - 2>();
        __syncthreads();  // the stage is there for all warps, and all have read the one before
        load_unit();
      } else {
        cp_async_wait<C::STAGES - 1>();
        __syncwarp();
      }
#pragma unroll 1
      for (int x = 0; x < (BY_ROWS ? kDecodeWarps : 1); ++x) {
        const uint32_t tile = slot_out + (BY_ROWS ? x * C::RING : 0);
        const int t0 = unit * 64 + 16 * (BY_ROWS ? x : warp);
        if (t0 >= visible) break;
        if (NT > 1 && live_tiles < NT) {
          if (live_tiles > 0) step(std::integral_constant<int, 1>(), tile, t0);
        } else if (NT > 1 || !BY_ROWS || live_tiles > 0) {
          step(std::integral_constant<int, NT>(), tile, t0);
        }
      }
      if constexpr (!BY_ROWS) {
        __syncwarp();  // every lane has read the stage before it is loaded again
        load_unit();
      }
      slot_out += C::STAGE;
      if (++stage == C::STAGES) {
        stage = 0;
        slot_out -= C::RING;
      }
    }

    // ---- join the warps
    const int q0 = it.seq.q0 + tok0, head0 = it.kvh * p.group;
    const bool more = range.end > item_end(it);
    if (more) {
      next_item(it, p.seqs, shape);
      load_q(it);
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], x);
        if (n == 0) ml_smem[copy0 + row0 + t * row_step + 2 * j + e] = make_float2(m_sub[t][e], l[t][e]);
      }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = row0 + t * row_step + 2 * j + e;
        if (r >= rows) continue;
        float mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < C::COPIES; ++w) mx = fmaxf(mx, ml_smem[w * C::ROWS + r].x);
        const float f = ex2_approx(m_sub[t][e] - mx);
        float* dst = merge + (copy0 + r) * C::O_LD;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          const int d0 = QUANT ? n * (HD / 8) + 2 * i : 16 * i + n;
          const int d1 = QUANT ? d0 + 1 : d0 + 8;
          dst[d0] = o[i][t][e] * f;
          dst[d1] = o[i][t][2 + e] * f;
        }
      }
    __syncthreads();
    const int slot = 2 * blockIdx.x + (first ? 0 : 1);
    for (int x = threadIdx.x; x < rows * (HD / 4); x += kDecodeThreads) {
      const int r = x / (HD / 4), d = (x % (HD / 4)) * 4;
      float mx = -INFINITY, sum = 0.f;
#pragma unroll
      for (int w = 0; w < C::COPIES; ++w) mx = fmaxf(mx, ml_smem[w * C::ROWS + r].x);
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < C::COPIES; ++w) {
        const float2 q = ml_smem[w * C::ROWS + r];
        sum += q.x == mx ? q.y : q.y * ex2_approx(q.x - mx);
        const float4 v = *reinterpret_cast<const float4*>(merge + (w * C::ROWS + r) * C::O_LD + d);
        a.x += v.x;
        a.y += v.y;
        a.z += v.z;
        a.w += v.w;
      }
      if (whole) {
        if (!B200_IN_BOUNDS(p.errs, q0 + r / p.group, 1, p.seqs.total_q, 136)) continue;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        __nv_bfloat16* dst = p.out + (long long)(q0 + r / p.group) * p.o_stride_t +
                             (long long)(head0 + r % p.group) * p.o_stride_h + d;
        *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(a.x * inv, a.y * inv), pack_bf16(a.z * inv, a.w * inv));
      } else if (B200_IN_BOUNDS(p.errs, (long long)slot * C::ROWS + r, 1, 2ll * gridDim.x * C::ROWS, 137)) {
        *reinterpret_cast<float4*>(ws.o + ((size_t)slot * C::ROWS + r) * HD + d) = a;
        if (d == 0) ws.ml[(size_t)slot * C::ROWS + r] = make_float2(mx, sum);
      }
    }
    if (!more) break;
    first = false;
    unit = 0;
    __syncthreads();  // the merge buffers are free
  }
  cp_async_wait<0>();
}

// Joins the parts of items that lie in more than one block's range.  Block x + 1 of the attention kernel
// starts inside an item, or does not; the first block that does joins the item.  WARPS_PER_ROW warps share
// the parts of a row; ROWS rows per part.  Few and large blocks: most find nothing to do, and a launch of one
// block per row (28000 for 64 rows) took 25 us for that alone.
constexpr int kJoinThreads = 256;
constexpr int kAhead = 4;
template <int HD, int ROWS, int WARPS_PER_ROW>
__global__ void __launch_bounds__(kJoinThreads)
    paged_join_kernel(const __grid_constant__ PagedAttnParams p, PagedShape shape, PagedWorkspace ws) {
  pdl_wait_and_release();
  constexpr int ROWS_AT_ONCE = kJoinThreads / 32 / WARPS_PER_ROW;
  constexpr int V = HD / 32;  // columns per lane
  const PagedJoin join = find_join(ws, blockIdx.x + 1);
  if (join.parts == 0) return;
  const PagedRecord& rec = join.rec;
  const int parts = join.parts;
  auto slot = [&](int i) { return join.slot(i); };
  const SeqInfo seq = seq_info(p.seqs, rec.b);
  const int tok0 = rec.rt * shape.tile_tokens;
  const int rows = min(shape.tile_tokens, seq.qn - tok0) * p.group;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = warp % WARPS_PER_ROW;
  __shared__ float part[kJoinThreads / 32][HD];
  __shared__ float part_l[kJoinThreads / 32];
  for (int r0 = blockIdx.y * ROWS_AT_ONCE; r0 < rows; r0 += gridDim.y * ROWS_AT_ONCE) {
    const int r = r0 + warp / WARPS_PER_ROW;
    const bool live = r < rows;
    // the first parts' sums are asked for together with the maxima
    float ahead[kAhead][V];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = sub + k * WARPS_PER_ROW;
      if (live && i < parts) {
        const float* src = ws.o + ((size_t)slot(i) * ROWS + r) * HD + lane * V;
#pragma unroll
        for (int e = 0; e < V; e += 2) {
          const float2 v = *reinterpret_cast<const float2*>(src + e);
          ahead[k][e] = v.x;
          ahead[k][e + 1] = v.y;
        }
      }
    }
    float mx = -INFINITY;
    if (live)
      for (int i = lane; i < parts; i += 32) mx = fmaxf(mx, ws.ml[(size_t)slot(i) * ROWS + r].x);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
    float acc[V], l = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = 0.f;
    if (live) {
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int i = sub + k * WARPS_PER_ROW;
        if (i < parts) {
          const float2 q = ws.ml[(size_t)slot(i) * ROWS + r];
          const float f = q.x == mx ? 1.f : ex2_approx(q.x - mx);
          l += q.y * f;
#pragma unroll
          for (int e = 0; e < V; ++e) acc[e] += ahead[k][e] * f;
        }
      }
#pragma unroll 8
      for (int i = sub + kAhead * WARPS_PER_ROW; i < parts; i += WARPS_PER_ROW) {
        const size_t at = (size_t)slot(i) * ROWS + r;
        const float2 q = ws.ml[at];
        const float f = q.x == mx ? 1.f : ex2_approx(q.x - mx);
        l += q.y * f;
        const float* src = ws.o + at * HD + lane * V;
        if constexpr (V == 4) {
          const float4 v = *reinterpret_cast<const float4*>(src);
          acc[0] += v.x * f;
          acc[1] += v.y * f;
          acc[2] += v.z * f;
          acc[3] += v.w * f;
        } else {
          const float2 v = *reinterpret_cast<const float2*>(src);
          acc[0] += v.x * f;
          acc[1] += v.y * f;
        }
      }
    }
    if constexpr (WARPS_PER_ROW > 1) {
#pragma unroll
      for (int e = 0; e < V; ++e) part[warp][lane * V + e] = acc[e];
      if (lane == 0) part_l[warp] = l;
      __syncthreads();
      if (sub == 0)
#pragma unroll
        for (int w = 1; w < WARPS_PER_ROW; ++w) {
          l += part_l[warp + w];
#pragma unroll
          for (int e = 0; e < V; ++e) acc[e] += part[warp + w][lane * V + e];
        }
      __syncthreads();
    }
    if (live && sub == 0 && B200_IN_BOUNDS(p.errs, seq.q0 + tok0 + r / p.group, 1, p.seqs.total_q, 138)) {
      const float inv = l == 0.f ? 0.f : 1.f / l;
      __nv_bfloat16* dst = p.out + (long long)(seq.q0 + tok0 + r / p.group) * p.o_stride_t +
                           (long long)(rec.kvh * p.group + r % p.group) * p.o_stride_h + lane * V;
      if constexpr (V == 4)
        *reinterpret_cast<uint2*>(dst) =
            make_uint2(pack_bf16(acc[0] * inv, acc[1] * inv), pack_bf16(acc[2] * inv, acc[3] * inv));
      else
        *reinterpret_cast<uint32_t*>(dst) = pack_bf16(acc[0] * inv, acc[1] * inv);
    }
  }
}

// Blocks of the kernel that the current device holds at once.
template <int FMT, int HD, int NT, bool BY_ROWS>
int decode_blocks() {
  using C = DecodeCfg<FMT, HD, NT, BY_ROWS>;
  static std::atomic<int> cached[64];
  int dev = 0;
  B200_CUDA_CHECK(cudaGetDevice(&dev));
  B200_CHECK(dev >= 0 && dev < 64, "device index out of range");
  int n = cached[dev].load(std::memory_order_acquire);
  if (n == 0) {
    auto* kernel = paged_decode_kernel<FMT, HD, NT, BY_ROWS>;
    B200_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    int per_sm = 0;
    B200_CUDA_CHECK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, kDecodeThreads, C::SMEM));
    B200_CHECK(per_sm > 0, "paged attention: the kernel does not fit an SM");
    n = per_sm * num_sms_cached();
    cached[dev].store(n, std::memory_order_release);
  }
  return n;
}

template <int FMT, int HD, int NT, bool BY_ROWS>
void launch_decode(const PagedAttnParams& p, const PagedAlloc& alloc, cudaStream_t s) {
  using C = DecodeCfg<FMT, HD, NT, BY_ROWS>;
  const int blocks = decode_blocks<FMT, HD, NT, BY_ROWS>();
  const PagedWorkspace ws = paged_workspace(alloc(paged_workspace_bytes(blocks, C::ROWS, HD), false), blocks, C::ROWS);
  const PagedShape shape{std::max(1, C::ROWS / p.group), kUnitLog2, p.pool.kv_heads};
  launch_k(paged_decode_kernel<FMT, HD, NT, BY_ROWS>, dim3(blocks), dim3(kDecodeThreads), C::SMEM, s, 1, p, shape, ws);
  // one row has many parts when there are few rows, and few when there are many
  constexpr int WARPS_PER_ROW = C::ROWS <= 16 ? 4 : 1;
  launch_k(paged_join_kernel<HD, C::ROWS, WARPS_PER_ROW>, dim3(blocks - 1, 4), dim3(kJoinThreads), 0, s, 1, p, shape,
           ws);
  B200_CUDA_CHECK(cudaGetLastError());
  count_launch(2);
}

template <int FMT, int HD>
void launch_rows(const PagedAttnParams& p, const PagedAlloc& alloc, cudaStream_t s) {
  const long long rows = (long long)p.seqs.max_q * p.group;
  if (rows <= 8)
    launch_decode<FMT, HD, 1, false>(p, alloc, s);
  else if (rows <= 16)
    launch_decode<FMT, HD, 2, false>(p, alloc, s);
  else if (rows <= 32)
    launch_decode<FMT, HD, 1, true>(p, alloc, s);
  else if (rows <= 64 && !(FMT == KV_BF16 && HD == 128))  // there two blocks fit an SM: 98 us against 62 in chunks
    launch_decode<FMT, HD, 2, true>(p, alloc, s);
  else
    paged_attention_chunk(p, alloc, s);
}

template <int FMT>
void launch_head_dim(const PagedAttnParams& p, const PagedAlloc& alloc, cudaStream_t s) {
  if (p.pool.head_dim == 64)
    launch_rows<FMT, 64>(p, alloc, s);
  else
    launch_rows<FMT, 128>(p, alloc, s);
}

}  // namespace

void paged_attention(const PagedAttnParams& p_in, const PagedAlloc& alloc, cudaStream_t s) {
  PagedAttnParams p = p_in;
  if (p.seqs.total_q == 0 || p.seqs.batch == 0) return;
  p.errs = device_errors_ptr();
  switch (p.pool.fmt) {
    case KV_E4M3: launch_head_dim<KV_E4M3>(p, alloc, s); break;
    case KV_INT8: launch_head_dim<KV_INT8>(p, alloc, s); break;
    default: launch_head_dim<KV_BF16>(p, alloc, s); break;
  }
}

}  // namespace b200
