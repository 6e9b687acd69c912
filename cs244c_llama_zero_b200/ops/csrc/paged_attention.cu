// Attention of new tokens over a paged key/value cache (causal, grouped heads, ragged batch): the form for
// few rows, the joining kernel of both forms, and the choice between them.
//
// Row i of a sequence with q_len new of kv_len cached tokens stands at position p = kv_len - q_len + i:
//   o = sum_{j <= p} softmax_j(scale * q . k_j) v_j      (p < 0: zeros)
//
// Few rows (at most 16 per kv head, so one new token in particular): every cached byte is used for a
// handful of products, and the cache's bandwidth is the bound.  The work is cut into equal runs of 64-token
// units over all sequences and heads (paged_sched.cuh).  Four warps per block, each on its own 16 tokens of
// the unit with its own ring of cp.async stages, so that nothing synchronises the warps until a run ends.
// A page holds a multiple of 16 tokens: the 16 tokens of a warp are one contiguous piece of memory.
//
// Products on the warp matrix instructions with the TOKENS along M and the rows along N (S^T = K Q^T,
// O^T = V^T P^T): with 8 rows along N no part of the instruction is padding for groups of up to 8 heads.
//   bf16: K by ldmatrix, V^T by ldmatrix.trans.
//   8-bit: 16-byte shared loads; the codes become bf16 in registers (exactly) by integer operations and one
//   packed add or multiply, with the order of head_dim inside a product and of O's rows chosen such that a
//   lane's 16 bytes feed its own fragments.  k_scale multiplies the scores in fp32, v_scale the probabilities
//   before they are rounded to bf16.
// The running maximum is raised only when a score exceeds it by more than 2^8 (one vote per 16 tokens).
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "kernels.h"
#include "paged.h"
#include "paged_sched.cuh"

namespace b200 {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRaise = 8.0f;  // log2 units
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
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
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
__device__ __forceinline__ float lds32f(uint32_t addr) {
  float f;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(f) : "r"(addr) : "memory");
  return f;
}

// Two 8-bit codes, each in both bytes of its 16-bit half of t, as a pair of bf16 (exact).
template <int FMT>
__device__ __forceinline__ uint32_t codes_to_bf16(uint32_t t) {
  if constexpr (FMT == KV_INT8) {
    // 128 + low 7 bits, minus 128 or (sign bit set) 256: bf16 holds all of these exactly
    const uint32_t a = (t & 0x007F007Fu) | 0x43004300u, c = (t & 0x00800080u) | 0x43004300u;
    __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&c));
    return *reinterpret_cast<uint32_t*>(&d);
  } else {
    // exponent and mantissa moved to bf16's places give the value times 2^-120, subnormals included
    const uint32_t a = ((t << 4) & 0x07F007F0u) | (t & 0x80008000u);
    const uint32_t unit = 0x7B807B80u;  // 2^120
    __nv_bfloat162 d = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&unit));
    return *reinterpret_cast<uint32_t*>(&d);
  }
}

template <int FMT, int HD, int NT>
struct DecodeCfg {
  static constexpr int ROWS = 8 * NT;
  static constexpr int ELEM = FMT == KV_BF16 ? 2 : 1;
  static constexpr int ROW_BYTES = HD * ELEM;
  static constexpr int TILE = 16 * ROW_BYTES;                  // one warp's K (or V) of a unit
  static constexpr int SCALES = FMT == KV_BF16 ? 0 : 128;      // 16 fp32 scales of K, 16 of V
  static constexpr int STAGE = 2 * TILE + SCALES;
  static constexpr int STAGES = 3;
  static constexpr int RING = STAGES * STAGE;                  // per warp
  static constexpr int O_LD = HD + 4;                          // row stride of the merge buffer, in floats
  static constexpr int MERGE = kDecodeWarps * ROWS * O_LD * 4;
  static constexpr int ML_OFF = kDecodeWarps * RING + MERGE;
  static constexpr int SMEM = ML_OFF + kDecodeWarps * ROWS * 8;
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

template <int FMT, int HD, int NT>
__global__ void __launch_bounds__(kDecodeThreads)
    paged_decode_kernel(const __grid_constant__ PagedAttnParams p, PagedShape shape, PagedWorkspace ws) {
  using C = DecodeCfg<FMT, HD, NT>;
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
  const long long u_begin = range_begin(blockIdx.x, range.total, range.blocks);
  const long long u_end = range_begin(blockIdx.x + 1, range.total, range.blocks);
  PagedItem it = item_at(p.seqs, shape, range.b, range.base, u_begin);
  if (threadIdx.x == 0) ws.records[blockIdx.x] = {it.start, it.n_units, it.b, it.kvh, it.rt};

  const uint32_t ring = smem_u32(smem) + warp * C::RING;
  float* merge = reinterpret_cast<float*>(smem + kDecodeWarps * C::RING);
  float2* ml_smem = reinterpret_cast<float2*>(smem + C::ML_OFF);
  const int page_log2 = p.seqs.page_log2, page_mask = (1 << page_log2) - 1;

  // ---- loads: a second walk over the same units, STAGES - 1 ahead
  PagedItem li = it;
  long long lu = u_begin;
  int slot_in = 0;
  auto first_page = [&](const PagedItem& x, int t) {  // page of token t of item x, -1 if it has none
    if (t >= item_visible(x.seq, x.rt, shape.tile_tokens)) return -1;
    const int page = p.seqs.table[(long long)x.b * p.seqs.table_stride + (t >> page_log2)];
    if (page >= 0 && page < p.seqs.n_pages) return page;
    if (lane == 0) report_error(p.errs, kErrBadIndex, x.b);
    return -1;
  };
  int page = first_page(li, (int)(lu - li.start) * 64 + 16 * warp);
  auto load_unit = [&]() {
    if (lu < u_end) {
      const int t0 = (int)(lu - li.start) * 64 + 16 * warp;
      const int live = page >= 0 ? min(16, item_visible(li.seq, li.rt, shape.tile_tokens) - t0) : 0;
      const long long cell =
          live > 0 ? (((long long)page * shape.kv_heads + li.kvh) << page_log2) + (t0 & page_mask) : 0;
      const uint32_t dst = ring + slot_in * C::STAGE;
      constexpr int PER_ROW = C::ROW_BYTES / 16;
#pragma unroll
      for (int i = 0; i < C::TILE / 512; ++i) {
        const int id = i * 32 + lane, tok = id / PER_ROW, c = id % PER_ROW;
        const int bytes = tok < live ? 16 : 0;  // rows behind the last visible token become zeros
        const size_t off = bytes ? (size_t)cell * C::ROW_BYTES + (size_t)id * 16 : 0;
        cp_async16(dst + chunk_offset<FMT, HD, false>(tok, c), reinterpret_cast<const uint8_t*>(p.pool.k) + off, bytes);
        cp_async16(dst + C::TILE + chunk_offset<FMT, HD, true>(tok, c),
                   reinterpret_cast<const uint8_t*>(p.pool.v) + off, bytes);
      }
      if constexpr (FMT != KV_BF16) {
        if (lane < 8) {
          const int i = lane & 3;
          const int bytes = max(0, min(16, (live - 4 * i) * 4));
          const float* src = (lane < 4 ? p.pool.k_scale : p.pool.v_scale) + (bytes ? cell + 4 * i : 0);
          cp_async16(dst + 2 * C::TILE + lane * 16, src, bytes);
        }
      }
      slot_in = slot_in + 1 == C::STAGES ? 0 : slot_in + 1;
      if (++lu < u_end) {
        if (lu == li.start + li.n_units) next_item(li, p.seqs, shape);
        page = first_page(li, (int)(lu - li.start) * 64 + 16 * warp);
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < C::STAGES - 1; ++i) load_unit();

  const float scale2 = p.scale * kLog2e;
  int slot_out = 0;
  long long u = u_begin;
  while (true) {  // one item, or the part of it in this block's range
    const long long seg_end = min(u_end, it.start + it.n_units);
    const bool whole = u == it.start && seg_end == it.start + it.n_units;
    const bool first = u == u_begin;
    const int tok0 = it.rt * shape.tile_tokens;
    const int rows = min(shape.tile_tokens, it.seq.qn - tok0) * p.group;
    const int base_pos = it.seq.len - it.seq.qn + tok0;  // position of the item's first row
    // Q^T fragments; rows that do not exist are zeros
    uint32_t qf[NT][HD / 16][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int r = 8 * t + n;
      const bool ok = r < rows;
      const __nv_bfloat16* src = p.q + (long long)(it.seq.q0 + tok0 + r / p.group) * p.q_stride_t +
                                 (long long)(it.kvh * p.group + r % p.group) * p.q_stride_h;
      if constexpr (FMT == KV_BF16) {
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks) {
          qf[t][ks][0] = ok ? *reinterpret_cast<const uint32_t*>(src + 16 * ks + 2 * j) : 0u;
          qf[t][ks][1] = ok ? *reinterpret_cast<const uint32_t*>(src + 16 * ks + 2 * j + 8) : 0u;
        }
      } else {  // product 4 g + s takes columns 64 g + 16 j + 4 s + {0, 2} and {1, 3}
#pragma unroll
        for (int g = 0; g < HD / 64; ++g) {
          uint4 w[2] = {make_uint4(0u, 0u, 0u, 0u), make_uint4(0u, 0u, 0u, 0u)};
          if (ok) {
            w[0] = *reinterpret_cast<const uint4*>(src + 64 * g + 16 * j);
            w[1] = *reinterpret_cast<const uint4*>(src + 64 * g + 16 * j + 8);
          }
          const uint32_t x[8] = {w[0].x, w[0].y, w[0].z, w[0].w, w[1].x, w[1].y, w[1].z, w[1].w};
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            qf[t][4 * g + s][0] = __byte_perm(x[2 * s], x[2 * s + 1], 0x5410);
            qf[t][4 * g + s][1] = __byte_perm(x[2 * s], x[2 * s + 1], 0x7632);
          }
        }
      }
    }
    // visible tokens of the rows this lane holds scores of, and the fewest of any row
    int lim[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = 8 * t + 2 * j + e;
        lim[t][e] = r < rows ? base_pos + r / p.group + 1 : 0x7FFFFFFF;
      }
    const int all_see = base_pos + 1;
    const int visible = item_visible(it.seq, it.rt, shape.tile_tokens);

    float o[HD / 16][NT][4];
#pragma unroll
    for (int i = 0; i < HD / 16; ++i)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][t][e] = 0.f;
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) m[t][0] = m[t][1] = -INFINITY, l[t][0] = l[t][1] = 0.f;

    for (; u < seg_end; ++u) {
      load_unit();
      cp_async_wait<C::STAGES - 1>();
      __syncwarp();
      const uint32_t ks_tile = ring + slot_out * C::STAGE, vs_tile = ks_tile + C::TILE;
      const int t0 = (int)(u - it.start) * 64 + 16 * warp;
      if (t0 < visible) {
        float s[NT][4];
#pragma unroll
        for (int t = 0; t < NT; ++t) s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.f;
        if constexpr (FMT == KV_BF16) {
          const int tok = lane & 15;
#pragma unroll
          for (int ks = 0; ks < HD / 16; ++ks) {
            uint32_t a[4];
            ldsm_x4(ks_tile + chunk_offset<FMT, HD, false>(tok, 2 * ks + (lane >> 4)), a);
#pragma unroll
            for (int t = 0; t < NT; ++t) mma_bf16(s[t], a, qf[t][ks][0], qf[t][ks][1]);
          }
        } else {
#pragma unroll
          for (int g = 0; g < HD / 64; ++g) {
            uint32_t lo[4], hi[4];
            lds128(ks_tile + chunk_offset<FMT, HD, false>(n, 4 * g + j), lo);
            lds128(ks_tile + chunk_offset<FMT, HD, false>(n + 8, 4 * g + j), hi);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const uint32_t a[4] = {codes_to_bf16<FMT>(__byte_perm(lo[x], 0, 0x2200)),
                                     codes_to_bf16<FMT>(__byte_perm(hi[x], 0, 0x2200)),
                                     codes_to_bf16<FMT>(__byte_perm(lo[x], 0, 0x3311)),
                                     codes_to_bf16<FMT>(__byte_perm(hi[x], 0, 0x3311))};
#pragma unroll
              for (int t = 0; t < NT; ++t) mma_bf16(s[t], a, qf[t][4 * g + x][0], qf[t][4 * g + x][1]);
            }
          }
        }
        // scores in log2 units
        float kf0 = scale2, kf1 = scale2, vf0 = 1.f, vf1 = 1.f;
        if constexpr (FMT != KV_BF16) {
          kf0 *= lds32f(ks_tile + 2 * C::TILE + n * 4);
          kf1 *= lds32f(ks_tile + 2 * C::TILE + n * 4 + 32);
          vf0 = lds32f(ks_tile + 2 * C::TILE + 64 + n * 4);
          vf1 = lds32f(ks_tile + 2 * C::TILE + 64 + n * 4 + 32);
        }
        bool raise = false;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          s[t][0] *= kf0;
          s[t][1] *= kf0;
          s[t][2] *= kf1;
          s[t][3] *= kf1;
          if (t0 + 16 > all_see) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              if (t0 + n >= min(lim[t][e], visible)) s[t][e] = -INFINITY;
              if (t0 + n + 8 >= min(lim[t][e], visible)) s[t][2 + e] = -INFINITY;
            }
          }
          raise |= fmaxf(s[t][0], s[t][2]) > m[t][0] + kRaise || fmaxf(s[t][1], s[t][3]) > m[t][1] + kRaise;
        }
        if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float mx = fmaxf(s[t][e], s[t][2 + e]);
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
              const float m_new = fmaxf(m[t][e], mx);
              const float alpha = m_new == m[t][e] ? 1.f : ex2_approx(m[t][e] - m_new);
              m[t][e] = m_new;
              l[t][e] *= alpha;
#pragma unroll
              for (int i = 0; i < HD / 16; ++i) {
                o[i][t][e] *= alpha;
                o[i][t][2 + e] *= alpha;
              }
            }
        }
        uint32_t pf[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const float m0 = m[t][0] == -INFINITY ? 0.f : m[t][0], m1 = m[t][1] == -INFINITY ? 0.f : m[t][1];
          const float p0 = ex2_approx(s[t][0] - m0), p1 = ex2_approx(s[t][1] - m1);
          const float p2 = ex2_approx(s[t][2] - m0), p3 = ex2_approx(s[t][3] - m1);
          l[t][0] += p0 + p2;
          l[t][1] += p1 + p3;
          // rounded to bf16 for the product with V: half a step of 2^-8 relative for each probability
          pf[t][0] = transpose_8x8(pack_bf16(p0 * vf0, p1 * vf0));
          pf[t][1] = transpose_8x8(pack_bf16(p2 * vf1, p3 * vf1));
        }
        if constexpr (FMT == KV_BF16) {
          const int tok = (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
          for (int i = 0; i < HD / 16; ++i) {
            uint32_t a[4];
            ldsm_x4_t(vs_tile + chunk_offset<FMT, HD, true>(tok, 2 * i + ((lane >> 3) & 1)), a);
#pragma unroll
            for (int t = 0; t < NT; ++t) mma_bf16(o[i][t], a, pf[t][0], pf[t][1]);
          }
        } else {
          // tile i: O's rows n and n + 8 are columns n * HD / 8 + 2 i and + 1 of V
          constexpr int W = HD / 32;  // words per lane and token
          uint32_t w[4][W];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int tok = 2 * j + (x & 1) + ((x >> 1) << 3);
            if constexpr (HD == 128) {
              lds128(vs_tile + chunk_offset<FMT, HD, true>(tok, n), w[x]);
            } else {
              lds64(vs_tile + chunk_offset<FMT, HD, true>(tok, n >> 1) + ((n & 1) << 3), w[x][0], w[x][1]);
            }
          }
#pragma unroll
          for (int i = 0; i < HD / 16; ++i) {
            const int k = i >> 1;
            const uint32_t s0 = (i & 1) ? 0x6622u : 0x4400u, s1 = (i & 1) ? 0x7733u : 0x5511u;
            const uint32_t a[4] = {codes_to_bf16<FMT>(__byte_perm(w[0][k], w[1][k], s0)),
                                   codes_to_bf16<FMT>(__byte_perm(w[0][k], w[1][k], s1)),
                                   codes_to_bf16<FMT>(__byte_perm(w[2][k], w[3][k], s0)),
                                   codes_to_bf16<FMT>(__byte_perm(w[2][k], w[3][k], s1))};
#pragma unroll
            for (int t = 0; t < NT; ++t) mma_bf16(o[i][t], a, pf[t][0], pf[t][1]);
          }
        }
      }
      __syncwarp();  // every lane has read the stage before it is loaded again
      slot_out = slot_out + 1 == C::STAGES ? 0 : slot_out + 1;
    }

    // ---- join the four warps
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], x);
        if (n == 0) ml_smem[warp * C::ROWS + 8 * t + 2 * j + e] = make_float2(m[t][e], l[t][e]);
      }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = 8 * t + 2 * j + e;
        float mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < kDecodeWarps; ++w) mx = fmaxf(mx, ml_smem[w * C::ROWS + r].x);
        const float f = m[t][e] == mx ? 1.f : ex2_approx(m[t][e] - mx);
        float* dst = merge + (warp * C::ROWS + r) * C::O_LD;
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) {
          const int d0 = FMT == KV_BF16 ? 16 * i + n : n * (HD / 8) + 2 * i;
          const int d1 = FMT == KV_BF16 ? d0 + 8 : d0 + 1;
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
      for (int w = 0; w < kDecodeWarps; ++w) mx = fmaxf(mx, ml_smem[w * C::ROWS + r].x);
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kDecodeWarps; ++w) {
        const float2 q = ml_smem[w * C::ROWS + r];
        sum += q.x == mx ? q.y : q.y * ex2_approx(q.x - mx);
        const float4 v = *reinterpret_cast<const float4*>(merge + (w * C::ROWS + r) * C::O_LD + d);
        a.x += v.x;
        a.y += v.y;
        a.z += v.z;
        a.w += v.w;
      }
      if (whole) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        __nv_bfloat16* dst = p.out + (long long)(it.seq.q0 + tok0 + r / p.group) * p.o_stride_t +
                             (long long)(it.kvh * p.group + r % p.group) * p.o_stride_h + d;
        *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(a.x * inv, a.y * inv), pack_bf16(a.z * inv, a.w * inv));
      } else {
        *reinterpret_cast<float4*>(ws.o + ((size_t)slot * C::ROWS + r) * HD + d) = a;
        if (d == 0) ws.ml[(size_t)slot * C::ROWS + r] = make_float2(mx, sum);
      }
    }
    if (u == u_end) break;
    next_item(it, p.seqs, shape);
    __syncthreads();  // the merge buffers are free
  }
  cp_async_wait<0>();
}

// Joins the parts of items that lie in more than one block's range.  Block x + 1 of the attention kernel
// starts inside an item, or does not; the first block that does joins the item.  WARPS_PER_ROW warps share
// the parts of a row; ROWS rows per part.
template <int HD, int ROWS, int WARPS_PER_ROW>
__global__ void __launch_bounds__(128)
    paged_join_kernel(const __grid_constant__ PagedAttnParams p, PagedShape shape, PagedWorkspace ws) {
  pdl_wait_and_release();
  constexpr int ROWS_AT_ONCE = 4 / WARPS_PER_ROW;
  constexpr int V = HD / 32;  // columns per lane
  const long long total = ws.total[0];
  const int blocks = (int)ws.total[1];
  const int c = blockIdx.x + 1;
  if (c >= blocks) return;
  const long long u = range_begin(c, total, blocks);
  const PagedRecord rec = ws.records[c];
  if (rec.start == u) return;                                     // no item is cut here
  if (range_begin(c - 1, total, blocks) > rec.start) return;      // cut before as well: another block's
  const int last = block_of_unit(rec.start + rec.n_units - 1, total, blocks);
  const int first_slot = 2 * (c - 1) + (range_begin(c - 1, total, blocks) == rec.start ? 0 : 1);
  const int parts = last - (c - 1) + 1;
  auto slot = [&](int i) { return i == 0 ? first_slot : 2 * (c - 1 + i); };
  const SeqInfo seq = seq_info(p.seqs, rec.b);
  const int tok0 = rec.rt * shape.tile_tokens;
  const int rows = min(shape.tile_tokens, seq.qn - tok0) * p.group;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = warp % WARPS_PER_ROW;
  __shared__ float part[4][HD];
  __shared__ float part_l[4];
  for (int r0 = blockIdx.y * ROWS_AT_ONCE; r0 < rows; r0 += gridDim.y * ROWS_AT_ONCE) {
    const int r = r0 + warp / WARPS_PER_ROW;
    const bool live = r < rows;
    float mx = -INFINITY;
    if (live)
      for (int i = lane; i < parts; i += 32) mx = fmaxf(mx, ws.ml[(size_t)slot(i) * ROWS + r].x);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
    float acc[V], l = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = 0.f;
    if (live) {
#pragma unroll 4
      for (int i = sub; i < parts; i += WARPS_PER_ROW) {
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
    if (live && sub == 0) {
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
template <int FMT, int HD, int NT>
int decode_blocks() {
  using C = DecodeCfg<FMT, HD, NT>;
  static std::atomic<int> cached[64];
  int dev = 0;
  B200_CUDA_CHECK(cudaGetDevice(&dev));
  B200_CHECK(dev >= 0 && dev < 64, "device index out of range");
  int n = cached[dev].load(std::memory_order_acquire);
  if (n == 0) {
    auto* kernel = paged_decode_kernel<FMT, HD, NT>;
    B200_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    int per_sm = 0;
    B200_CUDA_CHECK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, kDecodeThreads, C::SMEM));
    B200_CHECK(per_sm > 0, "paged attention: the kernel does not fit an SM");
    n = per_sm * num_sms_cached();
    cached[dev].store(n, std::memory_order_release);
  }
  return n;
}

template <int FMT, int HD, int NT>
void launch_decode(const PagedAttnParams& p, const PagedAlloc& alloc, cudaStream_t s) {
  using C = DecodeCfg<FMT, HD, NT>;
  const int blocks = decode_blocks<FMT, HD, NT>();
  const PagedWorkspace ws = paged_workspace(alloc(paged_workspace_bytes(blocks, C::ROWS, HD)), blocks, C::ROWS);
  const PagedShape shape{std::max(1, C::ROWS / p.group), kUnitLog2, p.pool.kv_heads};
  launch_k(paged_decode_kernel<FMT, HD, NT>, dim3(blocks), dim3(kDecodeThreads), C::SMEM, s, 1, p, shape, ws);
  launch_k(paged_join_kernel<HD, C::ROWS, 4>, dim3(blocks - 1, C::ROWS), dim3(128), 0, s, 1, p, shape, ws);
  B200_CUDA_CHECK(cudaGetLastError());
  count_launch(2);
}

template <int FMT, int HD>
void launch_rows(const PagedAttnParams& p, const PagedAlloc& alloc, cudaStream_t s) {
  const long long rows = (long long)p.seqs.max_q * p.group;
  if (rows <= 8)
    launch_decode<FMT, HD, 1>(p, alloc, s);
  else if (rows <= 16)
    launch_decode<FMT, HD, 2>(p, alloc, s);
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
