// Writing new tokens into a paged key/value cache (quantising them on the way) and reading them back.
//
// A row is one head of one token's K or V: head_dim bf16 values.  Quantised, with a = max|x| over the row
// and M the format's largest code: scale = a / M, code = round(x M / a), half to even.  Rows that are all
// zero get scale 0 and zero codes; rows with an infinity or a NaN get scale NaN and zero codes, so that
// they read back as NaN instead of as some finite value.
//
// The quotient is formed from n = x M (exact: 8 x 9 bits) as q0 = n r, r ~ 1/a, followed by one exact
// remainder step q = q0 + r (n - q0 a), whose error is below 2^-20 of q0's last bit: bf16 inputs that fall
// exactly between two codes come out exactly so, and no other quotient is closer than 2^-17 to a tie.  The scale
// a / M is rounded correctly in the same way.
//
// A warp takes K or V of a run of tokens.  Where the tokens lie is found by its lanes at once, one token each
// (a search over q_starts, the sequence's length, its page), and handed round; then 32 lanes x 16 bytes per
// access walk over (token, head, columns), four accesses in flight.  Bound by HBM for many tokens, by latency
// for a decode step.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "paged.h"

namespace b200 {

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ void unpack8(const uint4& q, float (&f)[8]) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = bf16lo(w[i]);
    f[2 * i + 1] = bf16hi(w[i]);
  }
}

// Where token t lies: index of its (page, head 0, offset) cell.  kNoPlace: before its sequence's first token,
// or in a page that does not exist; kNoSequence: a row of no sequence.
constexpr long long kNoPlace = -1, kNoSequence = -2;
__device__ __forceinline__ long long place_of(const PagedSeqs& s, int t, int kv_heads, DeviceErrors* errs) {
  const int b = seq_of_row(s, t);
  if (b < 0) return kNoSequence;
  const SeqInfo q = seq_info(s, b);
  if (!q.ok || t < q.q0 || t >= q.q0 + q.qn) {
    report_error(errs, kErrBadIndex, b);
    return kNoSequence;
  }
  const int pos = q.len - q.qn + (t - q.q0);
  if (pos < 0) return kNoPlace;
  const int page = s.table[(long long)b * s.table_stride + (pos >> s.page_log2)];
  if (page < 0 || page >= s.n_pages) {
    report_error(errs, kErrBadIndex, b);
    return kNoPlace;
  }
  return ((long long)page * kv_heads << s.page_log2) + (pos & ((1 << s.page_log2) - 1));
}

// A warp's run of tokens, and the walk over its 16-byte pieces: piece i is column group i % LANES of head
// i / LANES; `passes` accesses of 32 pieces cover a token.
struct TokenRun {
  int t0, count;
  bool is_v;
  long long place;  // lane l: of token t0 + l
};
__device__ __forceinline__ TokenRun token_run(const PagedSeqs& s, int kv_heads, int per_warp, DeviceErrors* errs) {
  const int w = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  TokenRun r;
  r.is_v = w & 1;
  const long long t0 = (long long)(w >> 1) * per_warp;
  r.count = (int)max(0ll, min((long long)per_warp, s.total_q - t0));
  r.t0 = (int)min(t0, (long long)s.total_q);
  // K's warp reports what is wrong, V's finds the same
  r.place = lane < r.count ? place_of(s, r.t0 + lane, kv_heads, r.is_v ? nullptr : errs) : kNoSequence;
  return r;
}
constexpr int kInFlight = 4;

template <int FMT, int LANES>
__global__ void __launch_bounds__(kThreads)
    kv_write_kernel(PagedSeqs seqs, KvPool pool, const __nv_bfloat16* __restrict__ k,
                    const __nv_bfloat16* __restrict__ v, long long k_stride_t, long long k_stride_h,
                    long long v_stride_t, long long v_stride_h, int per_warp, DeviceErrors* errs) {
  pdl_wait_and_release();
  constexpr int HD = LANES * 8;
  const int lane = threadIdx.x & 31, sub = lane % LANES;
  const TokenRun run = token_run(seqs, pool.kv_heads, per_warp, errs);
  const __nv_bfloat16* src = run.is_v ? v : k;
  const long long stride_t = run.is_v ? v_stride_t : k_stride_t, stride_h = run.is_v ? v_stride_h : k_stride_h;
  uint8_t* dst = reinterpret_cast<uint8_t*>(run.is_v ? pool.v : pool.k);
  float* scales = run.is_v ? pool.v_scale : pool.k_scale;
  constexpr int HEADS = 32 / LANES;  // per access
  const int passes = (pool.kv_heads + HEADS - 1) / HEADS;
  const int total = run.count * passes;
  // source of this lane's piece of the access, advanced from access to access
  const __nv_bfloat16* from = src + run.t0 * stride_t + (lane / LANES) * stride_h + sub * 8;
  const long long next_pass = HEADS * stride_h, next_token = stride_t - passes * next_pass;
  int tok = 0, pass = 0;
  for (int i0 = 0; i0 < total; i0 += kInFlight) {
    uint4 x[kInFlight];
    long long cell[kInFlight];
#pragma unroll
    for (int i = 0; i < kInFlight; ++i) {
      x[i] = make_uint4(0u, 0u, 0u, 0u);
      const long long place = __shfl_sync(0xffffffffu, run.place, tok & 31);
      const int h = pass * HEADS + lane / LANES;
      cell[i] = -1;
      if (i0 + i < total && place >= 0 && h < pool.kv_heads &&
          B200_IN_BOUNDS(errs, run.t0 + tok, 1, seqs.total_q, 130) &&
          B200_IN_BOUNDS(errs, place + (h << seqs.page_log2), 1, pool_cells(seqs, pool.kv_heads), 131)) {
        cell[i] = place + (h << seqs.page_log2);
        x[i] = *reinterpret_cast<const uint4*>(from);
      }
      from += next_pass;
      if (++pass == passes) pass = 0, ++tok, from += next_token;
    }
#pragma unroll
    for (int i = 0; i < kInFlight; ++i) {
      if constexpr (FMT == KV_BF16) {
        if (cell[i] >= 0) *reinterpret_cast<uint4*>(dst + cell[i] * (2 * HD) + sub * 16) = x[i];
      } else {
        // max|x| as integers: magnitudes order like their bit patterns, infinities and NaN above all others
        const uint32_t m2 = __vmaxu2(__vmaxu2(x[i].x & 0x7FFF7FFFu, x[i].y & 0x7FFF7FFFu),
                                     __vmaxu2(x[i].z & 0x7FFF7FFFu, x[i].w & 0x7FFF7FFFu));
        uint32_t m = max(m2 & 0xFFFFu, m2 >> 16);
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float a = __uint_as_float(m << 16);
        const bool finite = m < 0x7F80u;
        // a power of two that brings a near 1, so that neither n nor r leaves the normal range
        const float unit = __uint_as_float((uint32_t)min(max(254 - (int)(m >> 7), 1), 240) << 23);
        const float au = a * unit, um = unit * kv_code_max(FMT);
        const float r = m > 0u ? __fdividef(1.0f, au) : 0.0f;
        float f[8];
        unpack8(x[i], f);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float n = f[e] * um;
          const float q0 = n * r;
          f[e] = fmaf(fmaf(-q0, au, n), r, q0);
        }
        uint32_t w[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if constexpr (FMT == KV_E4M3) {
            const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(f[4 * h], f[4 * h + 1]), __NV_SATFINITE, __NV_E4M3);
            const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(f[4 * h + 2], f[4 * h + 3]), __NV_SATFINITE, __NV_E4M3);
            w[h] = lo | (hi << 16);
          } else {
            // rounded by adding 1.5 * 2^23, whose low byte is then the code
            uint32_t c[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) c[e] = __float_as_uint(f[4 * h + e] + 12582912.0f);
            w[h] = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
          }
          if (!finite) w[h] = 0u;
        }
        if (cell[i] >= 0) {
          *reinterpret_cast<uint2*>(dst + cell[i] * HD + sub * 8) = make_uint2(w[0], w[1]);
          if (sub == 0) {
            constexpr float M = kv_code_max(FMT), inv = 1.0f / M;
            const float s0 = a * inv;
            scales[cell[i]] = finite ? fmaf(fmaf(-s0, M, a), inv, s0) : __int_as_float(0x7FC00000);
          }
        }
      }
    }
  }
}

template <int FMT, int LANES, bool F32>
__global__ void __launch_bounds__(kThreads)
    kv_read_kernel(PagedSeqs seqs, KvPool pool, void* __restrict__ k, void* __restrict__ v, int per_warp,
                   DeviceErrors* errs) {
  pdl_wait_and_release();
  constexpr int HD = LANES * 8;
  const int lane = threadIdx.x & 31, sub = lane % LANES;
  const TokenRun run = token_run(seqs, pool.kv_heads, per_warp, errs);
  const uint8_t* src = reinterpret_cast<const uint8_t*>(run.is_v ? pool.v : pool.k);
  const float* scales = run.is_v ? pool.v_scale : pool.k_scale;
  void* out = run.is_v ? v : k;
  constexpr int HEADS = 32 / LANES;
  const int passes = (pool.kv_heads + HEADS - 1) / HEADS;
  int tok = 0, pass = 0;
  const int total = run.count * passes;
  for (int i0 = 0; i0 < total; i0 += kInFlight) {
    uint4 x[kInFlight];
    float sc[kInFlight];
    long long at[kInFlight];  // piece of the output, -1: none
#pragma unroll
    for (int i = 0; i < kInFlight; ++i) {
      x[i] = make_uint4(0u, 0u, 0u, 0u);  // a token before the sequence's first reads as zeros
      sc[i] = 0.f;
      at[i] = -1;
      const long long place = __shfl_sync(0xffffffffu, run.place, tok & 31);
      const int h = pass * HEADS + lane / LANES;
      if (i0 + i < total && place != kNoSequence && h < pool.kv_heads &&
          B200_IN_BOUNDS(errs, run.t0 + tok, 1, seqs.total_q, 132)) {
        at[i] = ((long long)(run.t0 + tok) * pool.kv_heads + h) * HD + sub * 8;
        const long long cell = place + ((long long)h << seqs.page_log2);
        if (place >= 0 && B200_IN_BOUNDS(errs, cell, 1, pool_cells(seqs, pool.kv_heads), 133)) {
          if constexpr (FMT == KV_BF16) {
            x[i] = *reinterpret_cast<const uint4*>(src + cell * (2 * HD) + sub * 16);
          } else {
            const uint2 c = *reinterpret_cast<const uint2*>(src + cell * HD + sub * 8);
            x[i].x = c.x;
            x[i].y = c.y;
            sc[i] = scales[cell];
          }
        }
      }
      if (++pass == passes) pass = 0, ++tok;
    }
#pragma unroll
    for (int i = 0; i < kInFlight; ++i) {
      float f[8];
      if constexpr (FMT == KV_BF16) {
        unpack8(x[i], f);
      } else {
        const uint32_t w[2] = {x[i].x, x[i].y};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if constexpr (FMT == KV_E4M3) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const __half2_raw raw =
                  __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)((w[h] >> (16 * e)) & 0xFFFFu), __NV_E4M3);
              const float2 c = __half22float2(*reinterpret_cast<const __half2*>(&raw));
              f[4 * h + 2 * e] = c.x;
              f[4 * h + 2 * e + 1] = c.y;
            }
          } else {
            // code + 128 as the low bits of 2^23, exactly; then 2^23 + 128 is taken off
            const uint32_t c = w[h] ^ 0x80808080u;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              f[4 * h + e] = __uint_as_float(__byte_perm(c, 0x4B000000u, 0x7440 + e)) - 8388736.0f;
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] *= sc[i];
      }
      if constexpr (F32) {
        // two lanes hold 64 bytes; they swap 16 so that each of their stores fills a 32-byte sector
        const bool odd = lane & 1;
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = __shfl_xor_sync(0xffffffffu, odd ? f[e] : f[4 + e], 1);
        if (at[i] >= 0) {
          float* dst = reinterpret_cast<float*>(out) + at[i];
          *reinterpret_cast<float4*>(odd ? dst - 4 : dst) =
              odd ? make_float4(x[0], x[1], x[2], x[3]) : make_float4(f[0], f[1], f[2], f[3]);
          *reinterpret_cast<float4*>(odd ? dst + 4 : dst + 8) =
              odd ? make_float4(f[4], f[5], f[6], f[7]) : make_float4(x[0], x[1], x[2], x[3]);
        }
      } else if (at[i] >= 0) {
        uint4 q;
        q.x = pack_bf16(f[0], f[1]);
        q.y = pack_bf16(f[2], f[3]);
        q.z = pack_bf16(f[4], f[5]);
        q.w = pack_bf16(f[6], f[7]);
        *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(out) + at[i]) = q;
      }
    }
  }
}

// Tokens per warp: one while the tokens do not fill the device, then more, to share the search for places.
int tokens_per_warp(const PagedSeqs& q) {
  const long long warps = (long long)num_sms_cached() * 64;  // resident at once
  return (int)std::min<long long>(8, std::max<long long>(1, 2ll * q.total_q / warps));
}
dim3 grid_for_tokens(const PagedSeqs& q, int per_warp) {
  const long long runs = ((long long)q.total_q + per_warp - 1) / per_warp * 2;
  return dim3((unsigned)((runs + kThreads / 32 - 1) / (kThreads / 32)));
}

template <int FMT>
void launch_write(const PagedSeqs& q, const KvPool& p, const __nv_bfloat16* k, const __nv_bfloat16* v, long long kt,
                  long long kh, long long vt, long long vh, cudaStream_t s) {
  const int n = tokens_per_warp(q);
  if (p.head_dim == 64)
    launch_k(kv_write_kernel<FMT, 8>, grid_for_tokens(q, n), dim3(kThreads), 0, s, 1, q, p, k, v, kt, kh, vt, vh, n,
             device_errors_ptr());
  else
    launch_k(kv_write_kernel<FMT, 16>, grid_for_tokens(q, n), dim3(kThreads), 0, s, 1, q, p, k, v, kt, kh, vt, vh, n,
             device_errors_ptr());
}

template <int FMT, bool F32>
void launch_read(const PagedSeqs& q, const KvPool& p, void* k, void* v, cudaStream_t s) {
  const int n = tokens_per_warp(q);
  if (p.head_dim == 64)
    launch_k(kv_read_kernel<FMT, 8, F32>, grid_for_tokens(q, n), dim3(kThreads), 0, s, 1, q, p, k, v, n,
             device_errors_ptr());
  else
    launch_k(kv_read_kernel<FMT, 16, F32>, grid_for_tokens(q, n), dim3(kThreads), 0, s, 1, q, p, k, v, n,
             device_errors_ptr());
}

}  // namespace

void kv_cache_write(const PagedSeqs& q, const KvPool& p, const __nv_bfloat16* k, const __nv_bfloat16* v, long long kt,
                    long long kh, long long vt, long long vh, cudaStream_t s) {
  if (q.total_q == 0 || q.batch == 0) return;
  switch (p.fmt) {
    case KV_E4M3: launch_write<KV_E4M3>(q, p, k, v, kt, kh, vt, vh, s); break;
    case KV_INT8: launch_write<KV_INT8>(q, p, k, v, kt, kh, vt, vh, s); break;
    default: launch_write<KV_BF16>(q, p, k, v, kt, kh, vt, vh, s); break;
  }
  B200_CUDA_CHECK(cudaGetLastError());
  count_launch();
}

void kv_cache_read(const PagedSeqs& q, const KvPool& p, void* k, void* v, bool out_f32, cudaStream_t s) {
  if (q.total_q == 0 || q.batch == 0) return;
  switch (p.fmt) {
    case KV_E4M3: out_f32 ? launch_read<KV_E4M3, true>(q, p, k, v, s) : launch_read<KV_E4M3, false>(q, p, k, v, s); break;
    case KV_INT8: out_f32 ? launch_read<KV_INT8, true>(q, p, k, v, s) : launch_read<KV_INT8, false>(q, p, k, v, s); break;
    default: out_f32 ? launch_read<KV_BF16, true>(q, p, k, v, s) : launch_read<KV_BF16, false>(q, p, k, v, s); break;
  }
  B200_CUDA_CHECK(cudaGetLastError());
  count_launch();
}

}  // namespace b200
