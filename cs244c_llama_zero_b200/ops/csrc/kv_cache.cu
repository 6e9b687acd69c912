// Writing new tokens into a paged key/value cache (quantising them on the way) and reading them back.
//
// A row is one head of one token's K or V: head_dim bf16 values.  Quantised, with a = max|x| over the row
// and M the format's largest code: scale = a / M, code = round(x M / a), half to even.  Rows that are all
// zero get scale 0 and zero codes; rows with an infinity or a NaN get scale NaN and zero codes, so that
// they read back as NaN instead of as some finite value.
//
// The quotient is formed from n = x M (exact: 8 x 9 bits) as q0 = n r, r = 1/a, followed by one exact
// remainder step q = q0 + r (n - q0 a), which returns the correctly rounded quotient: bf16 inputs that fall
// exactly between two codes do so in fp32 too, and no other quotient comes closer than 2^-17 to a tie.
//
// Both kernels move 16 bytes per lane on the bf16 side (head_dim / 8 lanes per row) and are bound by HBM.
#include <cuda_bf16.h>
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

// Where row (token t, head h) lies in the pool: index of its (page, head, offset) cell, -1 for none.
__device__ __forceinline__ long long cell_of(const PagedSeqs& s, int t, int h, int kv_heads, DeviceErrors* errs,
                                             bool* behind) {
  *behind = false;
  const int b = seq_of_row(s, t);
  if (b < 0) {  // the row belongs to no sequence
    *behind = true;
    return -1;
  }
  const SeqInfo q = seq_info(s, b);
  if (!q.ok || t < q.q0 || t >= q.q0 + q.qn) {
    report_error(errs, kErrBadIndex, b);
    *behind = true;
    return -1;
  }
  const int pos = q.len - q.qn + (t - q.q0);
  if (pos < 0) return -1;
  const int page = s.table[(long long)b * s.table_stride + (pos >> s.page_log2)];
  if (page < 0 || page >= s.n_pages) {
    report_error(errs, kErrBadIndex, b);
    return -1;
  }
  return (((long long)page * kv_heads + h) << s.page_log2) + (pos & ((1 << s.page_log2) - 1));
}

// LANES = head_dim / 8 lanes per row; rows are numbered (token, K or V, head).
template <int FMT, int LANES>
__global__ void __launch_bounds__(kThreads)
    kv_write_kernel(PagedSeqs seqs, KvPool pool, const __nv_bfloat16* __restrict__ k,
                    const __nv_bfloat16* __restrict__ v, long long k_stride_t, long long k_stride_h,
                    long long v_stride_t, long long v_stride_h, DeviceErrors* errs) {
  pdl_wait_and_release();
  constexpr int HD = LANES * 8;
  const int sub = threadIdx.x % LANES;
  const long long rows = (long long)seqs.total_q * 2 * pool.kv_heads;
  const long long step = (long long)gridDim.x * (kThreads / LANES);
  for (long long r0 = (long long)blockIdx.x * (kThreads / LANES); r0 < rows; r0 += step) {
    const long long r = r0 + threadIdx.x / LANES;
    const bool live = r < rows;
    const int t = live ? (int)(r / (2 * pool.kv_heads)) : 0;
    const int wh = live ? (int)(r % (2 * pool.kv_heads)) : 0;
    const bool is_v = wh >= pool.kv_heads;
    const int h = is_v ? wh - pool.kv_heads : wh;
    const __nv_bfloat16* src = is_v ? v + t * v_stride_t + h * v_stride_h : k + t * k_stride_t + h * k_stride_h;
    uint4 x = make_uint4(0u, 0u, 0u, 0u);
    long long cell = -1;
    if (live) {
      x = *reinterpret_cast<const uint4*>(src + sub * 8);
      bool behind;
      cell = cell_of(seqs, t, h, pool.kv_heads, sub == 0 ? errs : nullptr, &behind);
    }
    void* dst = is_v ? pool.v : pool.k;
    if constexpr (FMT == KV_BF16) {
      if (cell >= 0) *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(dst) + cell * HD + sub * 8) = x;
    } else {
      // max|x| as integers: magnitudes order like their bit patterns, infinities and NaN above all others
      const uint32_t m2 = __vmaxu2(__vmaxu2(x.x & 0x7FFF7FFFu, x.y & 0x7FFF7FFFu),
                                   __vmaxu2(x.z & 0x7FFF7FFFu, x.w & 0x7FFF7FFFu));
      uint32_t m = max(m2 & 0xFFFFu, m2 >> 16);
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
      const float a = __uint_as_float(m << 16);
      const bool finite = m < 0x7F80u;
      // a power of two that brings a near 1, so that neither n nor r leaves the normal range
      const float unit = __uint_as_float((uint32_t)min(max(254 - (int)(m >> 7), 1), 240) << 23);
      const float r = (finite && m > 0u) ? __frcp_rn(a * unit) : 0.0f;
      const float um = unit * kv_code_max(FMT);
      float f[8];
      unpack8(x, f);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float n = finite ? f[e] * um : 0.0f;
        const float q0 = n * r;
        f[e] = finite ? fmaf(fmaf(-q0, a * unit, n), r, q0) : 0.0f;
      }
      uint32_t w[2];
      if constexpr (FMT == KV_E4M3) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(f[4 * i], f[4 * i + 1]), __NV_SATFINITE, __NV_E4M3);
          const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(f[4 * i + 2], f[4 * i + 3]), __NV_SATFINITE, __NV_E4M3);
          w[i] = lo | (hi << 16);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          w[i] = 0u;
#pragma unroll
          for (int e = 0; e < 4; ++e) w[i] |= ((uint32_t)__float2int_rn(f[4 * i + e]) & 0xFFu) << (8 * e);
        }
      }
      if (cell >= 0) {
        *reinterpret_cast<uint2*>(reinterpret_cast<uint8_t*>(dst) + cell * HD + sub * 8) = make_uint2(w[0], w[1]);
        if (sub == 0) (is_v ? pool.v_scale : pool.k_scale)[cell] = finite ? a / kv_code_max(FMT) : __int_as_float(0x7FC00000);
      }
    }
  }
}

template <int FMT, int LANES, bool F32>
__global__ void __launch_bounds__(kThreads)
    kv_read_kernel(PagedSeqs seqs, KvPool pool, void* __restrict__ k, void* __restrict__ v, DeviceErrors* errs) {
  pdl_wait_and_release();
  constexpr int HD = LANES * 8;
  const int sub = threadIdx.x % LANES;
  const long long rows = (long long)seqs.total_q * 2 * pool.kv_heads;
  const long long step = (long long)gridDim.x * (kThreads / LANES);
  for (long long r = (long long)blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES; r < rows; r += step) {
    const int t = (int)(r / (2 * pool.kv_heads));
    const int wh = (int)(r % (2 * pool.kv_heads));
    const bool is_v = wh >= pool.kv_heads;
    const int h = is_v ? wh - pool.kv_heads : wh;
    bool behind;
    const long long cell = cell_of(seqs, t, h, pool.kv_heads, sub == 0 ? errs : nullptr, &behind);
    if (behind) continue;
    float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};  // a token before the sequence's first reads as zeros
    if (cell >= 0) {
      const void* src = is_v ? pool.v : pool.k;
      if constexpr (FMT == KV_BF16) {
        unpack8(*reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(src) + cell * HD + sub * 8), f);
      } else {
        const uint2 w2 = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint8_t*>(src) + cell * HD + sub * 8);
        const float s = (is_v ? pool.v_scale : pool.k_scale)[cell];
        const uint32_t w[2] = {w2.x, w2.y};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t c = (w[e >> 2] >> (8 * (e & 3))) & 0xFFu;
          if constexpr (FMT == KV_E4M3) {
            __nv_fp8_e4m3 c8;
            c8.__x = (__nv_fp8_storage_t)c;
            f[e] = (float)c8 * s;
          } else {
            f[e] = (float)(int8_t)c * s;
          }
        }
      }
    }
    const long long o = ((long long)t * pool.kv_heads + h) * HD + sub * 8;
    if constexpr (F32) {
      float4* dst = reinterpret_cast<float4*>(reinterpret_cast<float*>(is_v ? v : k) + o);
      dst[0] = make_float4(f[0], f[1], f[2], f[3]);
      dst[1] = make_float4(f[4], f[5], f[6], f[7]);
    } else {
      uint4 q;
      q.x = pack_bf16(f[0], f[1]);
      q.y = pack_bf16(f[2], f[3]);
      q.z = pack_bf16(f[4], f[5]);
      q.w = pack_bf16(f[6], f[7]);
      *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(is_v ? v : k) + o) = q;
    }
  }
}

int grid_for_rows(long long rows, int lanes) {
  const long long per = kThreads / lanes;
  return (int)std::max<long long>(1, std::min<long long>((rows + per - 1) / per, (long long)num_sms_cached() * 32));
}

template <int FMT>
void launch_write(const PagedSeqs& q, const KvPool& p, const __nv_bfloat16* k, const __nv_bfloat16* v, long long kt,
                  long long kh, long long vt, long long vh, cudaStream_t s) {
  const long long rows = (long long)q.total_q * 2 * p.kv_heads;
  if (p.head_dim == 64)
    launch_k(kv_write_kernel<FMT, 8>, dim3(grid_for_rows(rows, 8)), dim3(kThreads), 0, s, 1, q, p, k, v, kt, kh, vt,
             vh, device_errors_ptr());
  else
    launch_k(kv_write_kernel<FMT, 16>, dim3(grid_for_rows(rows, 16)), dim3(kThreads), 0, s, 1, q, p, k, v, kt, kh, vt,
             vh, device_errors_ptr());
}

template <int FMT, bool F32>
void launch_read(const PagedSeqs& q, const KvPool& p, void* k, void* v, cudaStream_t s) {
  const long long rows = (long long)q.total_q * 2 * p.kv_heads;
  if (p.head_dim == 64)
    launch_k(kv_read_kernel<FMT, 8, F32>, dim3(grid_for_rows(rows, 8)), dim3(kThreads), 0, s, 1, q, p, k, v,
             device_errors_ptr());
  else
    launch_k(kv_read_kernel<FMT, 16, F32>, dim3(grid_for_rows(rows, 16)), dim3(kThreads), 0, s, 1, q, p, k, v,
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
