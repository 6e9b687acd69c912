// Attention of new tokens over a paged key/value cache (causal, grouped heads, ragged batch).
//
// Row i of a sequence with q_len new of kv_len cached tokens stands at position p = kv_len - q_len + i:
//   o = sum_{j <= p} softmax_j(scale * q . k_j) v_j      (p < 0: zeros)
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "paged.h"

namespace b200 {

namespace {

constexpr float kLog2e = 1.4426950408889634f;

template <int FMT>
__device__ __forceinline__ float load_code(const void* base, long long idx) {
  if constexpr (FMT == KV_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(base)[idx]);
  if constexpr (FMT == KV_E4M3) return (float)reinterpret_cast<const __nv_fp8_e4m3*>(base)[idx];
  return (float)reinterpret_cast<const int8_t*>(base)[idx];
}

// One warp per (row, head): lane l holds columns l, l + 32, ...
template <int FMT, int HD>
__global__ void __launch_bounds__(256) paged_attn_simple_kernel(PagedAttnParams p) {
  pdl_wait_and_release();
  constexpr int N = HD / 32;
  const int lane = threadIdx.x & 31;
  const long long w = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (w >= (long long)p.seqs.total_q * p.heads) return;
  const int t = (int)(w / p.heads), h = (int)(w % p.heads);
  const int b = seq_of_row(p.seqs, t);
  if (b < 0) return;
  const SeqInfo si = seq_info(p.seqs, b);
  if (!si.ok || t < si.q0 || t >= si.q0 + si.qn) {
    if (lane == 0) report_error(p.errs, kErrBadIndex, b);
    return;
  }
  const int pos = si.len - si.qn + (t - si.q0);
  const int kvh = h / p.group;
  float q[N], o[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    q[i] = __bfloat162float(p.q[t * p.q_stride_t + h * p.q_stride_h + lane + 32 * i]) * p.scale * kLog2e;
    o[i] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int j = 0; j <= pos; ++j) {
    const int page = p.seqs.table[(long long)b * p.seqs.table_stride + (j >> p.seqs.page_log2)];
    if (page < 0 || page >= p.seqs.n_pages) {
      if (lane == 0) report_error(p.errs, kErrBadIndex, b);
      continue;
    }
    const long long cell = (((long long)page * p.pool.kv_heads + kvh) << p.seqs.page_log2) +
                           (j & ((1 << p.seqs.page_log2) - 1));
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) s += q[i] * load_code<FMT>(p.pool.k, cell * HD + lane + 32 * i);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    if (FMT != KV_BF16) s *= p.pool.k_scale[cell];
    const float m_new = fmaxf(m, s);
    const float alpha = m == m_new ? 1.f : exp2f(m - m_new);
    const float pr = exp2f(s - m_new);
    const float pv = FMT != KV_BF16 ? pr * p.pool.v_scale[cell] : pr;
    l = l * alpha + pr;
    m = m_new;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = o[i] * alpha + pv * load_code<FMT>(p.pool.v, cell * HD + lane + 32 * i);
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
#pragma unroll
  for (int i = 0; i < N; ++i)
    p.out[t * p.o_stride_t + h * p.o_stride_h + lane + 32 * i] = __float2bfloat16_rn(o[i] * inv);
}

template <int FMT>
void launch_simple(const PagedAttnParams& p, cudaStream_t s) {
  const long long warps = (long long)p.seqs.total_q * p.heads;
  const dim3 grid((unsigned)((warps + 7) / 8));
  if (p.pool.head_dim == 64)
    launch_k(paged_attn_simple_kernel<FMT, 64>, grid, dim3(256), 0, s, 1, p);
  else
    launch_k(paged_attn_simple_kernel<FMT, 128>, grid, dim3(256), 0, s, 1, p);
}

}  // namespace

void paged_attention(const PagedAttnParams& p_in, cudaStream_t s) {
  PagedAttnParams p = p_in;
  if (p.seqs.total_q == 0 || p.seqs.batch == 0) return;
  p.errs = device_errors_ptr();
  switch (p.pool.fmt) {
    case KV_E4M3: launch_simple<KV_E4M3>(p, s); break;
    case KV_INT8: launch_simple<KV_INT8>(p, s); break;
    default: launch_simple<KV_BF16>(p, s); break;
  }
  B200_CUDA_CHECK(cudaGetLastError());
  count_launch();
}

}  // namespace b200
