// Adjusting next-token logits: penalties for tokens that occurred, additive biases, a bitmask of allowed
// tokens.  For row b, with seen(t) <=> t in history[b, :len] and n(t) = count of t in history[b, prompt:len]:
//   l = seen ? (l > 0 ? l / repetition : l * repetition) : l
//   l = l - (frequency * n + presence * (n > 0)) + bias[t];   not allowed: -inf
// computed in fp32 and rounded once to the logits' type.
//
// A block owns a run of SPAN tokens of one row.  It counts the history's tokens that fall into its run in
// shared memory (bit 31: seen, bits 0..30: n), then streams the run through registers: one pass over the
// logits, 16 bytes per thread and access, issued before the counting so that both latencies overlap.
// Bound by HBM; the history is re-read by each of a row's blocks and comes from L2.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "paged.h"

namespace b200 {

namespace {

constexpr int kThreads = 256;

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }

template <typename T>
struct alignas(16) Vec {
  T e[16 / sizeof(T)];
};

// Rows start anywhere: a run is counted in 16-byte groups of the row's memory, `shift` elements of the
// first group belonging to what lies before the row.  Groups that the row does not fill, and all groups
// when input and output are aligned differently, go element by element.
template <typename T, int NV>
__global__ void __launch_bounds__(kThreads) adjust_logits_kernel(LogitsParams p, unsigned runs) {
  pdl_wait_and_release();
  constexpr int VE = 16 / (int)sizeof(T);
  constexpr int SPAN = kThreads * NV * VE;
  __shared__ uint32_t counts[SPAN];
  const int row = (int)(blockIdx.x / runs), run = (int)(blockIdx.x % runs);
  const T* src = reinterpret_cast<const T*>(p.logits) + row * p.stride;
  T* dst = reinterpret_cast<T*>(p.out) + row * p.out_stride;
  const int shift = (int)((reinterpret_cast<uintptr_t>(src) & 15) / sizeof(T));
  const bool same = shift == (int)((reinterpret_cast<uintptr_t>(dst) & 15) / sizeof(T));
  const int first = run * SPAN - shift;  // token of the run's element 0 (may be negative)
  if (first >= p.vocab) return;

  Vec<T> x[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int t0 = first + (i * kThreads + threadIdx.x) * VE;
    if (t0 >= 0 && t0 + VE <= p.vocab) {
      x[i] = *reinterpret_cast<const Vec<T>*>(src + t0);
    } else {
#pragma unroll
      for (int e = 0; e < VE; ++e)
        if (t0 + e >= 0 && t0 + e < p.vocab) x[i].e[e] = src[t0 + e];
    }
  }

  const bool penalise = p.history != nullptr;
  float rep = 1.f, freq = 0.f, pres = 0.f;
  if (penalise) {
    for (int i = threadIdx.x; i < SPAN / 4; i += kThreads) reinterpret_cast<uint4*>(counts)[i] = make_uint4(0u, 0u, 0u, 0u);
    if (p.repetition != nullptr) rep = p.repetition[row];
    if (p.frequency != nullptr) freq = p.frequency[row];
    if (p.presence != nullptr) pres = p.presence[row];
    int len = p.history_lens[row];
    const int prompt = p.prompt_lens != nullptr ? p.prompt_lens[row] : 0;
    if (len < 0 || len > p.max_history) {  // a length outside the tensor counts nothing
      if (threadIdx.x == 0 && run == 0) report_error(p.errs, kErrBadIndex, row);
      len = 0;
    }
    __syncthreads();
    const int64_t* hist = p.history + row * p.history_stride;
    for (int i = threadIdx.x; i < len; i += kThreads) {
      const int64_t id = hist[i];
      if (id < 0 || id >= p.vocab) {
        if (run == 0) report_error(p.errs, kErrBadIndex, row);
        continue;
      }
      const int at = (int)id - first;
      if (at < 0 || at >= SPAN) continue;
      atomicOr(&counts[at], 0x80000000u);
      if (i >= prompt) atomicAdd(&counts[at], 1u);
    }
    __syncthreads();
  }

  const float* bias = p.bias != nullptr ? p.bias + row * p.bias_stride : nullptr;
  const int* allowed = p.allowed != nullptr ? p.allowed + row * p.allowed_stride : nullptr;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int g = i * kThreads + threadIdx.x;
    const int t0 = first + g * VE;
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      const int t = t0 + e;
      if (t < 0 || t >= p.vocab) continue;
      float l = to_f32(x[i].e[e]);
      if (penalise) {
        const uint32_t c = counts[g * VE + e];
        if (c != 0u) {
          l = l > 0.f ? l / rep : l * rep;
          const uint32_t n = c & 0x7FFFFFFFu;
          if (n != 0u) l -= fmaf(freq, (float)n, pres);
        }
      }
      if (bias != nullptr) l += bias[t];
      if (allowed != nullptr && !((allowed[t >> 5] >> (t & 31)) & 1)) l = -INFINITY;
      x[i].e[e] = from_f32<T>(l);
    }
    if (same && t0 >= 0 && t0 + VE <= p.vocab) {
      *reinterpret_cast<Vec<T>*>(dst + t0) = x[i];
    } else {
#pragma unroll
      for (int e = 0; e < VE; ++e)
        if (t0 + e >= 0 && t0 + e < p.vocab) dst[t0 + e] = x[i].e[e];
    }
  }
}

template <typename T>
void launch(const LogitsParams& p, cudaStream_t s) {
  constexpr int VE = 16 / (int)sizeof(T);
  const int span = kThreads * 4 * VE;
  const unsigned runs = (unsigned)((p.vocab + VE - 1 + span - 1) / span);
  launch_k(adjust_logits_kernel<T, 4>, dim3(runs * p.batch), dim3(kThreads), 0, s, 1, p, runs);
}

}  // namespace

void adjust_logits(const LogitsParams& p_in, cudaStream_t s) {
  LogitsParams p = p_in;
  if (p.batch == 0 || p.vocab == 0) return;
  p.errs = device_errors_ptr();
  switch (p.dtype) {
    case 0: launch<__nv_bfloat16>(p, s); break;
    case 1: launch<__half>(p, s); break;
    default: launch<float>(p, s); break;
  }
  B200_CUDA_CHECK(cudaGetLastError());
  count_launch();
}

}  // namespace b200
