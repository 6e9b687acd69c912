// Adjusting next-token logits: penalties for tokens that occurred, additive biases, a bitmask of allowed
// tokens.  For row b, with seen(t) <=> t in history[b, :len] and n(t) = count of t in history[b, prompt:len]:
//   l = seen ? (l > 0 ? l / repetition : l * repetition) : l
//   l = l - (frequency * n + presence * (n > 0)) + bias[t];   not allowed: -inf
// computed in fp32 and rounded once to the logits' type.
//
// A block takes a RANGE of tokens of one row.  It first goes over the row's history: the tokens that lie in its
// range are counted in shared memory, and one thread for each distinct one replaces the counter by the
// penalised logit.  Then it streams the range, 16 bytes per thread and access, without any further barrier.
// (Counting per 4096-token step inside the streaming loop took three barriers for every step, and penalising
// there a division in the half of all warps that hold some token of the history: 89 us instead of 66 for
// 256 rows of 128256 fp32 logits with 1024 tokens of history on average.)  Bound by HBM.
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
constexpr int kHistory = 8;  // places of the history per thread that are loaded ahead

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

// Rows start anywhere: ranges are counted in 16-byte groups of the row's memory, `shift` elements of the first
// group belonging to what lies before the row.  Steps that the row does not fill, and all steps when input and
// output are aligned differently, go group by group, and element by element in groups that are not full.
template <typename T, int NV, int RANGE, int MIN_BLOCKS>
__global__ void __launch_bounds__(kThreads, MIN_BLOCKS) adjust_logits_kernel(LogitsParams p, unsigned blocks_per_row) {
  pdl_wait_and_release();
  constexpr int VE = 16 / (int)sizeof(T);
  constexpr int GROUPS = kThreads * VE;  // tokens between a thread's groups; a multiple of 32
  constexpr int SPAN = GROUPS * NV;      // tokens of a step
  static_assert(RANGE % SPAN == 0 && RANGE / 32 <= kThreads, "range");
  __shared__ __align__(16) uint32_t counts[RANGE];
  __shared__ uint32_t seen[RANGE / 32];
  __shared__ uint32_t todo[RANGE / 32];
  const int row = (int)(blockIdx.x / blocks_per_row);
  const T* src = reinterpret_cast<const T*>(p.logits) + row * p.stride;
  T* dst = reinterpret_cast<T*>(p.out) + row * p.out_stride;
  const int shift = (int)((reinterpret_cast<uintptr_t>(src) & 15) / sizeof(T));
  const bool same = shift == (int)((reinterpret_cast<uintptr_t>(dst) & 15) / sizeof(T));
  const bool first_block = blockIdx.x % blocks_per_row == 0;
  const int base = (int)(blockIdx.x % blocks_per_row) * RANGE - shift;  // token of element 0 (may be negative)
  const uint32_t* allowed =
      p.allowed != nullptr ? reinterpret_cast<const uint32_t*>(p.allowed) + row * p.allowed_stride : nullptr;
  const float* bias = p.bias != nullptr ? p.bias + row * p.bias_stride : nullptr;
  const bool bias_vec = shift == 0 && (reinterpret_cast<uintptr_t>(bias) & 15) == 0;
  const int tid = (int)threadIdx.x;
  const int bit = (base + tid * VE) & 31;  // of a group's first token in its mask word, in every step
  auto whole = [&](int at) { return same && at >= 0 && at + SPAN <= p.vocab; };

  // One step's logits and mask words
  Vec<T> x[NV];
  uint32_t lo[NV], hi[NV];
  auto load_step = [&](int at) {
    const T* s = src + at + tid * VE;
#pragma unroll
    for (int i = 0; i < NV; ++i) x[i] = *reinterpret_cast<const Vec<T>*>(s + i * GROUPS);
    if (allowed != nullptr) {
      const uint32_t* m = allowed + ((at + tid * VE) >> 5);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        lo[i] = m[i * (GROUPS / 32)];
        if (bit + VE > 32) hi[i] = m[i * (GROUPS / 32) + 1];
      }
    }
  };
  if (whole(base)) load_step(base);

  const bool penalise = p.history != nullptr;
  if (penalise) {
    const int64_t* hist = p.history + row * p.history_stride;
    int64_t raw[kHistory];  // token at place i * kThreads + tid
#pragma unroll
    for (int i = 0; i < kHistory; ++i)
      raw[i] = i * kThreads + tid < p.max_history ? hist[i * kThreads + tid] : 0;
    int len = p.history_lens[row];
    const int prompt = p.prompt_lens != nullptr ? p.prompt_lens[row] : 0;
    const float rep = p.repetition != nullptr ? p.repetition[row] : 1.f;
    const float freq = p.frequency != nullptr ? p.frequency[row] : 0.f;
    const float pres = p.presence != nullptr ? p.presence[row] : 0.f;
    if (tid < RANGE / 32) seen[tid] = todo[tid] = 0u;
#pragma unroll
    for (int i = 0; i < RANGE / 4 / kThreads; ++i)
      reinterpret_cast<uint4*>(counts)[i * kThreads + tid] = make_uint4(0u, 0u, 0u, 0u);
    if (len < 0 || len > p.max_history) {  // a length outside the tensor counts nothing
      if (tid == 0 && first_block) report_error(p.errs, kErrBadIndex, row);
      len = 0;
    }
    __syncthreads();
    // Counts the token at a place; true if it is this thread's to penalise (it was the first to see it).
    auto count = [&](int place, int64_t t) {
      if (t < 0 || t >= p.vocab) {
        if (first_block) report_error(p.errs, kErrBadIndex, row);
        return false;
      }
      const int at = (int)t - base;
      if (at < 0 || at >= RANGE || !B200_IN_BOUNDS(p.errs, place, 1, p.max_history, 153)) return false;
      if (place >= prompt) atomicAdd(&counts[at], 1u);
      return ((atomicOr(&seen[at >> 5], 1u << (at & 31)) >> (at & 31)) & 1u) == 0u;
    };
    auto penalised = [&](float l, int t) {
      uint32_t& c = counts[t - base];
      l = l > 0.f ? l / rep : l * rep;
      if (c != 0u) l -= fmaf(freq, (float)c, pres);
      c = __float_as_uint(l);
    };
    uint32_t mine = 0u;
    T value[kHistory];
#pragma unroll
    for (int i = 0; i < kHistory; ++i)
      if (i * kThreads + tid < len && count(i * kThreads + tid, raw[i])) {
        mine |= 1u << i;
        value[i] = src[raw[i]];
      }
    // places behind those in registers: a token that is new there is marked, and penalised by whoever clears
    // the mark
    for (int i = kHistory * kThreads + tid; i < len; i += kThreads) {
      const int64_t t = hist[i];
      if (count(i, t)) atomicOr(&todo[((int)t - base) >> 5], 1u << (((int)t - base) & 31));
    }
    __syncthreads();
    if (mine != 0u) {
#pragma unroll
      for (int i = 0; i < kHistory; ++i)
        if ((mine >> i) & 1u) penalised(to_f32(value[i]), (int)raw[i]);
    }
    for (int i = kHistory * kThreads + tid; i < len; i += kThreads) {
      const int64_t t = hist[i];
      const long long at = t - base;
      if (t < 0 || t >= p.vocab || at < 0 || at >= RANGE) continue;
      const uint32_t m = 1u << (at & 31);
      if (atomicAnd(&todo[at >> 5], ~m) & m) penalised(to_f32(src[t]), (int)t);
    }
    __syncthreads();
  }

#pragma unroll 1
  for (int step = 0; step < RANGE; step += SPAN) {
    const int at = base + step;
    if (at >= p.vocab) break;
    if (!whole(at)) {
      auto adjusted = [&](float l, int t) {
        const int g = t - base;
        if (penalise && ((seen[g >> 5] >> (g & 31)) & 1u)) l = __uint_as_float(counts[g]);
        if (bias != nullptr) l += bias[t];
        if (allowed != nullptr && !((allowed[t >> 5] >> (t & 31)) & 1u)) l = -INFINITY;
        return from_f32<T>(l);
      };
#pragma unroll 1
      for (int t0 = at + tid * VE; t0 < min(at + SPAN, p.vocab); t0 += GROUPS) {
        if (same && t0 >= 0 && t0 + VE <= p.vocab) {
          Vec<T> y = *reinterpret_cast<const Vec<T>*>(src + t0);
#pragma unroll
          for (int e = 0; e < VE; ++e) y.e[e] = adjusted(to_f32(y.e[e]), t0 + e);
          if (B200_IN_BOUNDS(p.errs, t0, VE, p.vocab, 151)) *reinterpret_cast<Vec<T>*>(dst + t0) = y;
        } else {
#pragma unroll 1
          for (int t = max(t0, 0); t < min(t0 + VE, p.vocab); ++t)
            if (B200_IN_BOUNDS(p.errs, t, 1, p.vocab, 152)) dst[t] = adjusted(to_f32(src[t]), t);
        }
      }
      continue;
    }
    if (step > 0) load_step(at);
    float add[NV][VE];
    if (bias != nullptr) {
      const float* b = bias + at + tid * VE;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (bias_vec) {
#pragma unroll
          for (int e = 0; e < VE; e += 4) {
            const float4 v = *reinterpret_cast<const float4*>(b + i * GROUPS + e);
            add[i][e] = v.x, add[i][e + 1] = v.y, add[i][e + 2] = v.z, add[i][e + 3] = v.w;
          }
        } else {
#pragma unroll
          for (int e = 0; e < VE; ++e) add[i][e] = b[i * GROUPS + e];
        }
      }
    }
    T* out = dst + at + tid * VE;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float l[VE];
#pragma unroll
      for (int e = 0; e < VE; ++e) l[e] = to_f32(x[i].e[e]);
      if (penalise) {
        const int g = step + i * GROUPS + tid * VE;
        const uint32_t hit = (seen[g >> 5] >> (g & 31)) & ((1u << VE) - 1u);  // VE divides 32
        if (hit != 0u) {
#pragma unroll
          for (int e = 0; e < VE; ++e)
            if ((hit >> e) & 1u) l[e] = __uint_as_float(counts[g + e]);
        }
      }
      if (bias != nullptr) {
#pragma unroll
        for (int e = 0; e < VE; ++e) l[e] += add[i][e];
      }
      if (allowed != nullptr) {
        const uint32_t m = bit + VE > 32 ? __funnelshift_r(lo[i], hi[i], bit) : lo[i] >> bit;
#pragma unroll
        for (int e = 0; e < VE; ++e)
          if (!(m & (1u << e))) l[e] = -INFINITY;
      }
      Vec<T> y;
#pragma unroll
      for (int e = 0; e < VE; ++e) y.e[e] = from_f32<T>(l[e]);
      if (B200_IN_BOUNDS(p.errs, at + tid * VE + i * GROUPS, VE, p.vocab, 150))
        *reinterpret_cast<Vec<T>*>(out + i * GROUPS) = y;
    }
  }
}

template <typename T, int NV, int RANGE, int MIN_BLOCKS>
void launch_range(const LogitsParams& p, cudaStream_t s) {
  constexpr int VE = 16 / (int)sizeof(T);
  const unsigned per_row = (unsigned)(((long long)p.vocab + VE - 1 + RANGE - 1) / RANGE);
  launch_k(adjust_logits_kernel<T, NV, RANGE, MIN_BLOCKS>, dim3(per_row * p.batch), dim3(kThreads), 0, s, 1, p, per_row);
}

// Ranges of 8192 tokens; with few rows, where those would not give every SM two blocks, of one access per thread.
template <typename T>
void launch(const LogitsParams& p, cudaStream_t s) {
  constexpr int VE = 16 / (int)sizeof(T);
  if ((long long)(p.vocab + 8191) / 8192 * p.batch >= 2 * num_sms_cached())
    launch_range<T, 16 / VE, 8192, 4>(p, s);
  else
    launch_range<T, 1, kThreads * VE, 2>(p, s);
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
