// Paged key/value cache: layout, per-sequence metadata and the launchers of the kernels that work on it.
//
// One layer's K (or V) is a pool of pages [n_pages, kv_heads, page_size, head_dim]: the tokens of one
// head and page are contiguous, so 16 tokens of one head are one run of memory.  Formats: bf16, or 8-bit
// codes (e4m3 / int8) with one fp32 scale per token and head in [n_pages, kv_heads, page_size].
// Sequence b owns row b of the block table: its token t lies in page table[b][t / page_size], offset
// t % page_size.  Its last q_len tokens (rows q_starts[b] .. q_starts[b + 1]) are the new ones.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <functional>

#include "common.cuh"

namespace b200 {

enum KvFormat : int { KV_BF16 = 0, KV_E4M3 = 1, KV_INT8 = 2 };

// Largest code of a format: a row's scale is max|x| divided by it.
__host__ __device__ constexpr float kv_code_max(int fmt) { return fmt == KV_E4M3 ? 448.0f : 127.0f; }

struct PagedSeqs {
  const int* table;  // [batch, max_pages], row stride table_stride
  const int* kv_lens;
  const int* q_starts;  // [batch + 1], or null: one new token per sequence
  long long table_stride;
  int batch, max_pages, n_pages, page_log2;
  int total_q;  // rows of the token tensors
  int max_q;    // bound on a sequence's new tokens
};

// Rows of a pool: (page, head, offset) cells.
__host__ __device__ inline long long pool_cells(const PagedSeqs& s, int kv_heads) {
  return (long long)s.n_pages * kv_heads << s.page_log2;
}

struct SeqInfo {
  int q0, qn, len;
  bool ok;
};

// Metadata of sequence b.  Values that do not fit the tensors (rows outside them, more new tokens than
// max_q, more cached tokens than the block table has room for) make the sequence invalid: the kernels
// skip it and leave a record.
__host__ __device__ inline SeqInfo seq_info(const PagedSeqs& s, int b) {
  SeqInfo r;
  r.q0 = s.q_starts != nullptr ? s.q_starts[b] : b;
  const int q1 = s.q_starts != nullptr ? s.q_starts[b + 1] : b + 1;
  r.len = s.kv_lens[b];
  r.ok = r.q0 >= 0 && r.q0 <= q1 && q1 <= s.total_q && q1 - r.q0 <= s.max_q && r.len >= 0 &&
         (long long)r.len <= ((long long)s.max_pages << s.page_log2);
  r.qn = r.ok ? q1 - r.q0 : 0;
  return r;
}

// Sequence whose rows hold row t (-1: none).  Rows are in the order of the sequences.
__host__ __device__ inline int seq_of_row(const PagedSeqs& s, int t) {
  if (s.q_starts == nullptr) return t < s.batch ? t : -1;
  int lo = 0, hi = s.batch;  // the last b with q_starts[b] <= t lies in [lo, hi)
  if (t < s.q_starts[0] || t >= s.q_starts[s.batch]) return -1;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (s.q_starts[mid] <= t)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

#if defined(__CUDACC__)

// Biased exponent of the power of two that a row of q is divided by before it becomes fp16, from the largest |x| of
// the row (bf16 bits): the row's maximum lands in [1, 2).  A row of zeros is left alone: with the smallest
// power, its product with the scale and K's power could reach 0, and a masked score, -inf, times 0 is NaN.
__device__ __forceinline__ int q_row_exponent(uint32_t top) {
  return top == 0u ? 127 : min(max((int)(top >> 7), 2), 252);
}
// What the scores of such a row are multiplied by, kept a positive number (-inf stays -inf, 0 stays 0): where the
// product leaves the range of fp32 at the lower end, the scores are 0 to fp32 all the same.
__device__ __forceinline__ float score_factor(float scale, float q_power, float k_power) {
  return fminf(fmaxf(scale * q_power * k_power, 1.17549435e-38f), 3.40282347e38f);
}

// V that is all zero adds nothing to a row but its weights' sum.  Where V's size goes into the exponent of the
// weights it gets the lowest one: any size of its own could raise the maximum so far above the others' exponents
// that their fp16 weights sink into subnormals.  Not lower than this, so that weights of up to 2^14 times
// 2^80, summed over 2^31 tokens, stay below 2^126.
constexpr int kLowestExponent = -80;

#endif

struct KvPool {
  void* k;
  void* v;
  float* k_scale;  // null for bf16
  float* v_scale;
  int fmt, kv_heads, head_dim;
};

// Writes rows k, v [total_q, kv_heads, head_dim] (bf16, strides in elements) to their places.
void kv_cache_write(const PagedSeqs& seqs, const KvPool& pool, const __nv_bfloat16* k, const __nv_bfloat16* v,
                    long long k_stride_t, long long k_stride_h, long long v_stride_t, long long v_stride_h,
                    cudaStream_t s);
// Reads them back into contiguous [total_q, kv_heads, head_dim] tensors (bf16 or fp32).
void kv_cache_read(const PagedSeqs& seqs, const KvPool& pool, void* k, void* v, bool out_f32, cudaStream_t s);

struct PagedAttnParams {
  PagedSeqs seqs;
  KvPool pool;
  const __nv_bfloat16* q;  // [total_q, heads, head_dim]
  long long q_stride_t, q_stride_h;
  __nv_bfloat16* out;
  long long o_stride_t, o_stride_h;
  int heads, group;  // group = heads / kv_heads
  float scale;
  DeviceErrors* errs;
};
// `alloc` returns device memory of at least the given size (16-byte aligned) that stays valid for the work
// enqueued on the stream by this call; null where that much is not to be had and the caller can do without.
using PagedAlloc = std::function<void*(size_t bytes, bool can_do_without)>;
void paged_attention(const PagedAttnParams& p, const PagedAlloc& alloc, cudaStream_t s);
// Its form for more than 64 rows per kv head and sequence, 32 for bf16 pages of head_dim 128 (paged_chunk.cu).
void paged_attention_chunk(const PagedAttnParams& p, const PagedAlloc& alloc, cudaStream_t s);

struct LogitsParams {
  const void* logits;  // [batch, vocab], row stride in elements
  void* out;
  long long stride, out_stride;
  int dtype;  // 0 bf16, 1 fp16, 2 fp32
  int batch, vocab;
  const int64_t* history;  // [batch, max_history]
  long long history_stride;
  int max_history;
  const int* history_lens;
  const int* prompt_lens;     // null: 0
  const float* repetition;    // [batch] or null
  const float* frequency;
  const float* presence;
  const float* bias;          // [vocab] (stride 0) or [batch, vocab], or null
  long long bias_stride;
  const int* allowed;         // [batch, words] bitmask (row stride; 0 for one mask for all rows) or null
  long long allowed_stride;
  DeviceErrors* errs;
};
void adjust_logits(const LogitsParams& p, cudaStream_t s);

}  // namespace b200
