// Python bindings of the serving kernels: paged key/value cache, attention over it, logit adjustment.
// Shapes and types are checked before anything touches a device.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <cfloat>
#include <climits>
#include <cmath>
#include <initializer_list>
#include <optional>
#include <vector>

#include "paged.h"
#include "paged_sched.cuh"

namespace {

using at::Tensor;

// Numbers go into messages as text: this library carries its own copy of the C++ runtime, whose stream
// insertion of integers does not work with the streams of the one that PyTorch brings.
std::string shape(const Tensor& t) {
  std::string s = "[";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i > 0 ? ", " : "") + std::to_string(t.size(i));
  return s + "]";
}

// These operators have no backward pass: a result that a gradient would be wanted through is refused.
void no_backward(const char* name, std::initializer_list<const Tensor*> tensors) {
  if (!at::GradMode::is_enabled()) return;
  for (const Tensor* t : tensors)
    TORCH_CHECK(t == nullptr || !t->requires_grad(), name,
                " has no backward pass; call it under torch.no_grad() or on detached tensors");
}
const Tensor* given(const std::optional<Tensor>& t) { return t.has_value() ? &*t : nullptr; }

void check_device(const Tensor& t, const Tensor& first, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.device() == first.device(), name, " is on ", t.device().str(), ", expected ", first.device().str());
}

void check_aligned(const Tensor& t, const char* name) {
  TORCH_CHECK(reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0, name, " must be 16-byte aligned");
}

// Strides (token, head) of a [tokens, heads, head_dim] bf16 tensor; a dimension of one element has none.
struct RowStrides {
  long long t, h;
};
RowStrides check_rows(const Tensor& x, int64_t tokens, int64_t heads, int64_t hd, bool written, const char* name) {
  TORCH_CHECK(x.dim() == 3 && x.size(1) == heads && x.size(2) == hd && (tokens < 0 || x.size(0) == tokens), name,
              " must be [", tokens < 0 ? std::string("tokens") : std::to_string(tokens), ", ", std::to_string(heads), ", ",
              std::to_string(hd),
              "], got ", shape(x));
  TORCH_CHECK(x.scalar_type() == at::kBFloat16, name, " must be bfloat16");
  TORCH_CHECK(x.stride(2) == 1, name, " must have unit stride along head_dim");
  RowStrides s{x.size(0) > 1 ? x.stride(0) : heads * hd, x.size(1) > 1 ? x.stride(1) : hd};
  TORCH_CHECK(s.t % 8 == 0 && s.h % 8 == 0 && s.t > 0 && s.h > 0, name, " strides must be positive multiples of 8 elements");
  if (written)
    TORCH_CHECK(s.h >= hd && (x.size(0) <= 1 || s.t >= (heads - 1) * s.h + hd), name,
                " must not overlap itself and must be laid out token by token");
  check_aligned(x, name);
  return s;
}

int log2_page(int64_t page) {
  TORCH_CHECK(page == 16 || page == 32 || page == 64 || page == 128, "page_size must be 16, 32, 64 or 128, got ",
              std::to_string(page));
  return page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : 7;
}

// Pages [n_pages, kv_heads, page_size, head_dim] and their scales.
b200::KvPool check_pool(const Tensor& k, const Tensor& v, const std::optional<Tensor>& ks,
                        const std::optional<Tensor>& vs) {
  TORCH_CHECK(k.dim() == 4 && v.sizes() == k.sizes(), "pages must be two [n_pages, kv_heads, page_size, head_dim] "
              "tensors of one shape, got ", shape(k), " and ", shape(v));
  TORCH_CHECK(k.scalar_type() == v.scalar_type(), "k and v pages must have the same dtype");
  TORCH_CHECK(k.is_contiguous() && v.is_contiguous(), "pages must be contiguous");
  TORCH_CHECK(k.size(0) >= 1 && k.size(1) >= 1, "pages need at least one page and one kv head");
  TORCH_CHECK(k.size(3) == 64 || k.size(3) == 128, "head_dim must be 64 or 128, got ", std::to_string(k.size(3)));
  log2_page(k.size(2));
  TORCH_CHECK(k.size(0) * k.size(1) * k.size(2) <= INT_MAX, "the pool holds more than 2^31 - 1 rows");
  b200::KvPool p{};
  const at::ScalarType type = k.scalar_type();
  TORCH_CHECK(type == at::kBFloat16 || type == at::kFloat8_e4m3fn || type == at::kChar,
              "pages must be bfloat16, float8_e4m3fn or int8, got ", type);
  p.fmt = type == at::kBFloat16 ? b200::KV_BF16 : type == at::kFloat8_e4m3fn ? b200::KV_E4M3 : b200::KV_INT8;
  const bool quantised = p.fmt != b200::KV_BF16;
  TORCH_CHECK(ks.has_value() == quantised && vs.has_value() == quantised,
              "8-bit pages need k_scale and v_scale, bf16 pages have none");
  if (quantised) {
    for (const Tensor* s : {&*ks, &*vs})
      TORCH_CHECK(s->scalar_type() == at::kFloat && s->is_contiguous() && s->sizes() == k.sizes().slice(0, 3),
                  "scales must be contiguous float32 [n_pages, kv_heads, page_size]");
    check_aligned(*ks, "k_scale");
    check_aligned(*vs, "v_scale");
    p.k_scale = ks->data_ptr<float>();
    p.v_scale = vs->data_ptr<float>();
  }
  check_aligned(k, "k pages");
  check_aligned(v, "v pages");
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  p.kv_heads = (int)k.size(1);
  p.head_dim = (int)k.size(3);
  return p;
}

b200::PagedSeqs check_seqs(const Tensor& k_pages, const Tensor& table, const Tensor& lens,
                           const std::optional<Tensor>& starts, int64_t total_q, int64_t max_q) {
  TORCH_CHECK(table.dim() == 2 && table.scalar_type() == at::kInt && (table.size(1) <= 1 || table.stride(1) == 1),
              "block_table must be int32 [batch, pages] with unit column stride");
  const int64_t batch = table.size(0);
  TORCH_CHECK(lens.dim() == 1 && lens.scalar_type() == at::kInt && lens.is_contiguous() && lens.size(0) == batch,
              "kv_lens must be contiguous int32 [", std::to_string(batch), "]");
  if (starts.has_value()) {
    TORCH_CHECK(starts->dim() == 1 && starts->scalar_type() == at::kInt && starts->is_contiguous() &&
                    starts->size(0) == batch + 1,
                "q_starts must be contiguous int32 [", std::to_string(batch + 1), "]");
  } else {
    TORCH_CHECK(total_q == batch, "without q_starts every sequence has one new token: expected ",
                std::to_string(batch), " rows, got ", std::to_string(total_q));
  }
  TORCH_CHECK(total_q <= INT_MAX && batch < INT_MAX, "too many rows");
  b200::PagedSeqs s{};
  s.table = table.data_ptr<int>();
  s.table_stride = table.stride(0);
  s.kv_lens = lens.data_ptr<int>();
  s.q_starts = starts.has_value() ? starts->data_ptr<int>() : nullptr;
  s.batch = (int)batch;
  s.page_log2 = log2_page(k_pages.size(2));
  s.max_pages = (int)std::min<int64_t>(table.size(1), INT_MAX >> s.page_log2);
  s.n_pages = (int)k_pages.size(0);
  s.total_q = (int)total_q;
  s.max_q = (int)max_q;
  return s;
}

void check_devices(const Tensor& first, const Tensor& k, const Tensor& v, const std::optional<Tensor>& ks,
                   const std::optional<Tensor>& vs, const Tensor& table, const Tensor& lens,
                   const std::optional<Tensor>& starts) {
  check_device(k, first, "k pages");
  check_device(v, first, "v pages");
  if (ks.has_value()) check_device(*ks, first, "k_scale");
  if (vs.has_value()) check_device(*vs, first, "v_scale");
  check_device(table, first, "block_table");
  check_device(lens, first, "kv_lens");
  if (starts.has_value()) check_device(*starts, first, "q_starts");
}

cudaStream_t cur_stream() { return at::cuda::getCurrentCUDAStream().stream(); }

void kv_cache_write(const Tensor& k_pages, const Tensor& v_pages, const std::optional<Tensor>& k_scale,
                    const std::optional<Tensor>& v_scale, const Tensor& k, const Tensor& v, const Tensor& table,
                    const Tensor& lens, const std::optional<Tensor>& starts) {
  no_backward("kv_cache_write", {&k, &v, &k_pages, &v_pages, given(k_scale), given(v_scale)});
  const b200::KvPool pool = check_pool(k_pages, v_pages, k_scale, v_scale);
  const RowStrides sk = check_rows(k, -1, pool.kv_heads, pool.head_dim, false, "k");
  const RowStrides sv = check_rows(v, k.size(0), pool.kv_heads, pool.head_dim, false, "v");
  const b200::PagedSeqs seqs = check_seqs(k_pages, table, lens, starts, k.size(0), INT_MAX);
  check_device(k, k, "k");
  check_device(v, k, "v");
  check_devices(k, k_pages, v_pages, k_scale, v_scale, table, lens, starts);
  c10::cuda::CUDAGuard g(k.device());
  b200::kv_cache_write(seqs, pool, reinterpret_cast<const __nv_bfloat16*>(k.data_ptr()),
                       reinterpret_cast<const __nv_bfloat16*>(v.data_ptr()), sk.t, sk.h, sv.t, sv.h, cur_stream());
}

std::tuple<Tensor, Tensor> kv_cache_read(const Tensor& k_pages, const Tensor& v_pages,
                                         const std::optional<Tensor>& k_scale, const std::optional<Tensor>& v_scale,
                                         const Tensor& table, const Tensor& lens, const std::optional<Tensor>& starts,
                                         int64_t total, at::ScalarType type) {
  no_backward("kv_cache_read", {&k_pages, &v_pages, given(k_scale), given(v_scale)});
  const b200::KvPool pool = check_pool(k_pages, v_pages, k_scale, v_scale);
  TORCH_CHECK(type == at::kBFloat16 || type == at::kFloat, "the cache is read as bfloat16 or float32");
  TORCH_CHECK(total >= 0, "total must not be negative");
  const b200::PagedSeqs seqs = check_seqs(k_pages, table, lens, starts, total, INT_MAX);
  check_devices(k_pages, k_pages, v_pages, k_scale, v_scale, table, lens, starts);
  c10::cuda::CUDAGuard g(k_pages.device());
  const auto options = k_pages.options().dtype(type);
  Tensor k = at::empty({total, pool.kv_heads, pool.head_dim}, options);
  Tensor v = at::empty({total, pool.kv_heads, pool.head_dim}, options);
  b200::kv_cache_read(seqs, pool, k.data_ptr(), v.data_ptr(), type == at::kFloat, cur_stream());
  return {k, v};
}

Tensor paged_attention(const Tensor& q, const Tensor& k_pages, const Tensor& v_pages,
                       const std::optional<Tensor>& k_scale, const std::optional<Tensor>& v_scale,
                       const std::optional<Tensor>& out_, const Tensor& table, const Tensor& lens,
                       const std::optional<Tensor>& starts, int64_t max_q, std::optional<double> scale_) {
  no_backward("paged_attention", {&q, given(out_), &k_pages, &v_pages, given(k_scale), given(v_scale)});
  const b200::KvPool pool = check_pool(k_pages, v_pages, k_scale, v_scale);
  TORCH_CHECK(q.dim() == 3, "q must be [tokens, heads, head_dim], got ", shape(q));
  const int64_t heads = q.size(1);
  TORCH_CHECK(heads >= 1 && heads % pool.kv_heads == 0, "heads (", std::to_string(heads),
              ") must be a multiple of kv_heads (", std::to_string(pool.kv_heads), ")");
  TORCH_CHECK(heads / pool.kv_heads <= 128, "more than 128 query heads share a kv head");
  const RowStrides sq = check_rows(q, -1, heads, pool.head_dim, false, "q");
  if (out_.has_value()) {
    check_rows(*out_, q.size(0), heads, pool.head_dim, true, "out");
    TORCH_CHECK(!out_->is_alias_of(q) && !out_->is_alias_of(k_pages) && !out_->is_alias_of(v_pages),
                "out must not share memory with q or the pages");
  }
  TORCH_CHECK(max_q >= 1 && max_q <= INT_MAX, "max_q_len must be at least 1");
  const double scale = scale_.has_value() ? *scale_ : 1.0 / std::sqrt((double)pool.head_dim);
  TORCH_CHECK(scale >= FLT_MIN && scale <= 1e30, "scale must be between 2^-126 and 1e30");
  const b200::PagedSeqs seqs = check_seqs(k_pages, table, lens, starts, q.size(0), max_q);
  check_device(q, q, "q");
  if (out_.has_value()) check_device(*out_, q, "out");
  check_devices(q, k_pages, v_pages, k_scale, v_scale, table, lens, starts);
  c10::cuda::CUDAGuard g(q.device());
  Tensor out = out_.has_value() ? *out_ : at::empty(q.sizes(), q.options());
  const RowStrides so = check_rows(out, q.size(0), heads, pool.head_dim, true, "out");
  b200::PagedAttnParams p{};
  p.seqs = seqs;
  p.pool = pool;
  p.q = reinterpret_cast<const __nv_bfloat16*>(q.data_ptr());
  p.q_stride_t = sq.t;
  p.q_stride_h = sq.h;
  p.out = reinterpret_cast<__nv_bfloat16*>(out.data_ptr());
  p.o_stride_t = so.t;
  p.o_stride_h = so.h;
  p.heads = (int)heads;
  p.group = (int)(heads / pool.kv_heads);
  p.scale = (float)scale;
  // from PyTorch's allocator: reused in stream order, private to a graph that captures the call
  c10::DataPtr workspace;
  b200::paged_attention(
      p,
      [&](size_t bytes, bool can_do_without) -> void* {
        try {
          workspace = c10::cuda::CUDACachingAllocator::get()->allocate(bytes);
        } catch (const c10::OutOfMemoryError&) {
          if (!can_do_without) throw;
          return nullptr;
        }
        return workspace.get();
      },
      cur_stream());
  return out;
}

// Host-only view of how the attention kernels divide their work (CPU tensors, no GPU needed): per block and
// item (block, sequence, kv head, tile, first unit in the item, end unit, units of the item).
std::vector<std::vector<int64_t>> paged_schedule(Tensor starts, Tensor lens, int64_t max_tokens, int64_t total_q,
                                                 int64_t max_q, int64_t kv_heads, int64_t tile_tokens,
                                                 int64_t unit_log2, int64_t grid) {
  TORCH_CHECK(!lens.is_cuda() && !starts.is_cuda() && lens.scalar_type() == at::kInt &&
                  starts.scalar_type() == at::kInt && lens.is_contiguous() && starts.is_contiguous() &&
                  starts.numel() == lens.numel() + 1,
              "paged_schedule: contiguous int32 CPU tensors required");
  b200::PagedSeqs s{};
  s.kv_lens = lens.data_ptr<int>();
  s.q_starts = starts.data_ptr<int>();
  s.batch = (int)lens.numel();
  s.max_pages = (int)max_tokens;
  s.total_q = (int)total_q;
  s.max_q = (int)max_q;
  const b200::PagedShape shape{(int)tile_tokens, (int)unit_log2, (int)kv_heads};
  std::vector<std::vector<int64_t>> out;
  long long total = 0;
  std::vector<long long> base;
  for (int b = 0; b < s.batch; ++b) {
    base.push_back(total);
    total += b200::head_places(b200::seq_info(s, b), shape) * kv_heads;
  }
  const long long blocks = std::min<long long>(grid, total);
  auto item_of = [&](long long v) {
    int b = s.batch - 1;
    while (base[b] > v || b200::seq_info(s, b).qn == 0) --b;
    return b200::item_at(s, shape, b, base[b], v);
  };
  auto cut = [&](long long c) {
    if (c == blocks) return total;
    const long long v = b200::raw_begin(c, total, blocks);
    return b200::moved_cut(item_of(v), v);
  };
  for (long long c = 0; c < blocks; ++c) {
    const long long begin = cut(c), end = cut(c + 1);
    if (begin == end) continue;
    b200::PagedItem it = item_of(begin);
    int unit = b200::unit_of_cut(it, begin);
    while (true) {
      out.push_back({c, it.b, it.kvh, it.rt, unit, b200::unit_of_cut(it, end), it.n_units});
      if (end <= b200::item_end(it)) break;
      b200::next_item(it, s, shape);
      unit = 0;
    }
  }
  return out;
}

void check_per_row(const std::optional<Tensor>& t, const Tensor& logits, at::ScalarType type, const char* name) {
  if (!t.has_value()) return;
  TORCH_CHECK(t->dim() == 1 && t->size(0) == logits.size(0) && t->is_contiguous() && t->scalar_type() == type, name,
              " must be contiguous ", type, " [", std::to_string(logits.size(0)), "]");
}

Tensor adjust_logits(const Tensor& logits, const std::optional<Tensor>& out_, const std::optional<Tensor>& history,
                     const std::optional<Tensor>& history_lens, const std::optional<Tensor>& prompt_lens,
                     const std::optional<Tensor>& repetition, const std::optional<Tensor>& frequency,
                     const std::optional<Tensor>& presence, const std::optional<Tensor>& bias,
                     const std::optional<Tensor>& allowed) {
  no_backward("adjust_logits",
              {&logits, given(out_), given(repetition), given(frequency), given(presence), given(bias)});
  TORCH_CHECK(logits.dim() == 2 && (logits.size(1) <= 1 || logits.stride(1) == 1),
              "logits must be [batch, vocab] with unit column stride");
  const int64_t batch = logits.size(0), vocab = logits.size(1);
  TORCH_CHECK(vocab <= INT_MAX - 65536 && batch <= 1 << 20, "logits: too many rows or columns");
  if (out_.has_value()) {
    TORCH_CHECK(out_->sizes() == logits.sizes() && out_->scalar_type() == logits.scalar_type() &&
                    (vocab <= 1 || out_->stride(1) == 1),
                "out must have the logits' shape and dtype and unit column stride");
    TORCH_CHECK(batch <= 1 || out_->stride(0) >= vocab, "out rows must not overlap");
    if (out_->is_alias_of(logits))
      TORCH_CHECK(out_->data_ptr() == logits.data_ptr() && (batch <= 1 || out_->stride(0) == logits.stride(0)),
                  "out must be the logits themselves or not share memory with them");
  }
  b200::LogitsParams p{};
  const at::ScalarType type = logits.scalar_type();
  TORCH_CHECK(type == at::kBFloat16 || type == at::kHalf || type == at::kFloat,
              "logits must be bfloat16, float16 or float32, got ", type);
  p.dtype = type == at::kBFloat16 ? 0 : type == at::kHalf ? 1 : 2;
  const bool penalties = repetition.has_value() || frequency.has_value() || presence.has_value();
  TORCH_CHECK(history.has_value() == history_lens.has_value(), "history and history_lens go together");
  TORCH_CHECK(!penalties || history.has_value(), "penalties need a history");
  TORCH_CHECK(!prompt_lens.has_value() || history.has_value(), "prompt_lens needs a history");
  if (history.has_value()) {
    TORCH_CHECK(history->dim() == 2 && history->size(0) == batch && history->scalar_type() == at::kLong &&
                    (history->size(1) <= 1 || history->stride(1) == 1) && history->size(1) <= INT_MAX,
                "history must be int64 [", std::to_string(batch), ", length] with unit column stride");
    check_per_row(history_lens, logits, at::kInt, "history_lens");
    check_per_row(prompt_lens, logits, at::kInt, "prompt_lens");
  }
  check_per_row(repetition, logits, at::kFloat, "repetition_penalty");
  check_per_row(frequency, logits, at::kFloat, "frequency_penalty");
  check_per_row(presence, logits, at::kFloat, "presence_penalty");
  if (bias.has_value()) {
    TORCH_CHECK((bias->dim() == 1 || (bias->dim() == 2 && bias->size(0) == batch)) && bias->size(-1) == vocab &&
                    bias->scalar_type() == at::kFloat && (vocab <= 1 || bias->stride(-1) == 1),
                "bias must be float32 [vocab] or [batch, vocab] with unit column stride");
    p.bias = bias->data_ptr<float>();
    p.bias_stride = bias->dim() == 2 ? bias->stride(0) : 0;
  }
  if (allowed.has_value()) {
    const int64_t words = (vocab + 31) / 32;
    TORCH_CHECK((allowed->dim() == 1 || (allowed->dim() == 2 && allowed->size(0) == batch)) &&
                    allowed->size(-1) == words && allowed->scalar_type() == at::kInt &&
                    (words <= 1 || allowed->stride(-1) == 1),
                "allowed must be an int32 bitmask [", std::to_string(words), "] or [batch, ", std::to_string(words), "] with unit column stride");
    p.allowed = allowed->data_ptr<int>();
    p.allowed_stride = allowed->dim() == 2 ? allowed->stride(0) : 0;
  }
  check_device(logits, logits, "logits");
  if (out_.has_value()) check_device(*out_, logits, "out");
  const std::pair<const std::optional<Tensor>*, const char*> rest[] = {
      {&history, "history"},   {&history_lens, "history_lens"}, {&prompt_lens, "prompt_lens"},
      {&repetition, "repetition_penalty"}, {&frequency, "frequency_penalty"}, {&presence, "presence_penalty"},
      {&bias, "bias"},         {&allowed, "allowed"}};
  for (const auto& [t, name] : rest)
    if (t->has_value()) check_device(**t, logits, name);
  c10::cuda::CUDAGuard g(logits.device());
  Tensor out = out_.has_value() ? *out_ : at::empty(logits.sizes(), logits.options());
  p.logits = logits.data_ptr();
  p.out = out.data_ptr();
  p.stride = logits.stride(0);
  p.out_stride = out.stride(0);
  p.batch = (int)batch;
  p.vocab = (int)vocab;
  if (penalties) {
    p.history = history->data_ptr<int64_t>();
    p.history_stride = history->stride(0);
    p.max_history = (int)history->size(1);
    p.history_lens = history_lens->data_ptr<int>();
    p.prompt_lens = prompt_lens.has_value() ? prompt_lens->data_ptr<int>() : nullptr;
    p.repetition = repetition.has_value() ? repetition->data_ptr<float>() : nullptr;
    p.frequency = frequency.has_value() ? frequency->data_ptr<float>() : nullptr;
    p.presence = presence.has_value() ? presence->data_ptr<float>() : nullptr;
  }
  b200::adjust_logits(p, cur_stream());
  return out;
}

}  // namespace

void bind_serving(pybind11::module_& m) {
  m.def("kv_cache_write", &kv_cache_write);
  m.def("kv_cache_read",
        [](const Tensor& k, const Tensor& v, const std::optional<Tensor>& ks, const std::optional<Tensor>& vs,
           const Tensor& table, const Tensor& lens, const std::optional<Tensor>& starts, int64_t total,
           const py::object& dtype) {
          return kv_cache_read(k, v, ks, vs, table, lens, starts, total,
                               torch::python::detail::py_object_to_dtype(dtype));
        });
  m.def("paged_attention", &paged_attention);
  m.def("paged_schedule", &paged_schedule);
  m.def("adjust_logits", &adjust_logits);
}
