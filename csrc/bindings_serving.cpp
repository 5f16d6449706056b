// Bindings of the token-serving operators: paged cache append, paged attention, token sampling.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <cmath>
#include <map>
#include <mutex>

#include "api.h"
#include "common/launch.h"

namespace {

using at::Tensor;
using OptTensor = c10::optional<Tensor>;

cudaStream_t stream_of(const Tensor& t) { return at::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
bool given(const OptTensor& t) { return t.has_value() && t->defined(); }

void no_gradients(const char* op, std::initializer_list<const Tensor*> required, std::initializer_list<const OptTensor*> optional) {
  if (!at::GradMode::is_enabled()) return;
  bool asks = false;
  for (const Tensor* t : required) asks |= t->requires_grad();
  for (const OptTensor* t : optional) asks |= given(*t) && (*t)->requires_grad();
  if (asks) throw pybind11::value_error(std::string(op) + " has no backward pass: call it under torch.no_grad()");
}

int dtype16(const Tensor& t, const char* op) {
  if (t.scalar_type() == at::kHalf) return rt::DT_F16;
  TORCH_CHECK(t.scalar_type() == at::kBFloat16, op, ": fp16 or bf16 CUDA tensors required");
  return rt::DT_BF16;
}

// [n_tok, heads, D] of the cache's type and device with D contiguous
void check_rows(const Tensor& t, const Tensor& like, int64_t n, int64_t heads, int64_t d, const char* op, const char* name) {
  TORCH_CHECK(t.device() == like.device() && t.scalar_type() == like.scalar_type(), op, ": ", name, " must have the cache's device and dtype");
  TORCH_CHECK(t.dim() == 3 && t.size(0) == n && (heads < 0 || t.size(1) == heads) && t.size(2) == d, op, ": ", name, " must be [n_tok, ",
              heads < 0 ? "heads" : "kv heads", ", head_dim], got ", t.sizes());
  TORCH_CHECK(t.stride(2) == 1 || d == 1, op, ": the last dimension of ", name, " must be contiguous");
}

// rows that are written: no two elements may share an address
void check_distinct(const Tensor& t, const char* op, const char* name) {
  std::vector<std::pair<int64_t, int64_t>> dims;
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.size(i) > 1) dims.emplace_back(t.stride(i), t.size(i));
  std::sort(dims.begin(), dims.end());
  int64_t need = 1;
  for (const auto& d : dims) {
    TORCH_CHECK(d.first >= need, op, ": ", name, " has elements that share memory");
    need = d.first * (d.second - 1) + need;
  }
}

const int* check_index(const Tensor& t, const Tensor& like, int64_t n, const char* op, const char* name) {
  TORCH_CHECK(t.device() == like.device() && t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == n && (n <= 1 || t.stride(0) == 1), op,
              ": ", name, " must be a contiguous int32 tensor of ", n, " elements on the cache's device");
  return t.data_ptr<int>();
}

rt::PagedCache make_cache(const Tensor& k, const Tensor& v, const Tensor& table, const char* op) {
  TORCH_CHECK(k.is_cuda() && k.dim() == 4 && v.sizes() == k.sizes() && v.strides() == k.strides() && v.device() == k.device() &&
                  v.scalar_type() == k.scalar_type(),
              op, ": k_pages and v_pages must be [n_pages, kv_heads, page, head_dim] alike in size, strides, dtype and device");
  TORCH_CHECK(k.stride(3) == 1 || k.size(3) == 1, op, ": the last dimension of the pages must be contiguous");
  TORCH_CHECK(k.size(1) > 0 && k.size(2) > 0 && k.size(3) > 0 && k.size(0) < (1ll << 31) && k.size(2) < (1ll << 31), op, ": empty pages, got ",
              k.sizes());
  TORCH_CHECK(table.device() == k.device() && table.scalar_type() == at::kInt && table.dim() == 2 && (table.size(1) <= 1 || table.stride(1) == 1), op,
              ": block_table must be int32 [n_seq, max_pages] with contiguous rows on the cache's device");
  rt::PagedCache c{};
  c.k = k.data_ptr();
  c.v = v.data_ptr();
  c.s_page = k.stride(0); c.s_head = k.stride(1); c.s_row = k.stride(2);
  c.n_pages = int(k.size(0)); c.Hkv = int(k.size(1)); c.page = int(k.size(2)); c.D = int(k.size(3));
  c.table = table.data_ptr<int>();
  c.table_stride = table.stride(0);
  c.n_seq = int(table.size(0)); c.max_pages = int(table.size(1));
  return c;
}

Tensor paged_append(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& k_pages, const Tensor& v_pages, const Tensor& table,
                    const Tensor& pos, const OptTensor& seq, const Tensor& inv_freq, bool interleaved, const OptTensor& q_norm,
                    const OptTensor& k_norm, double eps, const OptTensor& q_out, const OptTensor& k_out) {
  const char* op = "paged_append";
  no_gradients(op, {&q, &k, &v, &k_pages, &v_pages, &inv_freq}, {&q_norm, &k_norm, &q_out, &k_out});
  rt::PagedAppendArgs a{};
  a.dtype = dtype16(k_pages, op);
  a.cache = make_cache(k_pages, v_pages, table, op);
  const int64_t n = q.dim() == 3 ? q.size(0) : -1, D = a.cache.D;
  check_rows(q, k_pages, n, -1, D, op, "q");
  check_rows(k, k_pages, n, a.cache.Hkv, D, op, "k");
  check_rows(v, k_pages, n, a.cache.Hkv, D, op, "v");
  check_distinct(k_pages, op, "the cache");
  TORCH_CHECK(inv_freq.device() == q.device() && inv_freq.scalar_type() == at::kFloat && inv_freq.dim() == 1 && inv_freq.is_contiguous() &&
                  2 * inv_freq.numel() <= D,
              op, ": inv_freq must be contiguous fp32 with at most head_dim / 2 elements on the cache's device");
  TORCH_CHECK(std::isfinite(eps) && eps >= 0, op, ": eps must be finite and not negative");
  for (const OptTensor* w : {&q_norm, &k_norm})
    TORCH_CHECK(!given(*w) || ((*w)->device() == q.device() && (*w)->scalar_type() == q.scalar_type() && (*w)->dim() == 1 && (*w)->numel() == D &&
                               (*w)->is_contiguous()),
                op, ": q_norm and k_norm must be contiguous [head_dim] of the cache's dtype and device");
  const int64_t H = q.size(1);
  TORCH_CHECK(n < (1ll << 31) && n * (H + 2 * a.cache.Hkv) < (1ll << 33), op, ": too many tokens for one call");
  c10::cuda::CUDAGuard guard(q.device());
  Tensor out = given(q_out) ? *q_out : at::empty({n, H, D}, q.options());
  if (given(q_out)) {
    check_rows(out, k_pages, n, H, D, op, "q_out");
    check_distinct(out, op, "q_out");
  }
  if (given(k_out)) {
    check_rows(*k_out, k_pages, n, a.cache.Hkv, D, op, "k_out");
    check_distinct(*k_out, op, "k_out");
    a.k_out = k_out->data_ptr();
    a.ko_st = k_out->stride(0); a.ko_sh = k_out->stride(1);
  }
  a.q = q.data_ptr(); a.k = k.data_ptr(); a.v = v.data_ptr();
  a.q_st = q.stride(0); a.q_sh = q.stride(1);
  a.k_st = k.stride(0); a.k_sh = k.stride(1);
  a.v_st = v.stride(0); a.v_sh = v.stride(1);
  a.q_out = out.data_ptr();
  a.qo_st = out.stride(0); a.qo_sh = out.stride(1);
  a.pos = check_index(pos, q, n, op, "pos");
  a.seq = given(seq) ? check_index(*seq, q, n, op, "seq") : nullptr;
  a.inv_freq = inv_freq.data_ptr<float>();
  a.q_norm = given(q_norm) ? q_norm->data_ptr() : nullptr;
  a.k_norm = given(k_norm) ? k_norm->data_ptr() : nullptr;
  a.eps = float(eps);
  a.n_tok = int(n);
  a.H = int(H);
  a.rot = int(2 * inv_freq.numel());
  a.interleaved = interleaved ? 1 : 0;
  rt::paged_append(a, stream_of(q));
  return out;
}

// Parts of items that several CTAs share, behind zeroed arrival counters.  Calls on one stream follow one another, so a stream keeps
// one buffer; a captured graph may replay beside anything else, so each captured call gets memory of the graph's own.
Tensor attention_workspace(const Tensor& like, int64_t bytes) {
  const auto opts = like.options().dtype(at::kByte);
  const cudaStream_t stream = stream_of(like);
  auto fresh = [&]() {
    Tensor t = at::empty({bytes}, opts);
    C10_CUDA_CHECK(cudaMemsetAsync(t.data_ptr(), 0, rt::PAGED_ATTN_COUNTER_BYTES, stream));
    return t;
  };
  // (the per-thread default stream is one handle for many streams)
  if (stream == cudaStreamPerThread || c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) return fresh();
  static std::mutex mu;
  static auto* kept = new std::map<std::pair<int, cudaStream_t>, Tensor>();  // outlives the allocator's own shutdown
  std::lock_guard<std::mutex> lock(mu);
  Tensor& t = (*kept)[{like.device().index(), stream}];
  if (!t.defined() || t.numel() < bytes) t = fresh();
  return t;
}

Tensor paged_attention(const Tensor& q_in, const Tensor& k_pages, const Tensor& v_pages, const Tensor& table, const Tensor& kv_len,
                       const OptTensor& seq, double scale, int64_t window, double softcap, const OptTensor& out_) {
  const char* op = "paged_attention";
  no_gradients(op, {&q_in, &k_pages, &v_pages}, {&out_});
  rt::PagedAttnArgs a{};
  a.dtype = dtype16(k_pages, op);
  a.cache = make_cache(k_pages, v_pages, table, op);
  const int64_t n = q_in.dim() == 3 ? q_in.size(0) : -1, D = a.cache.D;
  check_rows(q_in, k_pages, n, -1, D, op, "q");
  const int64_t H = q_in.size(1);
  TORCH_CHECK(H > 0 && H % a.cache.Hkv == 0, op, ": ", H, " query heads are not a multiple of ", a.cache.Hkv, " kv heads");
  TORCH_CHECK(D % 8 == 0 && D <= 256, op, ": head_dim must be a multiple of 8 and at most 256, got ", D);
  TORCH_CHECK(a.cache.s_page % 8 == 0 && a.cache.s_head % 8 == 0 && a.cache.s_row % 8 == 0 && reinterpret_cast<uintptr_t>(a.cache.k) % 16 == 0 &&
                  reinterpret_cast<uintptr_t>(a.cache.v) % 16 == 0,
              op, ": the rows of the pages must start on 16-byte boundaries");
  TORCH_CHECK(std::isfinite(scale) && std::abs(scale) <= 1e30, op, ": scale must be finite");
  TORCH_CHECK(softcap == 0 || (softcap >= 1e-6 && softcap <= 1e30), op, ": softcap must be 0 (none) or from 1e-6 to 1e30");
  TORCH_CHECK(window >= 0, op, ": window must not be negative");
  TORCH_CHECK(n < (1ll << 31), op, ": too many tokens for one call");
  c10::cuda::CUDAGuard guard(q_in.device());
  const bool aligned = q_in.stride(0) % 8 == 0 && q_in.stride(1) % 8 == 0 && reinterpret_cast<uintptr_t>(q_in.data_ptr()) % 16 == 0;
  const Tensor q = aligned ? q_in : q_in.clone(at::MemoryFormat::Contiguous);
  Tensor out = given(out_) ? *out_ : at::empty({n, H, D}, q.options());
  if (given(out_)) {
    check_rows(out, k_pages, n, H, D, op, "out");
    check_distinct(out, op, "out");
  }
  a.q = q.data_ptr();
  a.q_st = q.stride(0); a.q_sh = q.stride(1);
  a.out = out.data_ptr();
  a.o_st = out.stride(0); a.o_sh = out.stride(1);
  a.kv_len = check_index(kv_len, q, n, op, "kv_len");
  a.seq = given(seq) ? check_index(*seq, q, n, op, "seq") : nullptr;
  a.n_tok = int(n);
  a.H = int(H);
  a.window = int(std::min<int64_t>(window, INT32_MAX));
  a.scale = float(scale);
  a.softcap = float(softcap);
  if (n == 0) return out;
  const rt::PagedAttnPlan plan = rt::paged_attention_plan(a);
  const Tensor workspace = attention_workspace(q, plan.workspace_bytes);
  rt::paged_attention(a, plan, workspace.data_ptr(), stream_of(q));
  return out;
}

Tensor sample_tokens(const Tensor& logits, const Tensor& uniform, double temperature, int64_t top_k, double top_p, double min_p,
                     const OptTensor& temperature_rows, const OptTensor& top_k_rows, const OptTensor& top_p_rows, const OptTensor& min_p_rows) {
  const char* op = "sample_tokens";
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && (logits.stride(1) == 1 || logits.size(1) == 1), op,
              ": logits must be a CUDA tensor [rows, vocab] with contiguous rows");
  rt::SampleArgs a{};
  a.dtype = logits.scalar_type() == at::kFloat ? int(rt::DT_F32) : dtype16(logits, op);
  const int64_t B = logits.size(0), V = logits.size(1);
  TORCH_CHECK(V >= 1 && V <= 262144, op, ": vocabulary must have 1 to 262144 tokens, got ", V);
  TORCH_CHECK(B < (1ll << 31), op, ": too many rows for one call");
  TORCH_CHECK(uniform.device() == logits.device() && (uniform.scalar_type() == at::kFloat || uniform.scalar_type() == at::kDouble) &&
                  uniform.dim() == 1 && uniform.size(0) == B && uniform.is_contiguous(),
              op, ": uniform must be a contiguous fp32 or fp64 tensor of ", B, " numbers on the logits' device");
  auto rows_f32 = [&](const OptTensor& t, const char* name) -> const float* {
    if (!given(t)) return nullptr;
    TORCH_CHECK(t->device() == logits.device() && t->scalar_type() == at::kFloat && t->dim() == 1 && t->size(0) == B && t->is_contiguous(), op, ": ",
                name, " per row must be a contiguous fp32 tensor of ", B, " numbers on the logits' device");
    return t->data_ptr<float>();
  };
  a.temperature_rows = rows_f32(temperature_rows, "temperature");
  a.top_p_rows = rows_f32(top_p_rows, "top_p");
  a.min_p_rows = rows_f32(min_p_rows, "min_p");
  if (given(top_k_rows)) a.top_k_rows = check_index(*top_k_rows, logits, B, op, "top_k per row");
  // settings are 32-bit numbers, whether they come one a row or one for all
  TORCH_CHECK(temperature >= 0 && std::isfinite(float(temperature)), op, ": temperature must be a finite 32-bit number and not negative");
  TORCH_CHECK(top_k >= 0, op, ": top_k must not be negative");
  TORCH_CHECK(top_p > 0 && top_p <= 1, op, ": top_p must be in (0, 1]");
  TORCH_CHECK(min_p >= 0 && min_p <= 1, op, ": min_p must be in [0, 1]");
  c10::cuda::CUDAGuard guard(logits.device());
  Tensor out = at::empty({B}, logits.options().dtype(at::kLong));
  a.logits = logits.data_ptr();
  a.ld = logits.stride(0);
  a.rows = int(B);
  a.vocab = int(V);
  a.uniform = uniform.data_ptr();
  a.uniform_f64 = uniform.scalar_type() == at::kDouble;
  a.temperature = float(temperature);
  a.top_p = float(top_p);
  a.min_p = float(min_p);
  a.top_k = int(std::min<int64_t>(top_k, V));
  a.out = reinterpret_cast<long long*>(out.data_ptr<int64_t>());
  rt::sample_tokens(a, stream_of(logits));
  return out;
}

}  // namespace

void register_serving_ops(pybind11::module_& m) {
  m.def("paged_append", &paged_append, "per-head RMSNorm + rotary embedding of q / k and append of k / v to a paged cache");
  m.def("paged_attention", &paged_attention, "attention of new tokens over a paged key / value cache");
  m.def("sample_tokens", &sample_tokens, "one token a row by temperature, top-k, top-p and min-p from given random numbers");
}
