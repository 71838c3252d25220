// torch.ops.oslo_b200.{ragged_*, paged_*, sample_tokens}: argument checking and allocation around ragged_attention.cu, paged_cache.cu and
// sampling.cu. What needs the host to read device memory (offsets, lengths, page numbers) is not checked here but bounded in the kernels.
#include <c10/cuda/CUDAGuard.h>
#include <torch/library.h>

#include "bindings.h"
#include "oslo_kernels.h"

namespace {

using at::Tensor;
using c10::optional;
using namespace oslo_bind;

bool given(const optional<Tensor>& t) { return t.has_value() && t->defined(); }
void check_ints(const Tensor& t, const Tensor& like, int64_t numel, const char* op, const char* name) {
  TORCH_CHECK(t.device() == like.device() && t.scalar_type() == at::kInt && t.is_contiguous() && t.numel() == numel, op, ": ", name,
              " must be ", numel, " contiguous int32 numbers on ", like.device());
}
// [rows, heads, D] as the kernels read it: contiguous D, 16-byte aligned heads inside their row; a copy of what is laid out otherwise
Tensor rows_of(const Tensor& t, const char* op, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.dim() == 3 && t.size(2) % 8 == 0, op, ": ", name, " must be [rows, heads, D] with D a multiple of 8");
  TORCH_CHECK(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf, op, ": ", name, " must be bf16 or fp16");
  const int64_t r = t.stride(0), h = t.stride(1);
  const bool one_row = t.size(0) <= 1, one_head = t.size(1) <= 1;
  const bool good = t.stride(2) == 1 && (one_row || r % 8 == 0) && (one_head || h % 8 == 0) && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 &&
                    (one_row || r > 0) && (one_head || h > 0) && (one_row || one_head || r >= h);
  return good ? t : t.clone(at::MemoryFormat::Contiguous);
}

// ------------------------------------------------------------------------------------------------------------------ packed sequences
void check_ragged(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& off, const Tensor& koff, int64_t window, double scale) {
  TORCH_CHECK(k.sizes() == v.sizes() && k.size(2) == q.size(2) && k.size(1) > 0 && q.size(1) > 0 && q.size(1) % k.size(1) == 0 && q.size(2) > 0 &&
                  q.size(2) <= 256 && k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type() && k.device() == q.device() &&
                  v.device() == q.device(), "ragged_attention: q, k and v do not match");
  TORCH_CHECK(off.numel() >= 2, "ragged_attention: offsets must hold a sequence's start and end at least");
  check_ints(off, q, off.numel(), "ragged_attention", "offsets");
  check_ints(koff, q, off.numel(), "ragged_attention", "key_offsets");
  TORCH_CHECK(window >= 0 && window <= 0x7fffffff && scale > 0.0, "ragged_attention: the window must not be negative and the scale must be positive");
}

std::tuple<Tensor, Tensor> ragged_fwd(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& off, const Tensor& koff, double scale,
                                      int64_t window, bool with_lse) {
  TORCH_CHECK(q_.is_cuda(), "ragged_attention: q must be on a GPU");
  c10::cuda::CUDAGuard guard(q_.device());
  const Tensor q = rows_of(q_, "ragged_attention", "q"), k = rows_of(k_, "ragged_attention", "k"), v = rows_of(v_, "ragged_attention", "v");
  check_ragged(q, k, v, off, koff, window, scale);
  Tensor o = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
  Tensor lse = at::empty({with_lse ? q.size(0) : 0, q.size(1)}, q.options().dtype(at::kFloat));
  if (q.numel() == 0) return {o, lse};
  if (k.size(0) == 0) {                      // nothing to see
    o.zero_();
    lse.zero_();
    return {o, lse};
  }
  check_rc(oslo_ragged_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), with_lse ? lse.data_ptr<float>() : nullptr, off.data_ptr<int>(),
                           koff.data_ptr<int>(), static_cast<int>(off.numel() - 1), static_cast<int>(q.size(1)), static_cast<int>(k.size(1)),
                           q.size(0), k.size(0), static_cast<int>(q.size(2)), q.stride(0), q.stride(1), k.stride(0), k.stride(1), v.stride(0),
                           v.stride(1), o.stride(0), o.stride(1), static_cast<float>(scale), static_cast<int>(window), dt_code(q),
                           error_word(q.get_device()), cur_stream()), "ragged_fwd");
  return {o, lse};
}

std::tuple<Tensor, Tensor, Tensor> ragged_bwd(const Tensor& dout_, const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& o,
                                              const Tensor& lse, const Tensor& off, const Tensor& koff, double scale, int64_t window) {
  TORCH_CHECK(q_.is_cuda(), "ragged_attention: q must be on a GPU");
  c10::cuda::CUDAGuard guard(q_.device());
  const Tensor q = rows_of(q_, "ragged_attention", "q"), k = rows_of(k_, "ragged_attention", "k"), v = rows_of(v_, "ragged_attention", "v");
  const Tensor dout = rows_of(dout_, "ragged_attention", "the output's gradient");
  check_ragged(q, k, v, off, koff, window, scale);
  TORCH_CHECK(o.sizes() == q.sizes() && o.is_contiguous() && dout.sizes() == q.sizes() && dout.scalar_type() == q.scalar_type() &&
                  o.scalar_type() == q.scalar_type() && dout.device() == q.device() && lse.numel() == q.size(0) * q.size(1),
              "ragged_attention: the output and its gradient must be like q");
  // gradients of slices of one projection's rows are slices of one tensor too, so that nobody has to join them. The given strides alone
  // decide, not addresses: a trace, which has none, must be told the same layout
  const int64_t D = q.size(2), Wq = q.size(1) * D, Wk = k.size(1) * D, W = Wq + 2 * Wk;
  Tensor dq, dk, dv;
  auto sliced = [&](const Tensor& t) { return t.stride(0) == W && t.stride(1) == D && t.stride(2) == 1; };
  if (q.size(0) == k.size(0) && sliced(q_) && sliced(k_) && sliced(v_)) {
    Tensor all = at::empty({q.size(0), W}, q.options());
    dq = all.slice(1, 0, Wq).view(q.sizes());
    dk = all.slice(1, Wq, Wq + Wk).view(k.sizes());
    dv = all.slice(1, Wq + Wk, W).view(v.sizes());
  } else {
    dq = at::empty(q.sizes(), q.options());
    dk = at::empty(k.sizes(), k.options());
    dv = at::empty(v.sizes(), v.options());
  }
  if (q.numel() == 0 || k.numel() == 0) {
    dq.zero_(); dk.zero_(); dv.zero_();
    return {dq, dk, dv};
  }
  Tensor stats = at::empty({q.size(0), q.size(1), 2}, q.options().dtype(at::kFloat));
  check_rc(oslo_ragged_bwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), dout.data_ptr(), lse.data_ptr<float>(), stats.data_ptr<float>(),
                           dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), off.data_ptr<int>(), koff.data_ptr<int>(), static_cast<int>(off.numel() - 1),
                           static_cast<int>(q.size(1)), static_cast<int>(k.size(1)), q.size(0), k.size(0), static_cast<int>(D), q.stride(0),
                           q.stride(1), k.stride(0), k.stride(1), v.stride(0), v.stride(1), o.stride(0), o.stride(1), dout.stride(0), dout.stride(1),
                           dq.stride(0), dq.stride(1), dk.stride(0), dk.stride(1), dv.stride(0), dv.stride(1), static_cast<float>(scale),
                           static_cast<int>(window), dt_code(q), error_word(q.get_device()), cur_stream(D > 128 ? 4 : 3)), "ragged_bwd");
  return {dq, dk, dv};
}

// ------------------------------------------------------------------------------------------------------------------ pages
struct Pool {
  bool q8;
  int64_t pages, heads, page, D, columns, B;
};
Pool check_pool(const char* op, const Tensor& kp, const Tensor& vp, const optional<Tensor>& ks, const optional<Tensor>& vs, const Tensor& table,
                const Tensor& like, at::ScalarType dtype) {
  TORCH_CHECK(kp.is_cuda() && kp.dim() == 4 && kp.is_contiguous() && vp.is_contiguous() && kp.sizes() == vp.sizes() &&
                  kp.scalar_type() == vp.scalar_type() && kp.device() == vp.device() && kp.device() == like.device(),
              op, ": the pools must be two contiguous [pages, heads, page, D] tensors of one type on one device");
  Pool p;
  p.q8 = kp.scalar_type() == at::kFloat8_e4m3fn;
  p.pages = kp.size(0); p.heads = kp.size(1); p.page = kp.size(2); p.D = kp.size(3);
  TORCH_CHECK(p.q8 || kp.scalar_type() == dtype, op, ": a pool holds e4m3 values or the type of its keys and values");
  TORCH_CHECK(dtype == at::kBFloat16 || dtype == at::kHalf, op, ": keys and values are bf16 or fp16");
  TORCH_CHECK(p.pages > 0 && p.heads > 0 && p.page > 0 && p.D > 0 && p.D % 8 == 0 && p.D <= 256 && p.page <= 0x7fffffff && p.pages <= 0x7fffffff,
              op, ": pools need pages, and heads of a multiple of 8 values, 256 at most");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(kp.data_ptr()) % 16 == 0 && reinterpret_cast<uintptr_t>(vp.data_ptr()) % 16 == 0 && (!p.q8 || p.D % 16 == 0),
              op, ": pools must be 16-byte aligned, and heads of 8-bit ones a multiple of 16 values");
  TORCH_CHECK(given(ks) == p.q8 && given(vs) == p.q8, op, ": k_scale and v_scale belong to e4m3 pools");
  if (p.q8)
    for (const Tensor* s : {&*ks, &*vs})
      TORCH_CHECK(s->scalar_type() == at::kFloat && s->is_contiguous() && s->device() == kp.device() && s->sizes() == kp.sizes().slice(0, 3), op,
                  ": scales are contiguous fp32 [pages, heads, page]");
  TORCH_CHECK(table.dim() == 2 && table.scalar_type() == at::kInt && table.is_contiguous() && table.device() == kp.device() && table.size(0) > 0 &&
                  table.size(1) > 0 && table.size(1) * p.page <= 0x7fffffff, op, ": the page table must be contiguous int32 [sequences, pages of one]");
  p.B = table.size(0);
  p.columns = table.size(1);
  return p;
}
float* scale_ptr(const optional<Tensor>& t) { return given(t) ? t->data_ptr<float>() : nullptr; }

void paged_append(const Tensor& k_, const Tensor& v_, const Tensor& kp, const Tensor& vp, const Tensor& table, const Tensor& lengths,
                  const optional<Tensor>& offsets, const optional<Tensor>& ks, const optional<Tensor>& vs) {
  TORCH_CHECK(k_.is_cuda(), "paged_append: k must be on a GPU");
  c10::cuda::CUDAGuard guard(k_.device());
  const Tensor k = rows_of(k_, "paged_append", "k"), v = rows_of(v_, "paged_append", "v");
  const Pool p = check_pool("paged_append", kp, vp, ks, vs, table, k, k.scalar_type());
  TORCH_CHECK(k.sizes() == v.sizes() && v.scalar_type() == k.scalar_type() && v.device() == k.device() && k.size(1) == p.heads && k.size(2) == p.D,
              "paged_append: k and v must be [rows, heads, D] like the pools");
  check_ints(lengths, k, p.B, "paged_append", "lengths");
  if (given(offsets)) check_ints(*offsets, k, p.B + 1, "paged_append", "offsets");
  else TORCH_CHECK(k.size(0) == p.B, "paged_append: one row per sequence, or offsets");
  if (k.size(0) == 0) return;
  check_rc(oslo_paged_append(k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), v.stride(0), v.stride(1), kp.data_ptr(), vp.data_ptr(), scale_ptr(ks),
                             scale_ptr(vs), table.data_ptr<int>(), lengths.data_ptr<int>(), given(offsets) ? offsets->data_ptr<int>() : nullptr, k.size(0),
                             static_cast<int>(p.B), static_cast<int>(p.heads), static_cast<int>(p.D), p.pages, static_cast<int>(p.page),
                             static_cast<int>(p.columns), dt_code(k), p.q8, error_word(k.get_device()), sms(k.get_device()), cur_stream()), "paged_append");
}

std::tuple<Tensor, Tensor> paged_read(const Tensor& kp, const Tensor& vp, const Tensor& table, const Tensor& offsets, int64_t tokens,
                                      const optional<Tensor>& ks, const optional<Tensor>& vs, at::ScalarType dtype) {
  const Pool p = check_pool("paged_read", kp, vp, ks, vs, table, kp, dtype);
  check_ints(offsets, kp, p.B + 1, "paged_read", "offsets");
  TORCH_CHECK(tokens >= 0, "paged_read: the number of tokens must not be negative");
  c10::cuda::CUDAGuard guard(kp.device());
  Tensor k = at::empty({tokens, p.heads, p.D}, kp.options().dtype(dtype)), v = at::empty_like(k);
  if (tokens == 0) return {k, v};
  check_rc(oslo_paged_read(kp.data_ptr(), vp.data_ptr(), scale_ptr(ks), scale_ptr(vs), k.data_ptr(), v.data_ptr(), table.data_ptr<int>(),
                           offsets.data_ptr<int>(), tokens, static_cast<int>(p.B), static_cast<int>(p.heads), static_cast<int>(p.D), p.pages,
                           static_cast<int>(p.page), static_cast<int>(p.columns), dt_code(k), p.q8, error_word(kp.get_device()), sms(kp.get_device()),
                           cur_stream()), "paged_read");
  return {k, v};
}

Tensor paged_attn(const Tensor& q_, const Tensor& kp, const Tensor& vp, const Tensor& table, const Tensor& lengths, double scale, int64_t window,
                  const optional<Tensor>& ks, const optional<Tensor>& vs) {
  TORCH_CHECK(q_.is_cuda(), "paged_attention: q must be on a GPU");
  c10::cuda::CUDAGuard guard(q_.device());
  const Tensor q = rows_of(q_, "paged_attention", "q");
  const Pool p = check_pool("paged_attention", kp, vp, ks, vs, table, q, q.scalar_type());
  TORCH_CHECK(q.size(0) == p.B && q.size(1) > 0 && q.size(1) % p.heads == 0 && q.size(2) == p.D, "paged_attention: q must be [sequences, heads, D]");
  TORCH_CHECK(window >= 0 && window <= 0x7fffffff, "paged_attention: the window must not be negative");
  check_ints(lengths, q, p.B, "paged_attention", "lengths");
  Tensor o = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
  check_rc(oslo_paged_attn(q.data_ptr(), q.stride(0), q.stride(1), kp.data_ptr(), vp.data_ptr(), scale_ptr(ks), scale_ptr(vs), o.data_ptr(),
                           table.data_ptr<int>(), lengths.data_ptr<int>(), static_cast<int>(p.B), static_cast<int>(q.size(1)), static_cast<int>(p.heads),
                           static_cast<int>(p.D), p.pages, static_cast<int>(p.page), static_cast<int>(p.columns), static_cast<float>(scale),
                           static_cast<int>(window), dt_code(q), p.q8, error_word(q.get_device()), sms(q.get_device()), cur_stream()), "paged_attention");
  return o;
}

// ------------------------------------------------------------------------------------------------------------------ sampling
Tensor sample_tokens(const Tensor& logits, const Tensor& uniform, const optional<Tensor>& temperature, const optional<Tensor>& top_k,
                     const optional<Tensor>& top_p, const optional<Tensor>& min_p, double temperature1, int64_t top_k1, double top_p1, double min_p1) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && logits.size(1) > 0 && (logits.size(1) == 1 || logits.stride(1) == 1),
              "sample_tokens: logits must be [rows, vocabulary] with contiguous rows");
  const int64_t rows = logits.size(0), V = logits.size(1);
  const int dt = dt_code(logits);
  TORCH_CHECK(V <= oslo_sample_max_vocab(dt) && rows <= (1 << 24), "sample_tokens: at most ", oslo_sample_max_vocab(dt), " tokens and 2^24 rows");
  auto per_row = [&](const optional<Tensor>& t, at::ScalarType type, const char* name) {
    if (given(t)) TORCH_CHECK(t->device() == logits.device() && t->scalar_type() == type && t->is_contiguous() && t->numel() == rows, "sample_tokens: ", name,
                              " must be a number or ", rows, " contiguous ", type, " numbers on ", logits.device());
  };
  TORCH_CHECK(uniform.scalar_type() == at::kFloat || uniform.scalar_type() == at::kDouble, "sample_tokens: uniform must be fp32 or fp64");
  per_row(uniform, uniform.scalar_type(), "uniform");
  per_row(temperature, at::kFloat, "temperature");
  per_row(top_k, at::kInt, "top_k");
  per_row(top_p, at::kFloat, "top_p");
  per_row(min_p, at::kFloat, "min_p");
  c10::cuda::CUDAGuard guard(logits.device());
  Tensor out = at::empty({rows}, logits.options().dtype(at::kLong));
  if (rows == 0) return out;
  auto ptr = [](const optional<Tensor>& t) { return given(t) ? t->data_ptr<float>() : nullptr; };
  const int k1 = static_cast<int>(std::min<int64_t>(std::max<int64_t>(top_k1, 0), 0x7fffffff));
  check_rc(oslo_sample_tokens(logits.data_ptr(), logits.stride(0), uniform.data_ptr(), uniform.scalar_type() == at::kDouble, ptr(temperature),
                              given(top_k) ? top_k->data_ptr<int>() : nullptr, ptr(top_p), ptr(min_p), temperature1, k1, top_p1, min_p1,
                              reinterpret_cast<long long*>(out.data_ptr<int64_t>()),
                              static_cast<int>(rows), static_cast<int>(V), dt, sms(logits.get_device()), cur_stream()), "sample_tokens");
  return out;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(oslo_b200, m) {
  m.def("ragged_fwd(Tensor q, Tensor k, Tensor v, Tensor offsets, Tensor key_offsets, float scale, int window, bool with_lse) -> (Tensor, Tensor)");
  m.def("ragged_bwd(Tensor dout, Tensor q, Tensor k, Tensor v, Tensor o, Tensor lse, Tensor offsets, Tensor key_offsets, float scale, int window) -> (Tensor, Tensor, Tensor)");
  m.def("paged_append(Tensor k, Tensor v, Tensor(a!) k_pages, Tensor(b!) v_pages, Tensor table, Tensor lengths, Tensor? offsets=None, Tensor(c!)? k_scale=None, Tensor(d!)? v_scale=None) -> ()");
  m.def("paged_read(Tensor k_pages, Tensor v_pages, Tensor table, Tensor offsets, int tokens, Tensor? k_scale, Tensor? v_scale, ScalarType dtype) -> (Tensor, Tensor)");
  m.def("paged_attn(Tensor q, Tensor k_pages, Tensor v_pages, Tensor table, Tensor lengths, float scale, int window, Tensor? k_scale=None, Tensor? v_scale=None) -> Tensor");
  m.def("sample_tokens(Tensor logits, Tensor uniform, Tensor? temperature, Tensor? top_k, Tensor? top_p, Tensor? min_p, float temperature1, int top_k1, float top_p1, float min_p1) -> Tensor");
}
TORCH_LIBRARY_IMPL(oslo_b200, CUDA, m) {
  m.impl("ragged_fwd", &ragged_fwd);
  m.impl("ragged_bwd", &ragged_bwd);
  m.impl("paged_append", &paged_append);
  m.impl("paged_read", &paged_read);
  m.impl("paged_attn", &paged_attn);
  m.impl("sample_tokens", &sample_tokens);
}
