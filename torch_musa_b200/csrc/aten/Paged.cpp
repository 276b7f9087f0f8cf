// Serving with a paged key-value cache: the rotary embedding that writes it, the attention of the newest tokens over it, and
// the verification of drafted tokens (csrc/kernels/{paged_attn,verify_drafts}.cu).  Lengths, block tables and random numbers are
// device tensors that only the kernels read, so that a step which calls these operators can be captured into a graph.
// Page numbers and positions that do not fit are noted in the device's assertion word (core/DeviceAssert.h).
// Parity: no counterpart in the reference (its cache is contiguous: reference torch_musa/csrc/aten/ops/attention/mudnn/SDP.cpp).
#include "aten/Ops.h"
#include "core/DeviceAssert.h"

#include <ATen/Functions.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/core/grad_mode.h>
#include <torch/library.h>

#include <algorithm>
#include <climits>
#include <cmath>

namespace b200 {
namespace ops {

namespace {

void check_no_grad(const char* op, std::initializer_list<const at::Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return;
  for (const at::Tensor* t : ts) TORCH_CHECK(!t->defined() || !t->requires_grad(), op, " has no gradient: call it under torch.no_grad()");
}

void check_int32(const char* op, const char* name, const at::Tensor& t, int64_t dim) {
  TORCH_CHECK(t.scalar_type() == at::kInt && t.dim() == dim && (t.numel() <= 1 || t.stride(-1) == 1), op, ": ", name, " must be int32 with ",
              dim, " dimension(s), the last one contiguous");
}

int fit_int(const char* op, int64_t v) {
  TORCH_CHECK(v <= INT_MAX, op, ": a size of ", v, " is not supported");
  return (int)v;
}

// Pools are used where they are: a cache is never copied.
void check_pools(const char* op, const at::Tensor& k, const at::Tensor& v, int64_t D, at::ScalarType dt) {
  TORCH_CHECK(k.dim() == 4 && k.sizes() == v.sizes() && k.size(3) == D && k.size(1) > 0, op,
              ": pools must be [pages, kv heads, page size, head_dim] of one shape, got ", k.sizes(), " and ", v.sizes());
  TORCH_CHECK(k.scalar_type() == dt && v.scalar_type() == dt, op, ": one dtype for tokens and pools");
  TORCH_CHECK(k.size(2) > 0 && k.size(2) % 16 == 0, op, ": the page size must be a multiple of 16, got ", k.size(2));
  for (const at::Tensor* t : {&k, &v}) {
    bool ok = t->stride(3) == 1 && (reinterpret_cast<uintptr_t>(t->const_data_ptr()) & 15) == 0;
    for (int d = 0; d < 3; ++d) ok = ok && (t->size(d) == 1 || t->stride(d) % 8 == 0);
    TORCH_CHECK(ok, op, ": rows of the pools must be contiguous and start on 16 bytes");
  }
}

// strides of a dimension of size one say nothing: 0 keeps them out of the alignment checks
int64_t stride_of(const at::Tensor& t, int64_t d) { return t.size(d) == 1 ? 0 : t.stride(d); }

at::Tensor aligned_rows(const at::Tensor& t) {
  bool ok = t.stride(-1) == 1 && (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15) == 0;
  for (int64_t d = 0; d + 1 < t.dim(); ++d) ok = ok && stride_of(t, d) % 8 == 0;
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

at::Tensor paged_attention(const at::Tensor& q_, const at::Tensor& k_pages, const at::Tensor& v_pages, const at::Tensor& block_table,
                           const at::Tensor& seq_lens, std::optional<int64_t> window, int64_t sinks, std::optional<double> scale) {
  const char* op = "paged_attention";
  TORCH_CHECK(on_device(q_), op, ": expected a blackwell tensor, got ", q_.device());
  check_devices(op, q_, k_pages, v_pages, block_table, seq_lens);
  check_no_grad(op, {&q_, &k_pages, &v_pages});
  TORCH_CHECK(q_.dim() == 4, op, ": q must be [sequences, new tokens, heads, head_dim], got ", q_.sizes());
  const int64_t B = q_.size(0), n = q_.size(1), H = q_.size(2), D = q_.size(3);
  TORCH_CHECK((q_.scalar_type() == at::kBFloat16 || q_.scalar_type() == at::kHalf) && (D == 64 || D == 128), op,
              ": bf16 / fp16 with head_dim 64 or 128");
  check_pools(op, k_pages, v_pages, D, q_.scalar_type());
  TORCH_CHECK(H > 0 && H % k_pages.size(1) == 0, op, ": ", H, " heads do not divide over ", k_pages.size(1), " kv heads");
  check_int32(op, "block_table", block_table, 2);
  check_int32(op, "seq_lens", seq_lens, 1);
  TORCH_CHECK(block_table.size(0) == B && seq_lens.size(0) == B, op, ": block_table and seq_lens must have a row per sequence");
  TORCH_CHECK(!window.has_value() || *window > 0, op, ": window must be positive");
  TORCH_CHECK(sinks >= 0, op, ": sinks must not be negative");
  TORCH_CHECK(!scale.has_value() || (*scale > 0 && std::isfinite(*scale)), op, ": the scale must be positive, got ", scale.value_or(0.0));
  TORCH_CHECK(block_table.size(1) <= (1 << 30) / k_pages.size(2), op, ": block_table covers more than 2^30 tokens");
  if (block_table.size(1) == 0) return at::zeros({B, n, H, D}, q_.options());
  at::Tensor out = at::empty({B, n, H, D}, q_.options());
  if (out.numel() == 0) return out;
  const at::Tensor q = aligned_rows(q_);
  b200_paged_attn_t a{};
  a.dtype = kdtype(q.scalar_type());
  a.head_dim = (int)D;
  a.B = fit_int(op, B); a.n = fit_int(op, n); a.H = fit_int(op, H); a.Hkv = fit_int(op, k_pages.size(1));
  a.num_pages = fit_int(op, k_pages.size(0));
  a.page_size = fit_int(op, k_pages.size(2));
  a.table_width = (int)block_table.size(1);
  a.window = window.has_value() ? (int)std::min<int64_t>(*window, 1 << 30) : 0;      // differences of positions stay in 32 bits
  a.sinks = (int)std::min<int64_t>(sinks, 1 << 30);
  a.scale = (float)scale.value_or(1.0 / std::sqrt((double)D));
  a.q_sb = stride_of(q, 0); a.q_sn = stride_of(q, 1); a.q_sh = stride_of(q, 2);
  a.k_sp = stride_of(k_pages, 0); a.k_sh = stride_of(k_pages, 1); a.k_sr = k_pages.stride(2);
  a.v_sp = stride_of(v_pages, 0); a.v_sh = stride_of(v_pages, 1); a.v_sr = v_pages.stride(2);
  a.table_sb = block_table.stride(0);
  at::Tensor ws;
  if (const int64_t n = b200_paged_attention_workspace(&a)) ws = at::empty({n}, q.options().dtype(at::kFloat));
  DeviceSwitch sw(q.device().index());
  const int e = b200_paged_attention(&a, out.mutable_data_ptr(), q.const_data_ptr(), k_pages.const_data_ptr(), v_pages.const_data_ptr(),
                                     block_table.const_data_ptr<int>(), seq_lens.const_data_ptr<int>(),
                                     ws.defined() ? ws.mutable_data_ptr<float>() : nullptr, device_assert_word(q.device().index()), current_raw_stream(q));
  TORCH_CHECK(e != (int)cudaErrorNotSupported, op, ": unsupported sizes or strides");
  B200_KERNEL_CALL(e);
  return out;
}

at::Tensor paged_rope_cache(const at::Tensor& q_, const at::Tensor& k_, const at::Tensor& v_, const at::Tensor& cos, const at::Tensor& sin,
                            at::Tensor& k_pages, at::Tensor& v_pages, const at::Tensor& block_table, const at::Tensor& seq_lens,
                            const std::optional<at::Tensor>& cu_seqlens) {
  const char* op = "paged_rope_cache";
  TORCH_CHECK(on_device(q_), op, ": expected a blackwell tensor, got ", q_.device());
  check_devices(op, q_, k_, v_, cos, sin, k_pages, v_pages, block_table, seq_lens, cu_seqlens);
  check_no_grad(op, {&q_, &k_, &v_, &k_pages, &v_pages});
  TORCH_CHECK(q_.dim() == 3 && k_.dim() == 3 && v_.sizes() == k_.sizes() && k_.size(0) == q_.size(0) && k_.size(2) == q_.size(2), op,
              ": q must be [tokens, heads, head_dim], k and v [tokens, kv heads, head_dim], got ", q_.sizes(), ", ", k_.sizes(), " and ",
              v_.sizes());
  const int64_t T = q_.size(0), H = q_.size(1), D = q_.size(2), Hkv = k_.size(1);
  TORCH_CHECK((q_.scalar_type() == at::kBFloat16 || q_.scalar_type() == at::kHalf) && (D == 64 || D == 128) && k_.scalar_type() == q_.scalar_type() &&
                  v_.scalar_type() == q_.scalar_type(), op, ": bf16 / fp16 with head_dim 64 or 128");
  check_pools(op, k_pages, v_pages, D, q_.scalar_type());
  at::assert_no_internal_overlap(k_pages);      // an expanded pool: heads or pages would be written over one another
  at::assert_no_internal_overlap(v_pages);
  TORCH_CHECK(k_pages.size(1) == Hkv && H > 0, op, ": the pools have ", k_pages.size(1), " kv heads, k has ", Hkv);
  TORCH_CHECK(cos.scalar_type() == at::kFloat && sin.scalar_type() == at::kFloat && cos.dim() == 2 && cos.size(1) == D / 2 && cos.size(0) > 0 &&
                  sin.sizes() == cos.sizes() && cos.is_contiguous() && sin.is_contiguous(), op,
              ": cos / sin must be contiguous float32 [positions, head_dim / 2]");
  check_int32(op, "block_table", block_table, 2);
  check_int32(op, "seq_lens", seq_lens, 1);
  const int64_t B = seq_lens.size(0);
  TORCH_CHECK(block_table.size(0) == B, op, ": block_table and seq_lens must have a row per sequence");
  TORCH_CHECK(block_table.size(1) <= (1 << 30) / k_pages.size(2), op, ": block_table covers more than 2^30 tokens");
  const bool packed = cu_seqlens.has_value() && cu_seqlens->defined();
  if (packed) {
    check_int32(op, "cu_seqlens", *cu_seqlens, 1);
    TORCH_CHECK(cu_seqlens->size(0) == B + 1, op, ": cu_seqlens must have one element more than there are sequences");
  } else {
    TORCH_CHECK(B > 0 ? T % B == 0 : T == 0, op, ": ", T, " tokens do not divide over ", B, " sequences");
  }
  if (B == 0) return at::zeros({T, H, D}, q_.options());
  at::Tensor out = at::empty({T, H, D}, q_.options());
  if (T == 0) return out;
  const at::Tensor q = aligned_rows(q_), k = aligned_rows(k_), v = aligned_rows(v_), cosr = aligned_rows(cos), sinr = aligned_rows(sin);
  b200_paged_write_t a{};
  a.dtype = kdtype(q.scalar_type());
  a.head_dim = (int)D;
  a.T = fit_int(op, T); a.B = fit_int(op, B); a.H = fit_int(op, H); a.Hkv = fit_int(op, Hkv);
  a.num_pages = fit_int(op, k_pages.size(0));
  a.page_size = fit_int(op, k_pages.size(2));
  a.table_width = (int)block_table.size(1);
  a.table_len = fit_int(op, cos.size(0));
  a.q_st = stride_of(q, 0); a.q_sh = stride_of(q, 1);
  a.k_st = stride_of(k, 0); a.k_sh = stride_of(k, 1);
  a.v_st = stride_of(v, 0); a.v_sh = stride_of(v, 1);
  a.kp_sp = stride_of(k_pages, 0); a.kp_sh = stride_of(k_pages, 1); a.kp_sr = k_pages.stride(2);
  a.vp_sp = stride_of(v_pages, 0); a.vp_sh = stride_of(v_pages, 1); a.vp_sr = v_pages.stride(2);
  a.table_sb = block_table.stride(0);
  DeviceSwitch sw(q.device().index());
  const int e = b200_paged_rope_cache(&a, out.mutable_data_ptr(), q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(),
                                      cosr.const_data_ptr<float>(), sinr.const_data_ptr<float>(), k_pages.mutable_data_ptr(),
                                      v_pages.mutable_data_ptr(), block_table.const_data_ptr<int>(), seq_lens.const_data_ptr<int>(),
                                      packed ? cu_seqlens->const_data_ptr<int>() : nullptr, device_assert_word(q.device().index()),
                                      current_raw_stream(q));
  TORCH_CHECK(e != (int)cudaErrorNotSupported, op, ": unsupported sizes or strides");
  B200_KERNEL_CALL(e);
  return out;
}

std::tuple<at::Tensor, at::Tensor> verify_drafts(const at::Tensor& target_, const at::Tensor& tokens_, const at::Tensor& uniforms_,
                                                 const std::optional<at::Tensor>& draft_) {
  const char* op = "verify_drafts";
  TORCH_CHECK(on_device(target_), op, ": expected a blackwell tensor, got ", target_.device());
  check_devices(op, target_, tokens_, uniforms_, draft_);
  TORCH_CHECK(target_.dim() == 3 && kdtype(target_.scalar_type()) >= 0 && target_.size(1) > 0 && target_.size(2) > 0, op,
              ": target_probs must be [sequences, drafts + 1, vocabulary] in float32, bfloat16 or float16");
  const int64_t B = target_.size(0), n = target_.size(1) - 1, V = target_.size(2);
  TORCH_CHECK(tokens_.scalar_type() == at::kLong && tokens_.dim() == 2 && tokens_.size(0) == B && tokens_.size(1) == n, op,
              ": draft_tokens must be int64 [sequences, drafts]");
  TORCH_CHECK(uniforms_.scalar_type() == at::kFloat && uniforms_.dim() == 2 && uniforms_.size(0) == B && uniforms_.size(1) == n + 1, op,
              ": uniforms must be float32 [sequences, drafts + 1]");
  check_no_grad(op, {&target_});
  if (draft_.has_value()) check_no_grad(op, {&*draft_});
  auto rows = [](const at::Tensor& t) { return t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous(); };
  const at::Tensor target = rows(target_), tokens = rows(tokens_), uniforms = rows(uniforms_);
  at::Tensor draft;
  if (draft_.has_value() && draft_->defined()) {
    TORCH_CHECK(draft_->dim() == 3 && draft_->size(0) == B && draft_->size(1) == n && draft_->size(2) == V &&
                    draft_->scalar_type() == target.scalar_type(), op, ": draft_probs must be [sequences, drafts, vocabulary] in the type of target_probs");
    draft = rows(*draft_);
  }
  at::Tensor taken = at::empty({B}, tokens.options()), out = at::empty({B, n + 1}, tokens.options());
  if (B == 0) return {taken, out};
  const int64_t strides[6] = {target.stride(0), target.stride(1), draft.defined() ? draft.stride(0) : 0, draft.defined() ? draft.stride(1) : 0,
                              tokens.stride(0), uniforms.stride(0)};
  DeviceSwitch sw(target.device().index());
  const int e = b200_verify_drafts(kdtype(target.scalar_type()), taken.mutable_data_ptr<int64_t>(), out.mutable_data_ptr<int64_t>(),
                                   target.const_data_ptr(), draft.defined() && n > 0 ? draft.const_data_ptr() : nullptr,
                                   tokens.const_data_ptr<int64_t>(), uniforms.const_data_ptr<float>(), fit_int(op, B), fit_int(op, n),
                                   fit_int(op, V), strides, current_raw_stream(target));
  TORCH_CHECK(e != (int)cudaErrorNotSupported, op, ": unsupported sizes");
  B200_KERNEL_CALL(e);
  return {taken, out};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(blackwell, m) {
  m.def("paged_attention(Tensor q, Tensor k_pages, Tensor v_pages, Tensor block_table, Tensor seq_lens, int? window=None, int sinks=0, float? scale=None) -> Tensor");
  m.def("paged_rope_cache(Tensor q, Tensor k, Tensor v, Tensor cos, Tensor sin, Tensor(a!) k_pages, Tensor(b!) v_pages, Tensor block_table, Tensor seq_lens, Tensor? cu_seqlens=None) -> Tensor");
  m.def("verify_drafts(Tensor target_probs, Tensor draft_tokens, Tensor uniforms, Tensor? draft_probs=None) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(blackwell, PrivateUse1, m) {
  m.impl("paged_attention", TORCH_FN(paged_attention));
  m.impl("paged_rope_cache", TORCH_FN(paged_rope_cache));
  m.impl("verify_drafts", TORCH_FN(verify_drafts));
}

}  // namespace ops
}  // namespace b200
