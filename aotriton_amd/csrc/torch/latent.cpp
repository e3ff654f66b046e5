// torch.ops.aotriton_amd.latent_attention_*, and latent_cache_attention: the operators of include/aotriton_amd/latent.h on tensors.  Argument
// meaning and refusals are documented in aotriton_amd/torch_ops.py and aotriton_amd/cache.py.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <optional>
#include <tuple>
#include <vector>

#include "aotriton_amd/latent.h"
#include "views.h"

namespace {

using namespace fa_host;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Maybe = std::optional<Tensor>;

bool has(const Maybe& t) { return t.has_value() && t->defined(); }

// ---- the expanded form ------------------------------------------------------------------------------------------------
using FwdSig = std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Maybe&, const Maybe&, c10::SymInt, c10::SymInt,
                                          bool, double);
using BwdSig = std::tuple<Tensor, Tensor, Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                                                          const Tensor&, const Maybe&, const Maybe&, c10::SymInt, c10::SymInt, bool, double);
const c10::TypedOperatorHandle<FwdSig>& forward_op() {
  static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("aotriton_amd::latent_attention_forward", "").typed<FwdSig>();
  return op;
}
const c10::TypedOperatorHandle<BwdSig>& backward_op() {
  static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("aotriton_amd::latent_attention_backward", "").typed<BwdSig>();
  return op;
}

// The inputs as the library takes them; copies of those whose rows are not aligned pieces are held here.
struct Inputs {
  Tensor q, k, v, s;
  bool packed;
  fa_latent_fwd_params p{};
  Inputs(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, const Tensor& s_in, const Maybe& cu_q, const Maybe& cu_k, int64_t max_q,
         int64_t max_k, bool causal, double sm_scale) {
    TORCH_CHECK_VALUE(q_in.dim() == 4 && k_in.dim() == 4 && v_in.dim() == 4 && s_in.dim() == 3,
                      "expected (batch, heads, seq, head_dim) tensors and a (batch, seq, columns) shared part of the keys");
    for (const Tensor* t : {&k_in, &v_in, &s_in})
      TORCH_CHECK_VALUE(t->device() == q_in.device() && t->scalar_type() == q_in.scalar_type(), "query, key, value and shared_key are of one type and on one device");
    packed = has(cu_q);
    TORCH_CHECK_VALUE(packed == has(cu_k), "cu_seqlens come for queries and keys or for neither");
    q = pieces(q_in);
    k = pieces(k_in);
    v = pieces(v_in);
    s = pieces(s_in).unsqueeze(1);
    TORCH_CHECK(view4(q, &p.Q) && view4(k, &p.K) && view4(v, &p.V) && view4(s, &p.S), "the last stride of tensors must be 1");
    if (packed) {
      for (const Tensor* t : {&*cu_q, &*cu_k})
        TORCH_CHECK_VALUE(t->dim() == 1 && t->numel() >= 2 && t->scalar_type() == at::kInt && t->is_contiguous() && t->device() == q_in.device() && t->numel() == cu_q->numel(),
                          "cu_seqlens are contiguous int32 tensors of the sequences + 1 offsets, on the device of the queries");
      TORCH_CHECK_VALUE(q_in.size(0) == 1, "packed sequences are (1, heads, tokens, head_dim) tensors");
      view1(*cu_q, &p.cu_seqlens_q);
      view1(*cu_k, &p.cu_seqlens_k);
      p.max_seqlen_q = as_int32(max_q, "max_seqlen_q");
      p.max_seqlen_k = as_int32(max_k, "max_seqlen_k");
    }
    p.Sm_scale = (float)sm_scale;
    p.causal = causal ? 1 : 0;
  }
};

// A new tensor of a result in the memory order of `like` as it came: the traced call, which knows of no copies, says so.
Tensor like_it(const Tensor& like) {
  const Tensor t = at::empty_like(like);
  return t.stride(-1) == 1 ? t : at::empty(like.sizes(), like.options());
}

std::tuple<Tensor, Tensor> forward_kernel(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& s, const Maybe& cu_q, const Maybe& cu_k,
                                          int64_t max_q, int64_t max_k, bool causal, double sm_scale) {
  const c10::DeviceGuard guard(q.device());
  Inputs in(q, k, v, s, cu_q, cu_k, max_q, max_k, causal, sm_scale);
  const Tensor out = at::empty({q.size(0), q.size(1), q.size(2), v.size(3)}, q.options());
  const Tensor lse = at::empty({q.size(0) * q.size(1), q.size(2)}, q.options().dtype(at::kFloat));
  TORCH_CHECK(view4(out, &in.p.Out) && view2(lse, &in.p.L), "outputs");
  Scratch scratch;
  check_rc(fa_latent_fwd(&in.p, current_stream(), &scratch.c), false);
  if (in.packed) check_rc(fa_zero_gaps(&in.p.Out, &in.p.cu_seqlens_q, &in.p.max_seqlen_q, 1, current_stream()), false);
  return {out, lse};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> backward_kernel(const Tensor& dout_in, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& s,
                                                           const Tensor& out_in, const Tensor& lse_in, const Maybe& cu_q, const Maybe& cu_k,
                                                           int64_t max_q, int64_t max_k, bool causal, double sm_scale) {
  const c10::DeviceGuard guard(q.device());
  TORCH_CHECK_VALUE(dout_in.dim() == 4 && out_in.dim() == 4 && lse_in.dim() == 2 && dout_in.device() == q.device() && out_in.device() == q.device() &&
                        lse_in.device() == q.device() && dout_in.scalar_type() == q.scalar_type() && out_in.scalar_type() == q.scalar_type(),
                    "expected the outputs of latent_attention_forward and a gradient like the first, on the device of the queries");
  Inputs in(q, k, v, s, cu_q, cu_k, max_q, max_k, causal, sm_scale);
  const Tensor out = pieces(out_in), dout = pieces(dout_in), lse = lse_in.contiguous();
  const Tensor dq = like_it(q), dk = like_it(k), dv = like_it(v), ds = like_it(s);
  const Tensor ds4 = ds.unsqueeze(1);
  fa_latent_bwd_params p{};
  p.fwd = in.p;
  TORCH_CHECK(view4(out, &p.fwd.Out) && view2(lse, &p.fwd.L) && view4(dout, &p.DO) && view4(dq, &p.DQ) && view4(dk, &p.DK) && view4(dv, &p.DV) && view4(ds4, &p.DS),
              "the last stride of tensors must be 1");
  Scratch scratch;
  check_rc(fa_latent_bwd(&p, current_stream(), &scratch.c), false);
  if (in.packed) {
    const fa_tensor4 grads[4] = {p.DQ, p.DK, p.DV, p.DS};
    const fa_tensor1 ends[4] = {p.fwd.cu_seqlens_q, p.fwd.cu_seqlens_k, p.fwd.cu_seqlens_k, p.fwd.cu_seqlens_k};
    const int32_t longest[4] = {p.fwd.max_seqlen_q, p.fwd.max_seqlen_k, p.fwd.max_seqlen_k, p.fwd.max_seqlen_k};
    check_rc(fa_zero_gaps(grads, ends, longest, 4, current_stream()), false);
  }
  return {dq, dk, dv, ds};
}

struct LatentFunction : torch::autograd::Function<LatentFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& s, const Maybe& cu_q, const Maybe& cu_k,
                               const c10::SymInt& max_q, const c10::SymInt& max_k, bool causal, double sm_scale) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [o, lse] = forward_op().call(q, k, v, s, cu_q, cu_k, max_q, max_k, causal, sm_scale);
    ctx->save_for_backward({q, k, v, s, o, lse, cu_q.value_or(Tensor()), cu_k.value_or(Tensor())});
    ctx->mark_non_differentiable({lse});
    ctx->set_materialize_grads(false);
    auto& d = ctx->saved_data;
    d["max_q"] = max_q;
    d["max_k"] = max_k;
    d["causal"] = causal;
    d["sm_scale"] = sm_scale;
    return {o, lse};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    auto& d = ctx->saved_data;
    const Tensor dout = grads[0].defined() ? grads[0] : at::zeros_like(s[4]);
    const auto maybe = [](const Tensor& t) { return t.defined() ? Maybe(t) : std::nullopt; };
    auto [dq, dk, dv, ds] = backward_op().call(dout, s[0], s[1], s[2], s[3], s[4], s[5], maybe(s[6]), maybe(s[7]), d["max_q"].toSymInt(),
                                               d["max_k"].toSymInt(), d["causal"].toBool(), d["sm_scale"].toDouble());
    return {dq, dk, dv, ds, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

std::tuple<Tensor, Tensor> forward_autograd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& s, const Maybe& cu_q, const Maybe& cu_k,
                                            c10::SymInt max_q, c10::SymInt max_k, bool causal, double sm_scale) {
  refuse_tangents({&q, &k, &v, &s});
  if (!(at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad() || s.requires_grad()))) {
    at::AutoDispatchBelowADInplaceOrView below;
    return forward_op().call(q, k, v, s, cu_q, cu_k, max_q, max_k, causal, sm_scale);
  }
  const variable_list r = LatentFunction::apply(q, k, v, s, cu_q, cu_k, max_q, max_k, causal, sm_scale);
  return {r[0], r[1]};
}

// (no derivative of its own, as the other backward operators)
struct LatentBackwardFunction : torch::autograd::Function<LatentBackwardFunction> {
  static variable_list forward(AutogradContext*, const Tensor& dout, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& s, const Tensor& out,
                               const Tensor& lse, const Maybe& cu_q, const Maybe& cu_k, const c10::SymInt& max_q, const c10::SymInt& max_k, bool causal,
                               double sm_scale) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [dq, dk, dv, ds] = backward_op().call(dout, q, k, v, s, out, lse, cu_q, cu_k, max_q, max_k, causal, sm_scale);
    return {dq, dk, dv, ds};
  }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK(false, "Trying to backward through aotriton_amd::latent_attention_backward, which has no autograd formula: "
                       "second derivatives of the attention operators are not implemented");
  }
};
std::tuple<Tensor, Tensor, Tensor, Tensor> backward_autograd(const Tensor& dout, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& s,
                                                             const Tensor& out, const Tensor& lse, const Maybe& cu_q, const Maybe& cu_k,
                                                             c10::SymInt max_q, c10::SymInt max_k, bool causal, double sm_scale) {
  refuse_tangents({&dout, &q, &k, &v, &s, &out, &lse});
  bool grad = false;
  for (const Tensor* t : {&dout, &q, &k, &v, &s, &out, &lse}) grad |= t->requires_grad();
  if (!(at::GradMode::is_enabled() && grad)) {
    at::AutoDispatchBelowADInplaceOrView below;
    return backward_op().call(dout, q, k, v, s, out, lse, cu_q, cu_k, max_q, max_k, causal, sm_scale);
  }
  const variable_list r = LatentBackwardFunction::apply(dout, q, k, v, s, out, lse, cu_q, cu_k, max_q, max_k, causal, sm_scale);
  return {r[0], r[1], r[2], r[3]};
}

// ---- the absorbed form, over a cache ------------------------------------------------------------------------------------
using CacheSig = std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, c10::SymInt, c10::SymInt, double);

std::tuple<Tensor, Tensor> cache_kernel(const Tensor& query, const Tensor& latent, const Tensor& table, const Tensor& lengths, const Tensor& starts,
                                        int64_t value_dim, int64_t max_length, double sm_scale) {
  const c10::DeviceGuard guard(latent.device());
  TORCH_CHECK_VALUE(query.dim() == 3 && latent.dim() == 4, "expected a (rows, heads, columns) query and a (pages, 1, slots, columns) cache");
  TORCH_CHECK_VALUE(query.device() == latent.device() && query.scalar_type() == latent.scalar_type(), "the query is of the cache's type and on its device");
  const auto ints = [&](const Tensor& t, int64_t n, fa_tensor1* v, const char* what) {
    TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == n && t.scalar_type() == at::kInt && t.device() == latent.device() && (n <= 1 || t.stride(0) == 1), what,
                      " is a contiguous int32 tensor of ", n, " values on the device of the cache");
    *v = fa_tensor1{t.data_ptr(), {(uint64_t)n}, {1}, FA_DTYPE_INT32};
  };
  TORCH_CHECK_VALUE(lengths.dim() == 1, "lengths are a vector");
  fa_latent_cache_params p{};
  const int64_t n = lengths.size(0);
  ints(lengths, n, &p.lengths, "lengths");
  ints(starts, n + 1, &p.starts, "starts");
  TORCH_CHECK_VALUE(table.dim() == 2 && table.size(0) == n && table.scalar_type() == at::kInt && table.device() == latent.device() &&
                        (table.size(1) <= 1 || table.stride(1) == 1),
                    "the page table is an int32 tensor of ", n, " rows with adjacent columns, on the device of the cache");
  p.table = fa_tensor2{table.data_ptr(), {(uint64_t)n, (uint64_t)table.size(1)}, {(uint64_t)table.stride(0), 1}, FA_DTYPE_INT32};
  TORCH_CHECK_VALUE(value_dim >= 1 && value_dim <= latent.size(3), "value_dim counts columns of the cache");
  const Tensor q = pieces(query).unsqueeze(0);
  const Tensor out = at::empty({query.size(0), query.size(1), value_dim}, query.options()), out4 = out.unsqueeze(0);
  const Tensor lse = at::empty({query.size(0), query.size(1)}, query.options().dtype(at::kFloat));
  TORCH_CHECK_VALUE(view4(q, &p.Q) && view4(latent, &p.latent), "the last stride of tensors must be 1");
  TORCH_CHECK(view4(out4, &p.Out) && view2(lse, &p.L), "outputs");
  p.Sm_scale = (float)sm_scale;
  p.max_length = as_int32(max_length, "max_length");
  Scratch scratch;
  check_rc(fa_latent_cache_attn(&p, current_stream(), &scratch.c), false);
  return {out, lse};
}

std::tuple<Tensor, Tensor> cache_autograd(const Tensor& query, const Tensor& latent, const Tensor& table, const Tensor& lengths, const Tensor& starts,
                                          c10::SymInt value_dim, c10::SymInt max_length, double sm_scale) {
  refuse_tangents({&query, &latent});
  TORCH_CHECK_NOT_IMPLEMENTED(!(at::GradMode::is_enabled() && (query.requires_grad() || latent.requires_grad())),
                              "latent_cache_attention has no gradient; call it under torch.no_grad()");
  static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("aotriton_amd::latent_cache_attention", "").typed<CacheSig>();
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(query, latent, table, lengths, starts, value_dim, max_length, sm_scale);
}

TORCH_LIBRARY_FRAGMENT(aotriton_amd, m) {
  const std::vector<at::Tag> compliant{at::Tag::pt2_compliant_tag};
  m.def("latent_attention_forward(Tensor query, Tensor key, Tensor value, Tensor shared_key, Tensor? cu_seqlens_q, Tensor? cu_seqlens_k, "
        "SymInt max_seqlen_q, SymInt max_seqlen_k, bool is_causal, float sm_scale) -> (Tensor, Tensor)", compliant);
  m.def("latent_attention_backward(Tensor dout, Tensor query, Tensor key, Tensor value, Tensor shared_key, Tensor out, Tensor lse, Tensor? cu_seqlens_q, "
        "Tensor? cu_seqlens_k, SymInt max_seqlen_q, SymInt max_seqlen_k, bool is_causal, float sm_scale) -> (Tensor, Tensor, Tensor, Tensor)", compliant);
  m.def("latent_cache_attention(Tensor query, Tensor latent_cache, Tensor page_table, Tensor lengths, Tensor starts, SymInt value_dim, SymInt max_length, "
        "float sm_scale) -> (Tensor, Tensor)", compliant);
}
TORCH_LIBRARY_IMPL(aotriton_amd, CUDA, m) {
  m.impl("latent_attention_forward", &forward_kernel);
  m.impl("latent_attention_backward", &backward_kernel);
  m.impl("latent_cache_attention", &cache_kernel);
}
TORCH_LIBRARY_IMPL(aotriton_amd, Autograd, m) {
  m.impl("latent_attention_forward", &forward_autograd);
  m.impl("latent_attention_backward", &backward_autograd);
  m.impl("latent_cache_attention", &cache_autograd);
}

}  // namespace
