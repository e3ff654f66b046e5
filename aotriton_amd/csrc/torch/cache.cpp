// torch.ops.aotriton_amd.tree_attention and cache_*: the operators of include/aotriton_amd/cache.h on tensors.  Argument meaning and
// refusals are documented in aotriton_amd/cache.py.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <torch/library.h>

#include <optional>
#include <tuple>
#include <type_traits>
#include <vector>

#include "aotriton_amd/cache.h"
#include "views.h"

namespace {

using namespace fa_host;

// an int32 vector of n values; one value is a vector too
void ints(const Tensor& t, int64_t n, const Tensor& like, fa_tensor1* v, const char* what) {
  TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == n && t.scalar_type() == at::kInt && t.device() == like.device() && (n <= 1 || t.stride(0) == 1),
                    what, " is a contiguous int32 tensor of ", n, " values on the device of the cache");
  *v = fa_tensor1{t.data_ptr(), {(uint64_t)n}, {1}, FA_DTYPE_INT32};
}

void int_rows(const Tensor& t, int64_t rows, const Tensor& like, fa_tensor2* v, const char* what) {
  TORCH_CHECK_VALUE(t.dim() == 2 && t.size(0) == rows && t.scalar_type() == at::kInt && t.device() == like.device() &&
                        (t.size(1) <= 1 || t.stride(1) == 1),
                    what, " is an int32 tensor of ", rows, " rows with adjacent columns, on the device of the cache");
  *v = fa_tensor2{t.data_ptr(), {(uint64_t)t.size(0), (uint64_t)t.size(1)}, {(uint64_t)t.stride(0), 1}, FA_DTYPE_INT32};
}

void rows4(const Tensor& t, const Tensor& like, fa_tensor4* v, const char* what) {
  TORCH_CHECK_VALUE(t.dim() == 4 && t.stride(-1) == 1 && t.scalar_type() == like.scalar_type() && t.device() == like.device(), what,
                    " is a 4-D tensor with unit last stride, of the cache's type and on its device");
  TORCH_CHECK(view4(t, v), "element type");
}

void pages(const Tensor& k, const Tensor& v, fa_tensor4* kv, fa_tensor4* vv) {
  rows4(k, k, kv, "the cache of keys");
  rows4(v, k, vv, "the cache of values");
}

fa_cache cache_of(const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& lengths) {
  fa_cache c{};
  pages(k, v, &c.K, &c.V);
  TORCH_CHECK_VALUE(lengths.dim() == 1, "lengths are a vector");
  ints(lengths, lengths.size(0), k, &c.lengths, "lengths");
  int_rows(table, lengths.size(0), k, &c.table, "the page table");
  return c;
}

std::tuple<Tensor, Tensor> tree_kernel(const Tensor& query, const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& lengths,
                                       const std::optional<Tensor>& parents, int64_t max_length, int64_t window, int64_t sinks, double sm_scale) {
  const c10::DeviceGuard guard(k.device());
  fa_tree_params p{};
  p.cache = cache_of(k, v, table, lengths);
  TORCH_CHECK_VALUE(query.dim() == 4, "expected a (sequences, heads, tokens, head_dim) query");
  const Tensor q = pieces(query);
  rows4(q, k, &p.Q, "the query");
  const Tensor out = at::empty({q.size(0), q.size(1), q.size(2), v.size(3)}, q.options());
  const Tensor lse = at::empty({q.size(0), q.size(1), q.size(2)}, q.options().dtype(at::kFloat));
  TORCH_CHECK(view4(out, &p.Out), "outputs");
  p.L = fa_tensor2{lse.data_ptr(), {(uint64_t)(q.size(0) * q.size(1)), (uint64_t)q.size(2)}, {(uint64_t)q.size(2), 1}, FA_DTYPE_FLOAT32};
  if (parents.has_value() && parents->defined()) {
    TORCH_CHECK_VALUE(parents->dim() == 2 && parents->size(1) == q.size(2), "parents are (sequences, tokens)");
    int_rows(*parents, q.size(0), k, &p.parents, "parents");
  }
  p.Sm_scale = (float)sm_scale;
  p.max_length = as_int32(max_length, "max_length");
  p.window = as_int32(window, "window");
  p.sinks = as_int32(sinks, "sinks");
  Scratch scratch;
  check_rc(fa_tree_attn(&p, current_stream(), &scratch.c), false);
  return {out, lse};
}

void append_kernel(const Tensor& key, const Tensor& value, const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& lengths,
                   const std::optional<Tensor>& counts) {
  const c10::DeviceGuard guard(k.device());
  const fa_cache c = cache_of(k, v, table, lengths);
  TORCH_CHECK_VALUE(key.dim() == 4 && value.dim() == 4, "expected (sequences, heads, tokens, head_dim) rows");
  const Tensor nk = pieces(key), nv = pieces(value);
  fa_tensor4 kv{}, vv{};
  rows4(nk, k, &kv, "the new keys");
  rows4(nv, k, &vv, "the new values");
  fa_tensor1 n{};
  const bool has = counts.has_value() && counts->defined();
  if (has) ints(*counts, lengths.size(0), k, &n, "counts");
  check_rc(fa_cache_append(&kv, &vv, &c, has ? &n : nullptr, current_stream()), false);
}

void copy_kernel(const Tensor& k, const Tensor& v, const Tensor& source, const Tensor& target) {
  const c10::DeviceGuard guard(k.device());
  fa_tensor4 kv{}, vv{};
  pages(k, v, &kv, &vv);
  TORCH_CHECK_VALUE(source.dim() == 1, "pages are vectors");
  fa_tensor1 s{}, t{};
  ints(source, source.size(0), k, &s, "source");
  ints(target, source.size(0), k, &t, "target");
  check_rc(fa_cache_copy_pages(&kv, &vv, &s, &t, current_stream()), false);
}

void fork_kernel(const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& lengths, const Tensor& uses, const Tensor& source,
                 const Tensor& target, const Tensor& spare) {
  const c10::DeviceGuard guard(k.device());
  const fa_cache c = cache_of(k, v, table, lengths);
  TORCH_CHECK_VALUE(source.dim() == 1, "sequences are vectors");
  fa_tensor1 u{}, s{}, t{}, x{};
  ints(uses, k.size(0), k, &u, "uses");
  ints(source, source.size(0), k, &s, "source");
  ints(target, source.size(0), k, &t, "target");
  ints(spare, source.size(0), k, &x, "spare");
  check_rc(fa_cache_fork(&c, &u, &s, &t, &x, current_stream()), false);
}

Tensor keep_kernel(const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& lengths, const Tensor& path, const Tensor& counts) {
  const c10::DeviceGuard guard(k.device());
  const fa_cache c = cache_of(k, v, table, lengths);
  fa_tensor2 p{};
  int_rows(path, lengths.size(0), k, &p, "the path");
  fa_tensor1 n{}, out{};
  ints(counts, lengths.size(0), k, &n, "counts");
  const Tensor after = at::empty({lengths.size(0)}, lengths.options());
  ints(after, lengths.size(0), k, &out, "lengths");
  check_rc(fa_cache_keep_path(&c, &p, &n, &out, current_stream()), false);
  return after;
}

void free_kernel(const Tensor& table, const Tensor& uses, const Tensor& sequences, const Tensor& first, const Tensor& last) {
  const c10::DeviceGuard guard(table.device());
  TORCH_CHECK_VALUE(table.dim() == 2 && uses.dim() == 1 && sequences.dim() == 1, "a table of rows, and vectors");
  fa_tensor2 t{};
  int_rows(table, table.size(0), table, &t, "the page table");
  fa_tensor1 u{}, s{}, a{}, b{};
  ints(uses, uses.size(0), table, &u, "uses");
  ints(sequences, sequences.size(0), table, &s, "sequences");
  ints(first, sequences.size(0), table, &a, "first");
  ints(last, sequences.size(0), table, &b, "last");
  check_rc(fa_cache_free(&t, &u, &s, &a, &b, current_stream()), false);
}

// (no derivatives: caches are inference state.  A call that would have to record one says so)
std::tuple<Tensor, Tensor> tree_autograd(const Tensor& query, const Tensor& k, const Tensor& v, const Tensor& table,
                                         const Tensor& lengths, const std::optional<Tensor>& parents, c10::SymInt max_length, c10::SymInt window,
                                         c10::SymInt sinks, double sm_scale) {
  refuse_tangents({&query, &k, &v});
  TORCH_CHECK_NOT_IMPLEMENTED(!(at::GradMode::is_enabled() && (query.requires_grad() || k.requires_grad() || v.requires_grad())),
                              "tree_attention has no gradient; call it under torch.no_grad()");
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("aotriton_amd::tree_attention", "")
                             .typed<std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                                                               const std::optional<Tensor>&, c10::SymInt, c10::SymInt, c10::SymInt, double)>();
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(query, k, v, table, lengths, parents, max_length, window, sinks, sm_scale);
}

// The ops that write, kWritten the places of what they write to: no derivatives either, and the version counters of those tensors move,
// so that a backward that has kept one of them says so.
constexpr char kAppend[] = "aotriton_amd::cache_append", kCopy[] = "aotriton_amd::cache_copy_pages", kFork[] = "aotriton_amd::cache_fork",
               kKeep[] = "aotriton_amd::cache_keep_path", kFree[] = "aotriton_amd::cache_free";
template <const char* kName, auto kKernel, size_t... kWritten> struct Writer;
template <const char* kName, typename R, typename... A, R (*kKernel)(A...), size_t... kWritten>
struct Writer<kName, kKernel, kWritten...> {
  static const c10::TypedOperatorHandle<R(A...)>& op() {
    static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow(kName, "").template typed<R(A...)>();
    return op;
  }
  static R autograd(c10::DispatchKeySet keys, A... a) {
    const auto refuse = [](const auto& t) {
      if constexpr (std::is_same_v<std::decay_t<decltype(t)>, Tensor>) {
        refuse_tangents({&t});
        TORCH_CHECK_NOT_IMPLEMENTED(!(at::GradMode::is_enabled() && t.requires_grad()), kName, " has no gradient; call it under torch.no_grad()");
      }
    };
    (refuse(a), ...);
    return op().redispatch(keys & c10::after_autograd_keyset, a...);
  }
  static R inplace(c10::DispatchKeySet keys, A... a) {
    const auto all = std::forward_as_tuple(a...);
    // (a tensor of inference mode has no counter)
    const auto written = [](const Tensor& t) {
      if (!t.is_inference()) torch::autograd::impl::bump_version(t);
    };
    if constexpr (std::is_void_v<R>) {
      op().redispatch(keys & c10::after_ADInplaceOrView_keyset, a...);
      (written(std::get<kWritten>(all)), ...);
    } else {
      R r = op().redispatch(keys & c10::after_ADInplaceOrView_keyset, a...);
      (written(std::get<kWritten>(all)), ...);
      return r;
    }
  }
};
using Append = Writer<kAppend, &append_kernel, 2, 3>;
using Copy = Writer<kCopy, &copy_kernel, 0, 1>;
using Fork = Writer<kFork, &fork_kernel, 0, 1, 2, 3, 4>;
using Keep = Writer<kKeep, &keep_kernel, 0, 1>;
using Free = Writer<kFree, &free_kernel, 0, 1>;

TORCH_LIBRARY_FRAGMENT(aotriton_amd, m) {
  const std::vector<at::Tag> compliant{at::Tag::pt2_compliant_tag};
  m.def("tree_attention(Tensor query, Tensor k_cache, Tensor v_cache, Tensor page_table, Tensor lengths, Tensor? parents, SymInt max_length, "
        "SymInt window, SymInt sinks, float sm_scale) -> (Tensor, Tensor)", compliant);
  m.def("cache_append(Tensor key, Tensor value, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor page_table, Tensor lengths, Tensor? counts) -> ()", compliant);
  m.def("cache_copy_pages(Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor source, Tensor target) -> ()", compliant);
  m.def("cache_fork(Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!) page_table, Tensor(d!) lengths, Tensor(e!) uses, Tensor source, "
        "Tensor target, Tensor spare) -> ()", compliant);
  m.def("cache_keep_path(Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor page_table, Tensor lengths, Tensor path, Tensor counts) -> Tensor", compliant);
  m.def("cache_free(Tensor(a!) page_table, Tensor(b!) uses, Tensor sequences, Tensor first, Tensor last) -> ()", compliant);
}
TORCH_LIBRARY_IMPL(aotriton_amd, CUDA, m) {
  m.impl("tree_attention", &tree_kernel);
  m.impl("cache_append", &append_kernel);
  m.impl("cache_copy_pages", &copy_kernel);
  m.impl("cache_fork", &fork_kernel);
  m.impl("cache_keep_path", &keep_kernel);
  m.impl("cache_free", &free_kernel);
}
TORCH_LIBRARY_IMPL(aotriton_amd, Autograd, m) {
  m.impl("tree_attention", &tree_autograd);
  m.impl("cache_append", &Append::autograd);
  m.impl("cache_copy_pages", &Copy::autograd);
  m.impl("cache_fork", &Fork::autograd);
  m.impl("cache_keep_path", &Keep::autograd);
  m.impl("cache_free", &Free::autograd);
}
TORCH_LIBRARY_IMPL(aotriton_amd, ADInplaceOrView, m) {
  m.impl("cache_append", &Append::inplace);
  m.impl("cache_copy_pages", &Copy::inplace);
  m.impl("cache_fork", &Fork::inplace);
  m.impl("cache_keep_path", &Keep::inplace);
  m.impl("cache_free", &Free::inplace);
}

}  // namespace
