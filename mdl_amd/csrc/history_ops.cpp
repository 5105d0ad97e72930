// Operators over long histories (namespace mdl_hip), in C++: the window
// attention, its single-token form over a cache, the relative position bias
// and the norms around a block.  Each operator's ROCm kernel calls the C ABI
// of libmdl_hip.so on the current HIP stream; CPU and fake kernels are
// registered by mdl_amd/history.py and mdl_amd/block_norm.py on these schemas.
// Gradients are autograd nodes made here, so that a training step's Python is
// one call.

#include <ATen/ATen.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/library.h>

#include <algorithm>
#include <string>
#include <tuple>

#include "../../include/mdl_hip.h"
#include "torch_ops.h"

namespace mdl_torch {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

// A new contiguous tensor on t's device (allocated without a dispatcher round
// trip: a small training step makes a dozen of them).
Tensor empty_on(const Tensor& t, at::IntArrayRef sizes, at::ScalarType type) {
  return Tensor(at::detail::empty_cuda(sizes, type, t.device(), std::nullopt));
}

// The last dimension contiguous (any strides over the others).
Tensor inner_contiguous(const Tensor& t) { return t.size(-1) == 1 || t.stride(-1) == 1 ? t : t.contiguous(); }

void same_device(const Tensor& t, const Tensor& q, const char* what) {
  TORCH_CHECK_VALUE(t.device() == q.device(), what, " must live on the queries' device");
}

// The operators have no forward-mode formulas, and run below autograd where
// nothing requires a gradient: a dual input would lose its tangent there, so
// it is refused.
template <typename... Inputs>
void refuse_tangents(const char* what, const Inputs&... inputs) {
  TORCH_CHECK_NOT_IMPLEMENTED(!(torch::autograd::isFwGradDefined(inputs) || ...), what,
                              " has no forward-mode derivative");
}

// The gradients have no formula of their own: under create_graph they lead to
// a node that raises when it is differentiated, on the way to whatever they
// were made from (saved inputs, upstream gradients).
variable_list differentiable_once(const char* what, variable_list grads, const variable_list& saved,
                                  const variable_list& upstream) {
  if (!at::GradMode::is_enabled()) return grads;
  auto edges = torch::autograd::collect_next_edges(saved, upstream);
  if (std::none_of(edges.begin(), edges.end(), [](const torch::autograd::Edge& e) { return e.is_valid(); })) return grads;
  const auto node = std::make_shared<torch::autograd::Error>(
      std::string(what) + " can be differentiated once: its gradients have no derivative", std::move(edges));
  for (const Tensor& g : grads)
    if (g.defined()) torch::autograd::set_history(g, node);
  return grads;
}

// ------------------------------------------------------------- attention --

struct AttentionArgs {
  Tensor q, k, v, mask, table, starts;  // as the kernels read them (held while they run)
  mdl_attention call{};
};

void bias_args(const std::optional<Tensor>& bias_table, const std::optional<Tensor>& bucket_starts, int64_t distances,
               const Tensor& q, int64_t heads, Tensor& table, Tensor& starts) {
  TORCH_CHECK_VALUE(bucket_starts.has_value(), "a bias table needs its buckets");
  TORCH_CHECK_VALUE(bias_table->dim() == 2 && bias_table->size(1) == heads && bias_table->size(0) >= 1,
                    "bias_table must be [buckets, ", heads, "]");
  dtype_code(bias_table->scalar_type());
  same_device(*bias_table, q, "bias_table");
  same_device(*bucket_starts, q, "bucket_starts");
  TORCH_CHECK_VALUE(bucket_starts->scalar_type() == at::kInt && bucket_starts->dim() == 1 &&
                        bucket_starts->is_contiguous() && bucket_starts->size(0) == bias_table->size(0) - 1,
                    "bucket_starts must be contiguous int32 with one entry fewer than the table has buckets");
  TORCH_CHECK_VALUE(distances >= 1 && distances <= 2049, "bias buckets must begin at distances up to 2048");
  table = bias_table->contiguous();
  starts = *bucket_starts;
}

AttentionArgs attention_args(const Tensor& q, const Tensor& k, const Tensor& v, const std::optional<Tensor>& mask,
                             const std::optional<Tensor>& bias_table, const std::optional<Tensor>& bucket_starts,
                             int64_t distances, int64_t window, int64_t sinks, double scale) {
  require_device(q, "attention queries");
  TORCH_CHECK_VALUE(q.dim() == 4 && k.dim() == 4 && v.dim() == 4,
                    "attention takes q [B, Lq, Hq, D], k and v [B, Lk, Hkv, D]");
  TORCH_CHECK_VALUE(k.sizes() == v.sizes() && k.size(0) == q.size(0) && k.size(3) == q.size(3),
                    "attention queries, keys and values are misaligned");
  TORCH_CHECK_VALUE(q.size(2) > 0 && k.size(2) > 0 && q.size(2) % k.size(2) == 0,
                    "attention query heads must be a multiple of the key heads");
  TORCH_CHECK_VALUE(q.size(1) <= k.size(1), "attention queries are the last rows of the keys: more queries than keys");
  TORCH_CHECK_VALUE(q.size(3) >= 1 && q.size(3) <= 128, "attention head dimension must be 1 to 128");
  TORCH_CHECK_TYPE(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
                   "attention queries, keys and values must have one dtype");
  TORCH_CHECK_VALUE(window >= 0, "attention window must be positive");
  TORCH_CHECK_VALUE(sinks >= 0, "attention sinks must not be negative");
  TORCH_CHECK_VALUE(scale > 0 && scale < 1e30, "attention scale must be positive");
  same_device(k, q, "attention keys");
  same_device(v, q, "attention values");
  AttentionArgs a;
  mdl_attention& c = a.call;
  c.dtype = dtype_code(q.scalar_type());
  a.q = inner_contiguous(q);
  a.k = inner_contiguous(k);
  a.v = inner_contiguous(v);
  if (mask.has_value()) {
    TORCH_CHECK_VALUE(mask->dim() == 2 && mask->size(0) == k.size(0) && mask->size(1) == k.size(1),
                      "attention mask must be [B, Lk]");
    TORCH_CHECK_TYPE(mask->scalar_type() == at::kBool, "attention mask must be torch.bool");
    same_device(*mask, q, "attention mask");
    a.mask = inner_contiguous(*mask);
    c.mask = static_cast<const uint8_t*>(a.mask.data_ptr());
    c.mask_row = a.mask.stride(0);
  }
  if (bias_table.has_value()) {
    bias_args(bias_table, bucket_starts, distances, q, q.size(2), a.table, a.starts);
    c.bias_table = a.table.data_ptr();
    c.bucket_starts = static_cast<const int32_t*>(a.starts.data_ptr());
    c.table_dtype = dtype_code(a.table.scalar_type());
    c.num_buckets = (int32_t)a.table.size(0);
    c.distances = (int32_t)distances;
  }
  c.q = a.q.data_ptr(); c.k = a.k.data_ptr(); c.v = a.v.data_ptr();
  c.batch = q.size(0); c.q_len = q.size(1); c.k_len = k.size(1);
  c.q_batch = a.q.stride(0); c.q_row = a.q.stride(1); c.q_head = a.q.stride(2);
  c.k_batch = a.k.stride(0); c.k_row = a.k.stride(1); c.k_head = a.k.stride(2);
  c.v_batch = a.v.stride(0); c.v_row = a.v.stride(1); c.v_head = a.v.stride(2);
  c.window = window;
  c.sinks = sinks;
  c.q_heads = (int32_t)q.size(2); c.kv_heads = (int32_t)k.size(2); c.head_dim = (int32_t)q.size(3);
  c.scale = (float)scale;
  return a;
}

std::tuple<Tensor, Tensor, Tensor> attention_forward_cuda(
    const Tensor& q, const Tensor& k, const Tensor& v, const std::optional<Tensor>& mask,
    const std::optional<Tensor>& bias_table, const std::optional<Tensor>& bucket_starts, int64_t distances,
    int64_t window, int64_t sinks, double scale, bool need_backward) {
  const AttentionArgs a =
      attention_args(q, k, v, mask, bias_table, bucket_starts, distances, window, sinks, scale);
  c10::DeviceGuard guard(q.device());
  void* stream = stream_of(q.device());
  Tensor out = empty_on(q, q.sizes(), q.scalar_type());
  Tensor stats = need_backward ? empty_on(q, {q.size(0), q.size(2), q.size(1), 2}, at::kFloat)
                               : empty_on(q, {0}, at::kFloat);
  const size_t bytes = mdl_attention_prepared_bytes(&a.call);
  Tensor prepared = empty_on(q, {(int64_t)bytes}, at::kByte);
  check(mdl_attention_prepare(&a.call, prepared.data_ptr(), bytes, stream), "mdl_attention_prepare");
  check(mdl_attention_forward(&a.call, prepared.data_ptr(), out.data_ptr(),
                              need_backward ? static_cast<float*>(stats.data_ptr()) : nullptr, stream),
        "mdl_attention_forward");
  return {out, stats, prepared};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> attention_backward_cuda(
    const Tensor& grad_out, const Tensor& q, const Tensor& k, const Tensor& v, const std::optional<Tensor>& mask,
    const std::optional<Tensor>& bias_table, const std::optional<Tensor>& bucket_starts, int64_t distances,
    int64_t window, int64_t sinks, double scale, const Tensor& out, const Tensor& stats, const Tensor& prepared,
    bool need_table) {
  const AttentionArgs a =
      attention_args(q, k, v, mask, bias_table, bucket_starts, distances, window, sinks, scale);
  TORCH_CHECK_VALUE(grad_out.sizes() == q.sizes() && out.sizes() == q.sizes() && out.is_contiguous(),
                    "attention gradient and output must have the queries' shape");
  TORCH_CHECK_TYPE(grad_out.scalar_type() == q.scalar_type() && out.scalar_type() == q.scalar_type(),
                   "attention gradient and output must have the queries' dtype");
  TORCH_CHECK_VALUE(stats.numel() == 2 * q.size(0) * q.size(1) * q.size(2) && stats.scalar_type() == at::kFloat &&
                        stats.is_contiguous() && (size_t)prepared.numel() >= mdl_attention_prepared_bytes(&a.call),
                    "attention backward needs the forward's statistics");
  same_device(grad_out, q, "attention gradient");
  c10::DeviceGuard guard(q.device());
  const Tensor go = inner_contiguous(grad_out);
  Tensor dq = empty_on(q, q.sizes(), q.scalar_type());
  Tensor dk = empty_on(k, k.sizes(), k.scalar_type());
  Tensor dv = empty_on(v, v.sizes(), v.scalar_type());
  need_table = need_table && bias_table.has_value();
  Tensor dtable = need_table ? empty_on(q, bias_table->sizes(), bias_table->scalar_type())
                             : empty_on(q, {0}, q.scalar_type());
  if (q.numel() == 0) {
    dk.zero_();
    dv.zero_();
    dtable.zero_();
    return {dq, dk, dv, dtable};
  }
  mdl_attention_grads g{};
  g.out = out.data_ptr();
  g.stats = static_cast<const float*>(stats.data_ptr());
  g.grad_out = go.data_ptr();
  g.grad_batch = go.stride(0); g.grad_row = go.stride(1); g.grad_head = go.stride(2);
  g.grad_q = dq.data_ptr(); g.grad_k = dk.data_ptr(); g.grad_v = dv.data_ptr();
  g.grad_table = need_table ? dtable.data_ptr() : nullptr;
  const size_t bytes = mdl_attention_backward_workspace_bytes(&a.call);
  Tensor ws = empty_on(q, {(int64_t)bytes}, at::kByte);
  check(mdl_attention_backward(&a.call, prepared.data_ptr(), &g, ws.data_ptr(), bytes, stream_of(q.device())),
        "mdl_attention_backward");
  return {dq, dk, dv, dtable};
}

std::tuple<Tensor, Tensor, Tensor> call_attention_forward(
    const Tensor& q, const Tensor& k, const Tensor& v, const std::optional<Tensor>& mask,
    const std::optional<Tensor>& bias_table, const std::optional<Tensor>& bucket_starts, int64_t distances,
    int64_t window, int64_t sinks, double scale, bool need_backward) {
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("mdl_hip::history_attention_forward", "")
                             .typed<decltype(attention_forward_cuda)>();
  return op.call(q, k, v, mask, bias_table, bucket_starts, distances, window, sinks, scale, need_backward);
}

std::optional<Tensor> optional_of(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }

struct HistoryAttention : public torch::autograd::Function<HistoryAttention> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                        const std::optional<Tensor>& mask, const std::optional<Tensor>& bias_table,
                        const std::optional<Tensor>& bucket_starts, int64_t distances, int64_t window, int64_t sinks,
                        double scale) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [out, stats, prepared] =
        call_attention_forward(q, k, v, mask, bias_table, bucket_starts, distances, window, sinks, scale, true);
    ctx->save_for_backward({q, k, v, mask.value_or(Tensor()), bias_table.value_or(Tensor()),
                            bucket_starts.value_or(Tensor()), out, stats, prepared});
    ctx->saved_data["distances"] = distances;
    ctx->saved_data["window"] = window;
    ctx->saved_data["sinks"] = sinks;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["need_table"] = bias_table.has_value() && bias_table->requires_grad();
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = c10::Dispatcher::singleton()
                               .findSchemaOrThrow("mdl_hip::history_attention_backward", "")
                               .typed<decltype(attention_backward_cuda)>();
    const bool need_table = ctx->saved_data["need_table"].toBool();
    auto [dq, dk, dv, dtable] =
        op.call(grads[0], s[0], s[1], s[2], optional_of(s[3]), optional_of(s[4]), optional_of(s[5]),
                ctx->saved_data["distances"].toInt(), ctx->saved_data["window"].toInt(),
                ctx->saved_data["sinks"].toInt(), ctx->saved_data["scale"].toDouble(), s[6], s[7], s[8],
                need_table);
    const Tensor none;
    return differentiable_once("history_attention",
                               {dq, dk, dv, none, need_table ? dtable : none, none, none, none, none, none},
                               {s[0], s[1], s[2], s[4]}, grads);
  }
};

Tensor history_attention_autograd(const Tensor& q, const Tensor& k, const Tensor& v, const std::optional<Tensor>& mask,
                                  const std::optional<Tensor>& bias_table, const std::optional<Tensor>& bucket_starts,
                                  int64_t distances, int64_t window, int64_t sinks, double scale) {
  refuse_tangents("history_attention", q, k, v, bias_table);
  const bool need = at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad() ||
                                                   (bias_table.has_value() && bias_table->requires_grad()));
  if (need) return HistoryAttention::apply(q, k, v, mask, bias_table, bucket_starts, distances, window, sinks, scale);
  at::AutoDispatchBelowADInplaceOrView below;
  return std::get<0>(
      call_attention_forward(q, k, v, mask, bias_table, bucket_starts, distances, window, sinks, scale, false));
}

// ------------------------------------------------------ single new tokens --

// cache [B, capacity, Hkv, D]: the descriptor's cache and prompt or token sides.
mdl_attention_step cache_args(const Tensor& k, const Tensor& v, const Tensor& cache_k, const Tensor& cache_v,
                              int64_t sinks) {
  require_device(cache_k, "history cache");
  TORCH_CHECK_VALUE(cache_k.dim() == 4 && cache_k.sizes() == cache_v.sizes(),
                    "history cache keys and values must be [B, capacity, Hkv, D]");
  TORCH_CHECK_VALUE(cache_k.stride(3) == 1 && cache_v.stride(3) == 1,
                    "history cache rows must be contiguous in the head dimension");
  TORCH_CHECK_TYPE(cache_k.scalar_type() == cache_v.scalar_type() && k.scalar_type() == cache_k.scalar_type() &&
                       v.scalar_type() == cache_k.scalar_type(),
                   "history cache, keys and values must have one dtype");
  TORCH_CHECK_VALUE(sinks >= 0 && cache_k.size(1) > sinks, "history cache capacity must exceed its sinks");
  TORCH_CHECK_VALUE(cache_k.size(3) >= 1 && cache_k.size(3) <= 128, "attention head dimension must be 1 to 128");
  TORCH_CHECK_VALUE(cache_k.size(2) >= 1, "history cache needs a head");
  same_device(cache_v, cache_k, "history cache");
  same_device(k, cache_k, "keys");
  same_device(v, cache_k, "values");
  mdl_attention_step a{};
  a.dtype = dtype_code(cache_k.scalar_type());
  a.cache_k = cache_k.data_ptr();
  a.cache_v = cache_v.data_ptr();
  a.batch = cache_k.size(0);
  a.capacity = cache_k.size(1);
  a.kv_heads = a.q_heads = (int32_t)cache_k.size(2);
  a.head_dim = (int32_t)cache_k.size(3);
  a.ck_batch = cache_k.stride(0); a.ck_slot = cache_k.stride(1); a.ck_head = cache_k.stride(2);
  a.cv_batch = cache_v.stride(0); a.cv_slot = cache_v.stride(1); a.cv_head = cache_v.stride(2);
  a.sinks = sinks;
  return a;
}

// The kernels write the cache through its address: autograd learns of it here,
// as an in-place operation of its own would tell it.
void cache_changed(const Tensor& cache_k, const Tensor& cache_v) {
  for (const Tensor* t : {&cache_k, &cache_v})
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

void check_positions(const Tensor& t, const Tensor& cache, const char* what) {
  TORCH_CHECK_TYPE(t.scalar_type() == at::kLong, what, " must be torch.long");
  TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == cache.size(0), what, " must hold one entry per row of the cache");
  same_device(t, cache, what);
}

Tensor cache_step_cuda(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cache_k, const Tensor& cache_v,
                       const Tensor& positions, const std::optional<Tensor>& bias_table,
                       const std::optional<Tensor>& bucket_starts, int64_t distances, int64_t window, int64_t sinks,
                       double scale) {
  mdl_attention_step a = cache_args(k, v, cache_k, cache_v, sinks);
  TORCH_CHECK_VALUE(q.dim() == 3 && k.dim() == 3 && v.sizes() == k.sizes() && q.size(0) == a.batch &&
                        k.size(0) == a.batch && k.size(1) == a.kv_heads && k.size(2) == a.head_dim &&
                        q.size(2) == a.head_dim,
                    "a step takes q [B, Hq, D], k and v [B, Hkv, D] of the cache's rows");
  TORCH_CHECK_VALUE(q.size(1) > 0 && q.size(1) % a.kv_heads == 0,
                    "attention query heads must be a multiple of the key heads");
  TORCH_CHECK_TYPE(q.scalar_type() == cache_k.scalar_type(), "history cache and queries must have one dtype");
  TORCH_CHECK_VALUE(window >= 0 && window <= a.capacity - sinks,
                    "attention window must fit the cache beside its sinks");
  TORCH_CHECK_VALUE(scale > 0 && scale < 1e30, "attention scale must be positive");
  same_device(q, cache_k, "queries");
  check_positions(positions, cache_k, "positions");
  const Tensor qi = inner_contiguous(q), ki = inner_contiguous(k), vi = inner_contiguous(v);
  const Tensor at = positions.contiguous();
  Tensor table, starts;
  a.q_heads = (int32_t)q.size(1);
  if (bias_table.has_value()) {
    bias_args(bias_table, bucket_starts, distances, q, q.size(1), table, starts);
    a.bias_table = table.data_ptr();
    a.bucket_starts = static_cast<const int32_t*>(starts.data_ptr());
    a.table_dtype = dtype_code(table.scalar_type());
    a.num_buckets = (int32_t)table.size(0);
    a.distances = (int32_t)distances;
  }
  a.q = qi.data_ptr(); a.k = ki.data_ptr(); a.v = vi.data_ptr();
  a.q_batch = qi.stride(0); a.q_head = qi.stride(1);
  a.k_batch = ki.stride(0); a.k_head = ki.stride(1);
  a.v_batch = vi.stride(0); a.v_head = vi.stride(1);
  a.positions = static_cast<const int64_t*>(at.data_ptr());
  a.window = window;
  a.scale = (float)scale;
  c10::DeviceGuard guard(q.device());
  Tensor out = empty_on(q, q.sizes(), q.scalar_type());
  if (a.batch == 0) return out;
  const size_t bytes = mdl_attention_step_workspace_bytes(&a);
  Tensor ws;
  if (bytes) ws = empty_on(q, {(int64_t)bytes}, at::kByte);
  check(mdl_attention_step_forward(&a, out.data_ptr(), bytes ? ws.data_ptr() : nullptr, bytes, stream_of(q.device())),
        "mdl_attention_step_forward");
  cache_changed(cache_k, cache_v);
  return out;
}

void cache_write_cuda(const Tensor& k, const Tensor& v, const Tensor& cache_k, const Tensor& cache_v,
                      const Tensor& lengths, int64_t sinks, bool right_aligned) {
  mdl_attention_step a = cache_args(k, v, cache_k, cache_v, sinks);
  TORCH_CHECK_VALUE(k.dim() == 4 && v.sizes() == k.sizes() && k.size(0) == a.batch && k.size(2) == a.kv_heads &&
                        k.size(3) == a.head_dim,
                    "a prompt's k and v must be [B, L, Hkv, D] of the cache's rows");
  check_positions(lengths, cache_k, "lengths");
  const Tensor ki = inner_contiguous(k), vi = inner_contiguous(v), ln = lengths.contiguous();
  a.k = ki.data_ptr(); a.v = vi.data_ptr();
  a.k_batch = ki.stride(0); a.k_head = ki.stride(2);
  a.v_batch = vi.stride(0); a.v_head = vi.stride(2);
  if (k.numel() == 0) return;
  c10::DeviceGuard guard(k.device());
  check(mdl_attention_cache_write(&a, k.size(1), ki.stride(1), vi.stride(1), static_cast<const int64_t*>(ln.data_ptr()),
                                  right_aligned ? 1 : 0, stream_of(k.device())),
        "mdl_attention_cache_write");
  cache_changed(cache_k, cache_v);
}

// --------------------------------------------------- relative position bias --

void check_bias(const Tensor& table, const Tensor& starts, bool bidirectional, int64_t q_len, int64_t k_len) {
  require_device(table, "bias table");
  TORCH_CHECK_VALUE(table.dim() == 2 && table.size(0) >= 1 && table.size(1) >= 1, "bias table must be [buckets, heads]");
  dtype_code(table.scalar_type());
  same_device(starts, table, "bucket_starts");
  const int64_t side = bidirectional ? table.size(0) / 2 : table.size(0);
  TORCH_CHECK_VALUE(starts.scalar_type() == at::kInt && starts.dim() == 1 && starts.is_contiguous() &&
                        starts.size(0) == side - 1 && side * (bidirectional ? 2 : 1) == table.size(0),
                    "bucket_starts must be contiguous int32 with one entry fewer than a direction has buckets");
  TORCH_CHECK_VALUE(q_len >= 0 && q_len <= k_len, "a relative bias has 0 <= q_len <= k_len");
}

Tensor relative_bias_cuda(const Tensor& table, const Tensor& starts, bool bidirectional, int64_t q_len, int64_t k_len) {
  check_bias(table, starts, bidirectional, q_len, k_len);
  c10::DeviceGuard guard(table.device());
  const Tensor t = table.contiguous();
  Tensor out = empty_on(t, {t.size(1), q_len, k_len}, t.scalar_type());
  check(mdl_relative_bias(t.data_ptr(), static_cast<const int32_t*>(starts.data_ptr()), (int32_t)t.size(0),
                          bidirectional, (int32_t)t.size(1), q_len, k_len, dtype_code(t.scalar_type()), out.data_ptr(),
                          stream_of(t.device())),
        "mdl_relative_bias");
  return out;
}

Tensor relative_bias_grad_cuda(const Tensor& grad, const Tensor& starts, int64_t num_buckets, bool bidirectional) {
  require_device(grad, "bias gradient");
  TORCH_CHECK_VALUE(grad.dim() == 3 && grad.size(0) >= 1, "bias gradient must be [heads, q_len, k_len]");
  same_device(starts, grad, "bucket_starts");
  const int64_t side = bidirectional ? num_buckets / 2 : num_buckets;
  TORCH_CHECK_VALUE(starts.scalar_type() == at::kInt && starts.is_contiguous() && starts.numel() == side - 1,
                    "bucket_starts must be contiguous int32 with one entry fewer than a direction has buckets");
  const int32_t dtype = dtype_code(grad.scalar_type());
  c10::DeviceGuard guard(grad.device());
  const Tensor g = grad.contiguous();
  Tensor out = empty_on(g, {num_buckets, g.size(0)}, g.scalar_type());
  const size_t bytes =
      mdl_relative_bias_grad_workspace_bytes((int32_t)num_buckets, (int32_t)g.size(0), g.size(1), g.size(2), dtype);
  Tensor ws = empty_on(g, {(int64_t)bytes}, at::kByte);
  check(mdl_relative_bias_grad(g.data_ptr(), static_cast<const int32_t*>(starts.data_ptr()), (int32_t)num_buckets,
                               bidirectional, (int32_t)g.size(0), g.size(1), g.size(2), dtype, out.data_ptr(),
                               ws.data_ptr(), bytes, stream_of(g.device())),
        "mdl_relative_bias_grad");
  return out;
}

Tensor call_relative_bias(const Tensor& table, const Tensor& starts, bool bidirectional, int64_t q_len, int64_t k_len) {
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("mdl_hip::relative_position_bias_forward", "")
                             .typed<decltype(relative_bias_cuda)>();
  return op.call(table, starts, bidirectional, q_len, k_len);
}

struct RelativeBias : public torch::autograd::Function<RelativeBias> {
  static Tensor forward(AutogradContext* ctx, const Tensor& table, const Tensor& starts, bool bidirectional,
                        int64_t q_len, int64_t k_len) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->save_for_backward({starts});
    ctx->saved_data["buckets"] = table.size(0);
    ctx->saved_data["bidirectional"] = bidirectional;
    return call_relative_bias(table, starts, bidirectional, q_len, k_len);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = c10::Dispatcher::singleton()
                               .findSchemaOrThrow("mdl_hip::relative_position_bias_backward", "")
                               .typed<decltype(relative_bias_grad_cuda)>();
    const Tensor none;
    return differentiable_once("relative_position_bias",
                               {op.call(grads[0], ctx->get_saved_variables()[0], ctx->saved_data["buckets"].toInt(),
                                        ctx->saved_data["bidirectional"].toBool()),
                                none, none, none, none},
                               {}, grads);
  }
};

Tensor relative_bias_autograd(const Tensor& table, const Tensor& starts, bool bidirectional, int64_t q_len,
                              int64_t k_len) {
  refuse_tangents("relative_position_bias", table);
  if (at::GradMode::is_enabled() && table.requires_grad())
    return RelativeBias::apply(table, starts, bidirectional, q_len, k_len);
  at::AutoDispatchBelowADInplaceOrView below;
  return call_relative_bias(table, starts, bidirectional, q_len, k_len);
}

// ------------------------------------------------------ norms around a block --

struct NormArgs {
  Tensor x, o, gate, scale, post, next;
  mdl_block_norm call{};
};

NormArgs norm_args(const Tensor& x, const std::optional<Tensor>& block_out, const std::optional<Tensor>& post_weight,
                   const Tensor& next_weight, const std::optional<Tensor>& gate,
                   const std::optional<Tensor>& residual_scale, double eps) {
  require_device(x, "block norm input");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, "block norm input needs a last dimension");
  TORCH_CHECK_VALUE(eps >= 0, "block norm eps must not be negative");
  TORCH_CHECK_VALUE(block_out.has_value() || (!post_weight.has_value() && !gate.has_value() && !residual_scale.has_value()),
                    "gate, residual_scale and post_weight belong to a block's output");
  NormArgs a;
  const int64_t dim = x.size(-1);
  auto rows = [&](const Tensor& t, const char* what) {
    TORCH_CHECK_VALUE(t.sizes() == x.sizes(), what, " must have the input's shape");
    TORCH_CHECK_TYPE(t.scalar_type() == x.scalar_type(), what, " must have the input's dtype");
    same_device(t, x, what);
    return t.contiguous();
  };
  auto weight = [&](const Tensor& t, const char* what) {
    TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == dim, what, " must be [", dim, "]");
    TORCH_CHECK_TYPE(t.scalar_type() == next_weight.scalar_type(), "block norm weights must have one dtype");
    same_device(t, x, what);
    return t.contiguous();
  };
  a.x = x.contiguous();
  a.next = weight(next_weight, "next_weight");
  if (block_out.has_value()) a.o = rows(*block_out, "block_out");
  if (gate.has_value()) a.gate = rows(*gate, "gate");
  if (residual_scale.has_value()) a.scale = weight(*residual_scale, "residual_scale");
  if (post_weight.has_value()) a.post = weight(*post_weight, "post_weight");
  auto at = [](const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
  mdl_block_norm& c = a.call;
  c.x = at(a.x); c.block_out = at(a.o); c.gate = at(a.gate);
  c.residual_scale = at(a.scale); c.post_weight = at(a.post); c.next_weight = at(a.next);
  c.dim = (int32_t)dim;
  c.rows = x.numel() / dim;
  c.dtype = dtype_code(x.scalar_type());
  c.weight_dtype = dtype_code(next_weight.scalar_type());
  c.eps = (float)eps;
  TORCH_CHECK_VALUE(dim <= (c.dtype == MDL_BF16 ? 8192 : 4096),
                    "block norm rows hold at most 8192 (bfloat16) or 4096 (float32) elements");
  return a;
}

std::tuple<Tensor, Tensor, Tensor> block_norm_forward_cuda(
    const Tensor& x, const std::optional<Tensor>& block_out, const std::optional<Tensor>& post_weight,
    const Tensor& next_weight, const std::optional<Tensor>& gate, const std::optional<Tensor>& residual_scale,
    double eps) {
  NormArgs a = norm_args(x, block_out, post_weight, next_weight, gate, residual_scale, eps);
  c10::DeviceGuard guard(x.device());
  Tensor y = a.o.defined() ? empty_on(x, x.sizes(), x.scalar_type())
                           : empty_on(x, {0}, x.scalar_type());
  Tensor h = empty_on(x, x.sizes(), x.scalar_type());
  Tensor rstd = empty_on(x, {2, a.call.rows}, at::kFloat);
  if (a.call.rows == 0) return {y, h, rstd};
  a.call.rstd = static_cast<float*>(rstd.data_ptr());
  check(mdl_block_norm_forward(&a.call, a.o.defined() ? y.data_ptr() : nullptr, h.data_ptr(), stream_of(x.device())),
        "mdl_block_norm_forward");
  return {y, h, rstd};
}

// needs: residual_scale, post_weight, next_weight (bits 0 to 2).
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> block_norm_backward_cuda(
    const std::optional<Tensor>& grad_y, const std::optional<Tensor>& grad_h, const Tensor& x,
    const std::optional<Tensor>& block_out, const std::optional<Tensor>& post_weight, const Tensor& next_weight,
    const std::optional<Tensor>& gate, const std::optional<Tensor>& residual_scale, const Tensor& rstd, double eps,
    int64_t needs) {
  NormArgs a = norm_args(x, block_out, post_weight, next_weight, gate, residual_scale, eps);
  TORCH_CHECK_VALUE(rstd.numel() == 2 * a.call.rows && rstd.is_contiguous() && rstd.scalar_type() == at::kFloat,
                    "block norm backward needs the forward's statistics");
  a.call.rstd = static_cast<float*>(rstd.data_ptr());
  c10::DeviceGuard guard(x.device());
  Tensor dy, dh;
  auto incoming = [&](const std::optional<Tensor>& t) {
    if (!t.has_value() || !t->defined()) return Tensor();
    TORCH_CHECK_VALUE(t->sizes() == x.sizes(), "block norm gradients must have the input's shape");
    TORCH_CHECK_TYPE(t->scalar_type() == x.scalar_type(), "block norm gradients must have the input's dtype");
    same_device(*t, x, "block norm gradient");
    return t->contiguous();
  };
  dy = incoming(grad_y);
  dh = incoming(grad_h);
  auto like_x = [&](bool want) {
    return want ? empty_on(x, x.sizes(), x.scalar_type()) : empty_on(x, {0}, x.scalar_type());
  };
  auto like_w = [&](bool want) {
    return empty_on(x, {want ? (int64_t)a.call.dim : 0}, next_weight.scalar_type());
  };
  Tensor dx = like_x(true), d_o = like_x(a.o.defined()), dgate = like_x(a.gate.defined());
  Tensor dscale = like_w(a.scale.defined() && (needs & 1)), dpost = like_w(a.post.defined() && (needs & 2)),
         dnext = like_w(needs & 4);
  auto ptr = [](const Tensor& t) { return t.defined() && t.numel() ? t.data_ptr() : nullptr; };
  mdl_block_norm_grads g{};
  g.grad_y = ptr(dy); g.grad_h = ptr(dh);
  g.grad_x = ptr(dx); g.grad_block_out = ptr(d_o); g.grad_gate = ptr(dgate);
  g.grad_residual_scale = ptr(dscale); g.grad_post_weight = ptr(dpost); g.grad_next_weight = ptr(dnext);
  const size_t bytes = mdl_block_norm_backward_workspace_bytes(&a.call);
  Tensor ws = empty_on(x, {(int64_t)bytes}, at::kByte);
  check(mdl_block_norm_backward(&a.call, &g, ws.data_ptr(), bytes, stream_of(x.device())), "mdl_block_norm_backward");
  return {dx, d_o, dgate, dscale, dpost, dnext};
}

std::tuple<Tensor, Tensor, Tensor> call_block_norm(
    const Tensor& x, const std::optional<Tensor>& block_out, const std::optional<Tensor>& post_weight,
    const Tensor& next_weight, const std::optional<Tensor>& gate, const std::optional<Tensor>& residual_scale,
    double eps) {
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("mdl_hip::block_norm_forward", "")
                             .typed<decltype(block_norm_forward_cuda)>();
  return op.call(x, block_out, post_weight, next_weight, gate, residual_scale, eps);
}

struct BlockNorm : public torch::autograd::Function<BlockNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& block_out,
                               const std::optional<Tensor>& post_weight, const Tensor& next_weight,
                               const std::optional<Tensor>& gate, const std::optional<Tensor>& residual_scale,
                               double eps) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [y, h, rstd] = call_block_norm(x, block_out, post_weight, next_weight, gate, residual_scale, eps);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, block_out.value_or(Tensor()), post_weight.value_or(Tensor()), next_weight,
                            gate.value_or(Tensor()), residual_scale.value_or(Tensor()), rstd});
    ctx->saved_data["eps"] = eps;
    auto wants = [](const std::optional<Tensor>& t) { return t.has_value() && t->requires_grad(); };
    ctx->saved_data["needs"] = int64_t((wants(residual_scale) ? 1 : 0) | (wants(post_weight) ? 2 : 0) |
                                       (next_weight.requires_grad() ? 4 : 0));
    if (!block_out.has_value()) return {h};
    return {y, h};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor none;
    const auto s = ctx->get_saved_variables();
    const bool two = s[1].defined();
    const Tensor dy = two ? grads[0] : none, dh = grads[two ? 1 : 0];
    if (!dy.defined() && !dh.defined()) return {none, none, none, none, none, none, none};
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = c10::Dispatcher::singleton()
                               .findSchemaOrThrow("mdl_hip::block_norm_backward", "")
                               .typed<decltype(block_norm_backward_cuda)>();
    const int64_t needs = ctx->saved_data["needs"].toInt();
    auto [dx, d_o, dgate, dscale, dpost, dnext] =
        op.call(optional_of(dy), optional_of(dh), s[0], optional_of(s[1]), optional_of(s[2]), s[3], optional_of(s[4]),
                optional_of(s[5]), s[6], ctx->saved_data["eps"].toDouble(), needs);
    return differentiable_once("gated_residual_norm",
                               {dx, two ? d_o : none, needs & 2 ? dpost : none, needs & 4 ? dnext : none,
                                s[4].defined() ? dgate : none, needs & 1 ? dscale : none, none},
                               {s[0], s[1], s[2], s[3], s[4], s[5]}, grads);
  }
};

// (y, h); y is x itself without a block's output.
std::tuple<Tensor, Tensor> block_norm_autograd(const Tensor& x, const std::optional<Tensor>& block_out,
                                               const std::optional<Tensor>& post_weight, const Tensor& next_weight,
                                               const std::optional<Tensor>& gate,
                                               const std::optional<Tensor>& residual_scale, double eps) {
  refuse_tangents("gated_residual_norm", x, block_out, post_weight, next_weight, gate, residual_scale);
  auto wants = [](const std::optional<Tensor>& t) { return t.has_value() && t->requires_grad(); };
  if (at::GradMode::is_enabled() && (x.requires_grad() || next_weight.requires_grad() || wants(block_out) ||
                                     wants(post_weight) || wants(gate) || wants(residual_scale))) {
    auto out = BlockNorm::apply(x, block_out, post_weight, next_weight, gate, residual_scale, eps);
    if (!block_out.has_value()) return {x, out[0]};
    return {out[0], out[1]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  auto [y, h, rstd] = call_block_norm(x, block_out, post_weight, next_weight, gate, residual_scale, eps);
  return {block_out.has_value() ? y : x, h};
}

}  // namespace
}  // namespace mdl_torch

TORCH_LIBRARY_FRAGMENT(mdl_hip, m) {
  m.def("history_attention(Tensor q, Tensor k, Tensor v, Tensor? mask, Tensor? bias_table, Tensor? bucket_starts, "
        "int distances, int window, int sinks, float scale) -> Tensor",
        &mdl_torch::history_attention_autograd);
  m.def("history_attention_forward(Tensor q, Tensor k, Tensor v, Tensor? mask, Tensor? bias_table, "
        "Tensor? bucket_starts, int distances, int window, int sinks, float scale, bool need_backward) "
        "-> (Tensor, Tensor, Tensor)");
  m.def("history_attention_backward(Tensor grad_out, Tensor q, Tensor k, Tensor v, Tensor? mask, Tensor? bias_table, "
        "Tensor? bucket_starts, int distances, int window, int sinks, float scale, Tensor out, Tensor stats, "
        "Tensor prepared, bool need_table) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("history_cache_step(Tensor q, Tensor k, Tensor v, Tensor(a!) cache_k, Tensor(b!) cache_v, Tensor positions, "
        "Tensor? bias_table, Tensor? bucket_starts, int distances, int window, int sinks, float scale) -> Tensor");
  m.def("history_cache_write_(Tensor k, Tensor v, Tensor(a!) cache_k, Tensor(b!) cache_v, Tensor lengths, int sinks, "
        "bool right_aligned) -> ()");
  m.def("relative_position_bias(Tensor table, Tensor bucket_starts, bool bidirectional, int q_len, int k_len) -> Tensor",
        &mdl_torch::relative_bias_autograd);
  m.def("relative_position_bias_forward(Tensor table, Tensor bucket_starts, bool bidirectional, int q_len, int k_len) "
        "-> Tensor");
  m.def("relative_position_bias_backward(Tensor grad, Tensor bucket_starts, int num_buckets, bool bidirectional) "
        "-> Tensor");
  m.def("gated_residual_norm(Tensor x, Tensor? block_out, Tensor? post_weight, Tensor next_weight, Tensor? gate, "
        "Tensor? residual_scale, float eps) -> (Tensor, Tensor)",
        &mdl_torch::block_norm_autograd);
  m.def("block_norm_forward(Tensor x, Tensor? block_out, Tensor? post_weight, Tensor next_weight, Tensor? gate, "
        "Tensor? residual_scale, float eps) -> (Tensor, Tensor, Tensor)");
  m.def("block_norm_backward(Tensor? grad_y, Tensor? grad_h, Tensor x, Tensor? block_out, Tensor? post_weight, "
        "Tensor next_weight, Tensor? gate, Tensor? residual_scale, Tensor rstd, float eps, int needs) "
        "-> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(mdl_hip, CUDA, m) {
  using namespace mdl_torch;
  m.impl("history_attention_forward", &attention_forward_cuda);
  m.impl("history_attention_backward", &attention_backward_cuda);
  m.impl("history_cache_step", &cache_step_cuda);
  m.impl("history_cache_write_", &cache_write_cuda);
  m.impl("relative_position_bias_forward", &relative_bias_cuda);
  m.impl("relative_position_bias_backward", &relative_bias_grad_cuda);
  m.impl("block_norm_forward", &block_norm_forward_cuda);
  m.impl("block_norm_backward", &block_norm_backward_cuda);
}

// Inference: nothing to differentiate, and no call of the dispatcher's boxed
// fallback for a missing autograd kernel.
TORCH_LIBRARY_IMPL(mdl_hip, Autograd, m) {
  m.impl("history_cache_step", torch::CppFunction::makeFallthrough());
  m.impl("history_cache_write_", torch::CppFunction::makeFallthrough());
}
TORCH_LIBRARY_IMPL(mdl_hip, ADInplaceOrView, m) {
  m.impl("history_cache_step", torch::CppFunction::makeFallthrough());
  m.impl("history_cache_write_", torch::CppFunction::makeFallthrough());
}
