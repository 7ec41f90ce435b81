// The operators of drafted decoding over a quantised pool, registered from
// C++ (a decode step makes several such calls, each of a few microseconds of
// GPU work): white_matter::kv_quant_store, kv_quant_read, tree_attention,
// token_scores and token_scores_bwd. What a user passes to the functions in
// kv_pool.py, tree_attention.py and token_scores.py is checked here, where a
// check costs nanoseconds (the same checks in Python took 6 of a decode step's
// 12 us); the CPU registrations and the _check operators serve the calls that
// end before a launch.
#include <ATen/core/dispatch/Dispatcher.h>
#include <torch/autograd.h>
#include <torch/library.h>

#include <c10/core/Allocator.h>

#include <cstring>
#include <initializer_list>
#include <limits>
#include <tuple>

#include "torch_common.h"

namespace {

using at::Tensor;
using c10::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using namespace wmx_torch;

// Device memory for the length of a call, from torch's caching allocator (on
// the current device and stream, and inside a capture from the graph's pool).
c10::DataPtr scratch(int64_t bytes) {
  return bytes > 0 ? c10::GetAllocator(c10::DeviceType::CUDA)->allocate((size_t)bytes) : c10::DataPtr();
}

void forward_only(const char* name, std::initializer_list<const Tensor*> tensors) {
  if (!at::GradMode::is_enabled()) return;
  for (const Tensor* t : tensors) TORCH_CHECK(!t || !t->defined() || !t->requires_grad(), name, " is forward-only");
}
const Tensor* given(const optional<Tensor>& t) { return t ? &*t : nullptr; }

bool int32_sizes(const Tensor& t) {
  for (const int64_t n : t.sizes())
    if (n > std::numeric_limits<int32_t>::max()) return false;
  return true;
}

int32_t pool_format(const Tensor& codes) {
  if (codes.scalar_type() == at::kFloat8_e4m3fn) return WMX_POOL_E4M3;
  TORCH_CHECK_VALUE(codes.scalar_type() == at::kChar, "pool codes must be float8_e4m3fn or int8");
  return WMX_POOL_INT8;
}

int32_t source_dtype(const Tensor& t) {
  if (t.scalar_type() == at::kFloat) return WMX_DTYPE_F32;
  TORCH_CHECK_TYPE(t.scalar_type() == at::kBFloat16, "keys, values, weights and tables must be float32 or bfloat16, got ", t.scalar_type());
  return WMX_DTYPE_BF16;
}

// Rows of unit stride that start 16-byte aligned (a copy otherwise).
Tensor aligned_rows(const Tensor& t) {
  bool ok = t.stride(-1) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int64_t d = 0; ok && d + 1 < t.dim(); ++d) ok = t.size(d) <= 1 || t.stride(d) * t.element_size() % 16 == 0;
  return ok ? t : dense16(t);
}

// Element strides of the first `n` dimensions; those of one element are never
// stepped over and count as 0.
void strides_of(const Tensor& t, int n, int64_t* out) {
  for (int d = 0; d < n; ++d) out[d] = t.size(d) > 1 ? t.stride(d) : 0;
}

void check_pool(const Tensor& codes, const Tensor& scales, const at::Device device, int64_t dims) {
  pool_format(codes);
  TORCH_CHECK_VALUE(scales.scalar_type() == at::kFloat, "pool scales must be float32");
  TORCH_CHECK_VALUE(codes.dim() == dims && scales.dim() == dims - 1 && codes.sizes().slice(0, dims - 1) == scales.sizes() && int32_sizes(codes),
                    "a quantised pool holds codes of ", dims, " dimensions and scales of the same shape without the last");
  TORCH_CHECK_VALUE(codes.device() == device && scales.device() == device, "the pool must be on the call's device");
  const int64_t dim = codes.size(-1);
  TORCH_CHECK_VALUE(dim == 64 || dim == 96 || dim == 128, "head_dim ", dim, " is not supported (64, 96 or 128)");
  bool rows = codes.stride(-1) == 1 && reinterpret_cast<uintptr_t>(codes.data_ptr()) % 8 == 0;
  for (int64_t d = 0; rows && d + 1 < dims; ++d) rows = codes.size(d) <= 1 || codes.stride(d) % 8 == 0;
  TORCH_CHECK_VALUE(rows, "pool views need unit stride along D and aligned rows of codes");
}

// Slots (T,) or (B, T) as int64 with unit stride, and the stride of a row.
Tensor slot_rows(const optional<Tensor>& slots, int64_t batch, int64_t tokens, const Tensor& like, int64_t& stride) {
  stride = 0;
  if (!slots) return Tensor();
  TORCH_CHECK_VALUE((slots->dim() == 1 && slots->size(0) == tokens) ||
                        (slots->dim() == 2 && slots->size(0) == batch && slots->size(1) == tokens),
                    "slots must be (T,) or (B, T)");
  TORCH_CHECK_VALUE(slots->scalar_type() == at::kLong || slots->scalar_type() == at::kInt, "slots must be integer");
  Tensor s = slots->to(like.device(), at::kLong);
  if (s.size(-1) > 1 && s.stride(-1) != 1) s = s.contiguous();
  if (s.dim() == 2) stride = s.size(0) > 1 ? s.stride(0) : 0;
  return s;
}

// ------------------------------------------------------ quantised pool ----
void kv_quant_store(const optional<Tensor>& key, const optional<Tensor>& value, const optional<Tensor>& weight,
                    const optional<Tensor>& cos, const optional<Tensor>& sin, const optional<Tensor>& slots,
                    const optional<Tensor>& key_codes, const optional<Tensor>& key_scales,
                    const optional<Tensor>& value_codes, const optional<Tensor>& value_scales, bool rope_by_slot,
                    double eps) {
  TORCH_CHECK_VALUE(key || value, "kv_quant_store needs keys or values");
  forward_only("the quantised pool write", {given(key), given(value), given(weight), given(cos), given(sin)});
  const Tensor& first = key ? *key : *value;
  TORCH_CHECK_VALUE(first.dim() == 5 && int32_sizes(first), "keys and values must be (B, C, H, T, D) of one shape");
  TORCH_CHECK_VALUE(!value || value->sizes() == first.sizes(), "key and value must be (B, C, H, T, D) of one shape");
  const int64_t batch = first.size(0), channels = first.size(1), heads = first.size(2), tokens = first.size(3), dim = first.size(4);
  wmx_kv_quant_args a;
  std::memset(&a, 0, sizeof(a));
  a.batch = (int32_t)batch;
  a.channels = (int32_t)channels;
  a.heads = (int32_t)heads;
  a.tokens = (int32_t)tokens;
  a.head_dim = (int32_t)dim;
  a.eps = (float)eps;
  a.rope_by_slot = rope_by_slot ? 1 : 0;
  a.pool_slots = -1;
  Tensor kept[2];  // the sources as the kernel reads them
  const struct {
    const optional<Tensor>&rows, &codes, &scales;
  } sides[2] = {{key, key_codes, key_scales}, {value, value_codes, value_scales}};
  for (int side = 0; side < 2; ++side) {
    const auto& s = sides[side];
    TORCH_CHECK_VALUE(s.rows.has_value() == s.codes.has_value() && s.rows.has_value() == s.scales.has_value(),
                      "a side's pool must be given exactly when its rows are");
    if (!s.rows) continue;
    TORCH_CHECK_VALUE(s.rows->sizes() == first.sizes() && s.rows->device() == first.device(), "key and value must be of one shape and device");
    source_dtype(*s.rows);
    check_pool(*s.codes, *s.scales, first.device(), 5);
    const auto n = s.codes->sizes();
    TORCH_CHECK_VALUE(n[0] == batch && n[1] == channels && n[2] == heads && n[4] == dim && (a.pool_slots < 0 || a.pool_slots == n[3]),
                      "the pool must be a (B, C, H, N, D) pool, of one shape for keys and values");
    TORCH_CHECK_VALUE(a.pool_slots < 0 || a.format == pool_format(*s.codes), "key and value pools must be of one code type");
    a.pool_slots = (int32_t)n[3];
    a.format = pool_format(*s.codes);
  }
  TORCH_CHECK_VALUE(key.has_value() == weight.has_value() && key.has_value() == cos.has_value() && key.has_value() == sin.has_value(),
                    "keys come with a norm weight, cos and sin");
  if (weight) {
    TORCH_CHECK_VALUE(weight->dim() == 2 && weight->size(0) == channels && weight->size(1) == dim && weight->device() == first.device(),
                      "k_norm_weight must be (C, D)");
    const bool tables = rope_by_slot ? cos->dim() == 2 && cos->size(0) == a.pool_slots && cos->size(1) == dim
                                     : cos->dim() == 3 && cos->size(0) == batch && cos->size(1) == tokens && cos->size(2) == dim;
    TORCH_CHECK_VALUE(tables && sin->sizes() == cos->sizes() && sin->scalar_type() == cos->scalar_type() &&
                          cos->device() == first.device() && sin->device() == first.device(),
                      "cos and sin must be (B, T, D), or with rope_by_slot (N, D) tables, of one dtype");
    source_dtype(*weight);
    source_dtype(*cos);
  }
  const Tensor at_slots = slot_rows(slots, batch, tokens, first, a.slots_stride);
  TORCH_CHECK(first.is_cuda(), "the quantised pool write runs on the HIP kernels: it takes GPU tensors");
  const c10::OptionalDeviceGuard guard(first.device());
  for (int side = 0; side < 2; ++side) {
    const auto& s = sides[side];
    if (!s.rows) continue;
    kept[side] = aligned_rows(*s.rows);
    (side ? a.value : a.key) = kept[side].data_ptr();
    (side ? a.value_dtype : a.key_dtype) = source_dtype(kept[side]);
    strides_of(kept[side], 4, side ? a.value_stride : a.key_stride);
    (side ? a.value_codes : a.key_codes) = s.codes->data_ptr();
    (side ? a.value_scales : a.key_scales) = s.scales->data_ptr<float>();
    strides_of(*s.codes, 4, side ? a.value_codes_stride : a.key_codes_stride);
    strides_of(*s.scales, 4, side ? a.value_scales_stride : a.key_scales_stride);
  }
  Tensor w, c, s;
  if (weight) {
    w = dense16(*weight);
    c = aligned_rows(*cos);
    s = aligned_rows(*sin);
    if (c.strides() != s.strides()) {
      c = dense16(c);
      s = dense16(s);
    }
    a.k_norm_weight = w.data_ptr();
    a.weight_dtype = source_dtype(w);
    a.cos = c.data_ptr();
    a.sin = s.data_ptr();
    a.rope_dtype = source_dtype(c);
    a.rope_stride[0] = !rope_by_slot && c.size(0) > 1 ? c.stride(0) : 0;
    a.rope_stride[1] = c.size(-2) > 1 ? c.stride(-2) : 0;
  }
  if (at_slots.defined()) a.slots = at_slots.data_ptr<int64_t>();
  check_rc(wmx_kv_quant_store(&a, stream_of(first)), "wmx_kv_quant_store");
}

Tensor kv_quant_read(const Tensor& codes, const Tensor& scales, const optional<Tensor>& slots) {
  check_pool(codes, scales, codes.device(), 5);
  forward_only("the pool read", {&scales});
  wmx_kv_read_args a;
  std::memset(&a, 0, sizeof(a));
  TORCH_CHECK_VALUE(!slots || slots->dim() >= 1, "slots must be (T,) or (B, T)");
  const int64_t tokens = slots ? slots->size(-1) : codes.size(3);
  const Tensor at_slots = slot_rows(slots, codes.size(0), tokens, codes, a.slots_stride);
  TORCH_CHECK(codes.is_cuda(), "the pool read runs on the HIP kernels: it takes GPU tensors");
  const c10::OptionalDeviceGuard guard(codes.device());
  Tensor out = at::empty({codes.size(0), codes.size(1), codes.size(2), tokens, codes.size(4)}, codes.options().dtype(at::kBFloat16));
  a.codes = codes.data_ptr();
  a.scales = scales.data_ptr<float>();
  a.slots = at_slots.defined() ? at_slots.data_ptr<int64_t>() : nullptr;
  a.out = out.data_ptr();
  strides_of(codes, 4, a.codes_stride);
  strides_of(scales, 4, a.scales_stride);
  a.format = pool_format(codes);
  a.batch = (int32_t)codes.size(0);
  a.channels = (int32_t)codes.size(1);
  a.heads = (int32_t)codes.size(2);
  TORCH_CHECK_VALUE(tokens <= std::numeric_limits<int32_t>::max(), "too many slots");
  a.tokens = (int32_t)tokens;
  a.head_dim = (int32_t)codes.size(4);
  a.pool_slots = (int32_t)codes.size(3);
  check_rc(wmx_kv_quant_read(&a, stream_of(codes)), "wmx_kv_quant_read");
  return out;
}

// ------------------------------------------------------ tree attention ----
void tree_attention_check(const Tensor& query, const Tensor& key, const Tensor& value, const optional<Tensor>& key_scales,
                          const optional<Tensor>& value_scales, const optional<Tensor>& kv_lengths, int64_t kv_length,
                          const optional<Tensor>& tree_mask, const optional<Tensor>& key_mask, bool use_dummy, double scale,
                          int64_t num_splits) {
  TORCH_CHECK_VALUE(key_scales.has_value() == value_scales.has_value(), "keys and values must both be tensors or both be quantised pools");
  if (key_scales) {
    check_pool(key, *key_scales, query.device(), 4);
    check_pool(value, *value_scales, query.device(), 4);
    TORCH_CHECK_VALUE(key.scalar_type() == value.scalar_type(), "key and value codes must be of one type");
  } else {
    TORCH_CHECK_VALUE(at::isFloatingType(key.scalar_type()) && at::isFloatingType(value.scalar_type()) && key.element_size() > 1 &&
                          value.element_size() > 1,
                      "keys and values must be floating point, or quantised pools");
  }
  TORCH_CHECK_VALUE(query.dim() == 4 && key.dim() == 4 && key.sizes() == value.sizes(), "Q/K/V require (B,H,T,D) tensors with matching K/V");
  const int64_t batch = query.size(0), nodes = query.size(2), slots = key.size(2);
  TORCH_CHECK_VALUE(key.size(0) == batch && key.size(3) == query.size(3) && key.size(1) > 0 && query.size(1) % key.size(1) == 0 &&
                        int32_sizes(query) && int32_sizes(key),
                    "Q/K/V require matching batch/head_dim and divisible heads");
  TORCH_CHECK_VALUE(key.device() == query.device() && value.device() == query.device(), "Q/K/V must share a device");
  TORCH_CHECK_VALUE(at::isFloatingType(query.scalar_type()), "queries must be floating point");
  forward_only("tree_attention", {&query, &key, &value, given(key_scales), given(value_scales)});
  TORCH_CHECK_VALUE(!kv_lengths || (kv_lengths->dim() == 1 && kv_lengths->size(0) == batch &&
                                    (kv_lengths->scalar_type() == at::kLong || kv_lengths->scalar_type() == at::kInt)),
                    "kv_lengths must be an integer or integer (B,)");
  TORCH_CHECK_VALUE(!tree_mask || (tree_mask->scalar_type() == at::kBool && tree_mask->device() == query.device() &&
                                   (tree_mask->dim() == 2 || (tree_mask->dim() == 3 && tree_mask->size(0) == batch)) &&
                                   tree_mask->size(-1) == nodes && tree_mask->size(-2) == nodes),
                    "tree_mask must be boolean (n,n) or (B,n,n) on the query's device");
  TORCH_CHECK_VALUE(!key_mask || (key_mask->scalar_type() == at::kBool && key_mask->device() == query.device() && key_mask->dim() == 2 &&
                                  key_mask->size(0) == batch && key_mask->size(1) == slots),
                    "key_mask must be boolean (B,N) on the query's device");
  TORCH_CHECK_VALUE(!use_dummy || slots > 0, "dummy-enabled K/V must contain the leading dummy slot");
  TORCH_CHECK_VALUE(num_splits >= 0 && num_splits <= std::numeric_limits<int32_t>::max(), "num_splits must not be negative");
  TORCH_CHECK(scale > 0, "tree_attention does not support softmax_scale ", scale);
}

Tensor tree_attention(const Tensor& query, const Tensor& key, const Tensor& value, const optional<Tensor>& key_scales,
                      const optional<Tensor>& value_scales, const optional<Tensor>& kv_lengths, int64_t kv_length,
                      const optional<Tensor>& tree_mask, const optional<Tensor>& key_mask, bool use_dummy, double scale,
                      int64_t num_splits) {
  tree_attention_check(query, key, value, key_scales, value_scales, kv_lengths, kv_length, tree_mask, key_mask, use_dummy, scale, num_splits);
  const c10::OptionalDeviceGuard guard(query.device());
  const int64_t batch = query.size(0), heads = query.size(1), nodes = query.size(2), dim = query.size(3);
  wmx_tree_args a;
  std::memset(&a, 0, sizeof(a));
  const Tensor q = operand(query);
  Tensor k = key, v = value, ks, vs;
  if (key_scales) {
    a.format = pool_format(key);
    const auto unit_slots = [](const Tensor& t) { return t.size(2) <= 1 || t.stride(2) == 1 ? t : t.contiguous(); };
    ks = unit_slots(*key_scales);
    vs = unit_slots(*value_scales);
    a.k_scales = ks.data_ptr<float>();
    a.v_scales = vs.data_ptr<float>();
    strides_of(ks, 2, a.k_scales_stride);
    strides_of(vs, 2, a.v_scales_stride);
  } else {
    a.format = WMX_POOL_BF16;
    k = operand(key);
    v = operand(value);
  }
  Tensor out = at::empty({batch, nodes, heads, dim}, q.options());
  a.q = q.data_ptr();
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.o = out.data_ptr();
  strides_of(q, 3, a.q_stride);
  strides_of(k, 3, a.k_stride);
  strides_of(v, 3, a.v_stride);
  a.o_stride[0] = out.stride(0);
  a.o_stride[1] = out.stride(2);
  a.o_stride[2] = out.stride(1);
  Tensor lengths, tree, mask;
  if (kv_lengths) {
    lengths = kv_lengths->to(q.device(), at::kLong).contiguous();
    a.kv_lengths = lengths.data_ptr<int64_t>();
  }
  a.kv_length_scalar = kv_length;
  if (tree_mask) {
    tree = tree_mask->stride(-1) == 1 ? *tree_mask : tree_mask->contiguous();
    a.tree_mask = (const uint8_t*)tree.data_ptr();
    a.tree_mask_stride[0] = tree.dim() == 3 && batch > 1 ? tree.stride(0) : 0;
    a.tree_mask_stride[1] = tree.stride(-2);
  }
  if (key_mask) {
    mask = key_mask->stride(1) == 1 ? *key_mask : key_mask->contiguous();
    a.key_mask = (const uint8_t*)mask.data_ptr();
    a.key_mask_stride = mask.stride(0);
  }
  a.batch = (int32_t)batch;
  a.q_heads = (int32_t)heads;
  a.kv_heads = (int32_t)key.size(1);
  a.nodes = (int32_t)nodes;
  a.capacity = (int32_t)key.size(2);
  a.head_dim = (int32_t)dim;
  a.use_dummy = use_dummy ? 1 : 0;
  a.num_splits = (int32_t)num_splits;
  a.softmax_scale = (float)scale;
  const int64_t need = wmx_tree_workspace_size(&a);
  const c10::DataPtr workspace = scratch(need);
  a.workspace = workspace.get();
  a.workspace_bytes = need;
  check_rc(wmx_tree_attn(&a, stream_of(q)), "wmx_tree_attn");
  return out;
}

// -------------------------------------------------------- token scores ----
// The stride of the equally spaced rows of (..., V) logits, unit along V.
bool even_rows(const Tensor& t, int64_t& stride) {
  stride = t.size(-1);
  if (t.size(-1) > 1 && t.stride(-1) != 1) return false;
  bool first = true;
  int64_t next = 0;
  for (int64_t d = t.dim() - 2; d >= 0; --d) {
    if (t.size(d) == 1) continue;
    if (first) stride = next = t.stride(d);
    else if (t.stride(d) != next) return false;
    first = false;
    next *= t.size(d);
  }
  return true;
}

void token_scores_check(const Tensor& logits, const Tensor& tokens, int64_t top_k) {
  const auto type = logits.scalar_type();
  TORCH_CHECK_TYPE(logits.dim() >= 1 && (type == at::kFloat || type == at::kBFloat16 || type == at::kHalf),
                   "logits must be float32, bfloat16 or float16 (..., V), got ", type);
  const auto ids = tokens.scalar_type();
  TORCH_CHECK_VALUE((ids == at::kLong || ids == at::kInt) && tokens.sizes() == logits.sizes().slice(0, logits.dim() - 1),
                    "tokens must be integer, one per row of logits");
  TORCH_CHECK_VALUE(tokens.device() == logits.device(), "tokens must be on the logits' device");
  const int64_t vocab = logits.size(-1), most = std::min<int64_t>(vocab, WMX_SCORE_MAX_TOP_K);
  TORCH_CHECK_VALUE(vocab >= 1 && vocab <= std::numeric_limits<int32_t>::max() - 65536 && top_k >= 0 && top_k <= most,
                    "top_k must be in [0, ", most, "] for ", vocab, " logits, got ", top_k);
}

// The arguments that both directions share; `rows`, `ids` keep what they point to.
void fill_scores(wmx_score_args& a, const Tensor& logits, const Tensor& tokens, int64_t ignore_index, Tensor& rows, Tensor& ids) {
  std::memset(&a, 0, sizeof(a));
  a.dtype = logits.scalar_type() == at::kFloat ? WMX_DTYPE_F32 : logits.scalar_type() == at::kBFloat16 ? WMX_DTYPE_BF16 : WMX_DTYPE_F16;
  rows = logits;
  if (!even_rows(rows, a.row_stride)) {
    rows = rows.contiguous();
    a.row_stride = logits.size(-1);
  }
  ids = tokens.to(at::kLong).contiguous();
  a.logits = rows.data_ptr();
  a.tokens = ids.data_ptr<int64_t>();
  a.rows = tokens.numel();
  a.vocab = (int32_t)logits.size(-1);
  a.ignore_index = ignore_index;
}

using Scores = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>;

// (log_probs, entropy, top_log_probs, top_indices, lse)
Scores token_scores(const Tensor& logits, const Tensor& tokens, int64_t top_k, int64_t ignore_index) {
  token_scores_check(logits, tokens, top_k);
  const c10::OptionalDeviceGuard guard(logits.device());
  wmx_score_args a;
  Tensor rows, ids;
  fill_scores(a, logits, tokens, ignore_index, rows, ids);
  a.top_k = (int32_t)top_k;
  const auto f32 = logits.options().dtype(at::kFloat);
  auto sizes = tokens.sizes().vec();
  Tensor log_probs = at::empty(sizes, f32), entropy = at::empty(sizes, f32), lse = at::empty(sizes, f32);
  sizes.push_back(top_k);
  Tensor top = at::empty(sizes, f32), indices = at::empty(sizes, ids.options());
  a.log_probs = log_probs.data_ptr<float>();
  a.entropy = entropy.data_ptr<float>();
  a.lse = lse.data_ptr<float>();
  a.top_log_probs = top.data_ptr<float>();
  a.top_indices = indices.data_ptr<int64_t>();
  a.workspace_bytes = wmx_score_workspace_size(&a);
  const c10::DataPtr workspace = scratch(a.workspace_bytes);
  a.workspace = workspace.get();
  check_rc(wmx_score(&a, stream_of(logits)), "wmx_score");
  return {log_probs, entropy, top, indices, lse};
}

Tensor token_scores_bwd(const Tensor& logits, const Tensor& tokens, const Tensor& entropy, const Tensor& lse, const Tensor& indices,
                        const optional<Tensor>& grad_log_probs, const optional<Tensor>& grad_entropy,
                        const optional<Tensor>& grad_top, int64_t ignore_index) {
  token_scores_check(logits, tokens, 0);
  const c10::OptionalDeviceGuard guard(logits.device());
  wmx_score_args a;
  Tensor rows, ids;
  fill_scores(a, logits, tokens, ignore_index, rows, ids);
  const int64_t n = a.rows;
  TORCH_CHECK_VALUE(indices.dim() == logits.dim() && indices.numel() == n * indices.size(-1) && indices.size(-1) <= WMX_SCORE_MAX_TOP_K &&
                        indices.scalar_type() == at::kLong,
                    "top indices must be int64 (..., k)");
  a.top_k = (int32_t)indices.size(-1);
  Tensor kept[6] = {entropy.contiguous(), lse.contiguous(), indices.contiguous()};
  const auto rows_of = [&](const optional<Tensor>& g, int64_t count, Tensor& keep) -> const float* {
    if (!g) return nullptr;
    TORCH_CHECK_VALUE(g->numel() == count && g->device() == logits.device(), "a gradient must be of its output's shape and device");
    keep = g->to(at::kFloat).contiguous();
    return keep.data_ptr<float>();
  };
  for (int i = 0; i < 2; ++i)
    TORCH_CHECK_VALUE(kept[i].numel() == n && kept[i].scalar_type() == at::kFloat, "entropy and lse must be float32 rows");
  for (int i = 0; i < 3; ++i) TORCH_CHECK_VALUE(kept[i].device() == logits.device(), "saved results must be on the logits' device");
  a.entropy = kept[0].data_ptr<float>();
  a.lse = kept[1].data_ptr<float>();
  a.top_indices = kept[2].data_ptr<int64_t>();
  a.grad_log_probs = rows_of(grad_log_probs, n, kept[3]);
  a.grad_entropy = rows_of(grad_entropy, n, kept[4]);
  a.grad_top = rows_of(grad_top, n * a.top_k, kept[5]);
  Tensor grad = at::empty(logits.sizes(), logits.options().memory_format(at::MemoryFormat::Contiguous));
  a.grad_logits = grad.data_ptr();
  check_rc(wmx_score_bwd(&a, stream_of(logits)), "wmx_score_bwd");
  return grad;
}

struct TokenScoresFn : public torch::autograd::Function<TokenScoresFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& tokens, int64_t top_k, int64_t ignore_index) {
    static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("white_matter::token_scores", "").typed<decltype(token_scores)>();
    at::AutoDispatchBelowADInplaceOrView below;
    auto [log_probs, entropy, top, indices, lse] = op.call(logits, tokens, top_k, ignore_index);
    ctx->save_for_backward({logits, tokens, entropy, lse, indices});
    ctx->saved_data["ignore"] = ignore_index;
    ctx->mark_non_differentiable({indices, lse});
    ctx->set_materialize_grads(false);
    return {log_probs, entropy, top, indices, lse};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    static auto op =
        c10::Dispatcher::singleton().findSchemaOrThrow("white_matter::token_scores_bwd", "").typed<decltype(token_scores_bwd)>();
    TORCH_CHECK(!at::GradMode::is_enabled(), "token_log_probs is differentiable once: its gradient has no gradient (create_graph)");
    const auto t = ctx->get_saved_variables();
    const auto opt = [](const Tensor& x) { return x.defined() ? optional<Tensor>(x) : c10::nullopt; };
    return {op.call(t[0], t[1], t[2], t[3], t[4], opt(grads[0]), opt(grads[1]), opt(grads[2]), ctx->saved_data["ignore"].toInt()),
            Tensor(), Tensor(), Tensor()};
  }
};

Scores token_scores_autograd(const Tensor& logits, const Tensor& tokens, int64_t top_k, int64_t ignore_index) {
  if (!at::GradMode::is_enabled() || !logits.requires_grad()) {
    static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("white_matter::token_scores", "").typed<decltype(token_scores)>();
    at::AutoDispatchBelowADInplaceOrView below;
    return op.call(logits, tokens, top_k, ignore_index);
  }
  auto r = TokenScoresFn::apply(logits, tokens, top_k, ignore_index);
  return {r[0], r[1], r[2], r[3], r[4]};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(white_matter, m) {
  m.def(
      "kv_quant_store(Tensor? key, Tensor? value, Tensor? weight, Tensor? cos, Tensor? sin, Tensor? slots, "
      "Tensor(a!)? key_codes, Tensor(b!)? key_scales, Tensor(c!)? value_codes, Tensor(d!)? value_scales, "
      "bool rope_by_slot, float eps) -> ()");
  m.def("kv_quant_read(Tensor codes, Tensor scales, Tensor? slots) -> Tensor");
  m.def(
      "tree_attention(Tensor query, Tensor key, Tensor value, Tensor? key_scales, Tensor? value_scales, Tensor? kv_lengths, "
      "int kv_length, Tensor? tree_mask, Tensor? key_mask, bool use_dummy, float scale, int num_splits) -> Tensor");
  m.def(
      "tree_attention_check(Tensor query, Tensor key, Tensor value, Tensor? key_scales, Tensor? value_scales, Tensor? kv_lengths, "
      "int kv_length, Tensor? tree_mask, Tensor? key_mask, bool use_dummy, float scale, int num_splits) -> ()",
      &tree_attention_check);
  m.def("token_scores_check(Tensor logits, Tensor tokens, int top_k) -> ()", &token_scores_check);
  m.def("token_scores(Tensor logits, Tensor tokens, int top_k, int ignore_index) -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def(
      "token_scores_bwd(Tensor logits, Tensor tokens, Tensor entropy, Tensor lse, Tensor top_indices, Tensor? grad_log_probs, "
      "Tensor? grad_entropy, Tensor? grad_top, int ignore_index) -> Tensor");
}

TORCH_LIBRARY_IMPL(white_matter, CUDA, m) {
  m.impl("kv_quant_store", &kv_quant_store);
  m.impl("kv_quant_read", &kv_quant_read);
  m.impl("tree_attention", &tree_attention);
  m.impl("token_scores", &token_scores);
  m.impl("token_scores_bwd", &token_scores_bwd);
}

// (refused after their checks: the kernels take GPU tensors)
TORCH_LIBRARY_IMPL(white_matter, CPU, m) {
  m.impl("kv_quant_store", &kv_quant_store);
  m.impl("kv_quant_read", &kv_quant_read);
}

TORCH_LIBRARY_IMPL(white_matter, Autograd, m) { m.impl("token_scores", &token_scores_autograd); }
