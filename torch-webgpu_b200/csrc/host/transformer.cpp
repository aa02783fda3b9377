// The `webgpu::` ops for the passes of a transformer between its matrix products: rotation by
// positions, the norm of queries and keys with it, dropout from a counter-based generator, and the log
// probabilities of given tokens - with their gradients, and `aten::dropout` on top of the third.
//
// No counterpart in the reference, whose op list (README.md:106-166) ends with the pointwise ops.
// Each op checks its arguments, allocates its results and makes one library call on the tensors'
// device and current stream.  The kernels also carry Meta implementations (shapes and checks
// without a device), which is what torch.compile traces through.
#include <ATen/core/dispatch/Dispatcher.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <mutex>

#include "twg_host.h"

namespace torch_webgpu {
namespace ops {

using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;
using OptTensor = std::optional<at::Tensor>;

static bool given(const OptTensor& t) { return t.has_value() && t->defined(); }

static int dtype_of(const char* name, const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return TWG_DTYPE_F32;
    case at::kHalf: return TWG_DTYPE_F16;
    case at::kBFloat16: return TWG_DTYPE_BF16;
    default: TORCH_CHECK(false, "torch_webgpu: ", name, " supports float32, float16 and bfloat16 tensors, got ", t.scalar_type());
  }
}
static int index_dtype_of(const char* name, const char* what, const at::Tensor& t) {
  TORCH_CHECK(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, "torch_webgpu: ", name, ": ", what,
              " must be int32 or int64, got ", t.scalar_type());
  return t.scalar_type() == at::kLong ? TWG_DTYPE_I64 : TWG_DTYPE_I32;
}
static void same_device(const char* name, const at::Tensor& a, const at::Tensor& b) {
  TORCH_CHECK(a.device() == b.device(), "torch_webgpu: ", name, " expects all tensors on one device, got ", a.device(), " and ", b.device());
}
static c10::DeviceIndex tensor_device(const at::Tensor& t) {
  return t.device().index() < 0 ? core::current_device() : t.device().index();
}

// Shapes of a traced graph may be symbols; the checks then wait for the call with the sizes themselves.
static bool symbolic(const at::Tensor& t) { return t.unsafeGetTensorImpl()->has_symbolic_sizes_strides(); }

// ---- rotation, and the norm of queries and keys in front of it -----------------------------
// q and k: [batch, seq, heads, dim] or [tokens, heads, dim].
static void put_strides(int64_t (&out)[4], const at::Tensor& t) {
  const int64_t d = t.dim();
  out[0] = d == 4 ? t.stride(0) : 0;
  for (int k = 1; k < 4; ++k) out[k] = t.stride(d - 4 + k);
}

struct Rotary {
  TwgRotaryDesc d;
  at::Tensor positions, inv_freq;  // as the descriptor describes them
};

static Rotary describe_rotary(const char* name, const at::Tensor& q, const at::Tensor* k, const at::Tensor& positions,
                              const at::Tensor& inv_freq, c10::IntArrayRef axis_of, bool adjacent) {
  Rotary r;
  std::memset(&r.d, 0, sizeof(r.d));
  TwgRotaryDesc& d = r.d;
  d.dtype = dtype_of(name, q);
  TORCH_CHECK(q.dim() == 3 || q.dim() == 4, "torch_webgpu: ", name, " expects [batch, seq, heads, dim] or [tokens, heads, dim], got ",
              q.dim(), " dimensions");
  const int64_t n = q.dim();
  if (k) {
    same_device(name, q, *k);
    TORCH_CHECK(k->scalar_type() == q.scalar_type(), "torch_webgpu: ", name, ": q and k must be of one type, got ", q.scalar_type(), " and ",
                k->scalar_type());
    TORCH_CHECK(k->dim() == n, "torch_webgpu: ", name, ": q and k must have as many dimensions, got ", n, " and ", k->dim());
    for (int64_t i = 0; i < n; ++i)
      TORCH_CHECK(i == n - 2 || k->size(i) == q.size(i), "torch_webgpu: ", name, ": q and k may differ in their heads only, got ", q.sizes(),
                  " and ", k->sizes());
  }
  d.batch = n == 4 ? q.size(0) : 1;
  d.seq = q.size(n - 3);
  d.heads[0] = q.size(n - 2);
  d.heads[1] = k ? k->size(n - 2) : 0;
  TORCH_CHECK(q.size(n - 1) >= 2 && q.size(n - 1) <= 512, "torch_webgpu: ", name, " supports heads of 2 to 512 elements, got ", q.size(n - 1));
  d.head_dim = static_cast<int32_t>(q.size(n - 1));

  same_device(name, q, inv_freq);
  TORCH_CHECK(inv_freq.dim() == 1, "torch_webgpu: ", name, ": inv_freq must have one dimension");
  TORCH_CHECK(inv_freq.scalar_type() == at::kFloat || inv_freq.scalar_type() == at::kDouble, "torch_webgpu: ", name,
              ": inv_freq must be float32 or float64, got ", inv_freq.scalar_type());
  TORCH_CHECK(inv_freq.size(0) >= 1 && 2 * inv_freq.size(0) <= d.head_dim, "torch_webgpu: ", name, ": ", inv_freq.size(0),
              " frequencies turn ", 2 * inv_freq.size(0), " elements of a head of ", d.head_dim);
  d.freq_dtype = inv_freq.scalar_type() == at::kDouble ? TWG_DTYPE_F64 : TWG_DTYPE_F32;
  d.rot_dim = static_cast<int32_t>(2 * inv_freq.size(0));
  r.inv_freq = inv_freq.contiguous();

  // positions: [axes, <tokens>], or without the axes; <tokens> is [batch, seq] or [seq], and may be
  // one of every batch (size 1, or [seq] beside a batch of q)
  same_device(name, q, positions);
  d.position_dtype = index_dtype_of(name, "positions", positions);
  const int64_t tokens_dims = n - 2;
  at::Tensor pos = positions;
  TORCH_CHECK(pos.dim() >= 1 && pos.dim() <= tokens_dims + 1, "torch_webgpu: ", name, ": positions of ", positions.sizes(),
              " do not belong to tokens of ", q.sizes().slice(0, tokens_dims));
  const bool with_axes = pos.dim() == tokens_dims + 1;
  d.axes = with_axes ? static_cast<int32_t>(std::min<int64_t>(pos.size(0), 1 << 20)) : 1;
  TORCH_CHECK(d.axes >= 1 && d.axes <= 8, "torch_webgpu: ", name, ": positions on 1 to 8 axes are supported, got ", d.axes);
  std::vector<int64_t> want;
  if (with_axes) want.push_back(pos.size(0));
  if (n == 4 && (with_axes || pos.dim() == 2)) want.push_back(d.batch);
  want.push_back(d.seq);
  for (size_t i = with_axes ? 1 : 0; i < want.size(); ++i) {
    const bool is_batch = i + 1 < want.size();
    TORCH_CHECK(pos.size(i) == want[i] || (is_batch && pos.size(i) == 1), "torch_webgpu: ", name, ": positions of ", positions.sizes(),
                " do not belong to tokens of ", q.sizes().slice(0, tokens_dims));
  }
  r.positions = pos;
  const int64_t last = pos.dim() - 1, lead = last - (with_axes ? 1 : 0);  // lead: batch dimensions before seq
  d.position_strides[0] = with_axes ? pos.stride(0) : 0;
  d.position_strides[1] = lead == 1 && pos.size(last - 1) > 1 ? pos.stride(last - 1) : 0;
  d.position_strides[2] = pos.stride(last);

  TORCH_CHECK(axis_of.empty() ? d.axes == 1 : static_cast<int64_t>(axis_of.size()) == inv_freq.size(0), "torch_webgpu: ", name,
              ": axis_of must name the axis of each of the ", inv_freq.size(0), " frequencies");
  for (size_t j = 0; j < axis_of.size(); ++j) {
    TORCH_CHECK(axis_of[j] >= 0 && axis_of[j] < d.axes, "torch_webgpu: ", name, ": frequency ", j, " belongs to axis ", axis_of[j], " of ", d.axes);
    d.axis_of[j] = static_cast<uint8_t>(axis_of[j]);
  }
  d.adjacent = adjacent;
  d.weight_dtype = d.dtype;
  put_strides(d.in_strides[0], q);
  if (k) put_strides(d.in_strides[1], *k);
  return r;
}

static void check_weight(const char* name, const at::Tensor& q, const OptTensor& w) {
  if (!given(w)) return;
  same_device(name, q, *w);
  TORCH_CHECK(w->dim() == 1 && w->size(0) == q.size(-1), "torch_webgpu: ", name, ": a weight must have ", q.size(-1), " elements, got ", w->sizes());
  TORCH_CHECK(w->scalar_type() == q.scalar_type() || w->scalar_type() == at::kFloat, "torch_webgpu: ", name,
              ": weights must be float32 or of q's type, got ", w->scalar_type());
}
static at::Tensor weight_or_none(const OptTensor& w) { return given(w) ? w->contiguous() : at::Tensor(); }
static const void* ptr_or_null(const at::Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
static void set_weight_dtype(const char* name, TwgRotaryDesc& d, const OptTensor& qw, const OptTensor& kw) {
  if (given(qw) && given(kw))
    TORCH_CHECK(qw->scalar_type() == kw->scalar_type(), "torch_webgpu: ", name, ": the two weights must be of one type");
  const OptTensor& w = given(qw) ? qw : kw;
  if (given(w) && w->scalar_type() == at::kFloat) d.weight_dtype = TWG_DTYPE_F32;
}

static std::tuple<at::Tensor, at::Tensor> run_rotary(const char* name, const at::Tensor& q, const at::Tensor* k, const at::Tensor& positions,
                                                     const at::Tensor& inv_freq, c10::IntArrayRef axis_of, bool adjacent, bool inverse) {
  if (symbolic(q) || (k && symbolic(*k)) || symbolic(positions)) return {at::empty_like(q), k ? at::empty_like(*k) : at::Tensor()};
  Rotary r = describe_rotary(name, q, k, positions, inv_freq, axis_of, adjacent);
  at::Tensor qo = at::empty_like(q), ko;
  if (k) ko = at::empty_like(*k);
  if (q.is_meta()) return {qo, ko};
  r.d.inverse = inverse;
  put_strides(r.d.out_strides[0], qo);
  if (k) put_strides(r.d.out_strides[1], ko);
  const c10::DeviceIndex dev = tensor_device(q);
  core::DeviceScope scope(dev);
  TWG_TORCH_CHECK(twg_rotary(&r.d, q.const_data_ptr(), k ? k->const_data_ptr() : nullptr, r.positions.const_data_ptr(),
                             r.inv_freq.const_data_ptr(), qo.data_ptr(), k ? ko.data_ptr() : nullptr, core::current_stream(dev)));
  return {qo, ko};
}
at::Tensor rotary(const at::Tensor& x, const at::Tensor& positions, const at::Tensor& inv_freq, c10::IntArrayRef axis_of, bool adjacent,
                  bool inverse) {
  return std::get<0>(run_rotary("rotary", x, nullptr, positions, inv_freq, axis_of, adjacent, inverse));
}
std::tuple<at::Tensor, at::Tensor> rotary_qk(const at::Tensor& q, const at::Tensor& k, const at::Tensor& positions, const at::Tensor& inv_freq,
                                             c10::IntArrayRef axis_of, bool adjacent, bool inverse) {
  return run_rotary("rotary_qk", q, &k, positions, inv_freq, axis_of, adjacent, inverse);
}

std::tuple<at::Tensor, at::Tensor> qk_norm_rotary(const at::Tensor& q, const at::Tensor& k, const OptTensor& q_weight, const OptTensor& k_weight,
                                                  const at::Tensor& positions, const at::Tensor& inv_freq, c10::IntArrayRef axis_of, double eps,
                                                  bool adjacent) {
  const char* name = "qk_norm_rotary";
  if (symbolic(q) || symbolic(k) || symbolic(positions)) return {at::empty_like(q), at::empty_like(k)};
  Rotary r = describe_rotary(name, q, &k, positions, inv_freq, axis_of, adjacent);
  TORCH_CHECK(eps >= 0, "torch_webgpu: qk_norm_rotary: eps must not be negative");
  check_weight(name, q, q_weight);
  check_weight(name, q, k_weight);
  set_weight_dtype(name, r.d, q_weight, k_weight);
  at::Tensor qo = at::empty_like(q), ko = at::empty_like(k);
  if (q.is_meta()) return {qo, ko};
  const at::Tensor qw = weight_or_none(q_weight), kw = weight_or_none(k_weight);
  r.d.eps = static_cast<float>(eps);
  put_strides(r.d.out_strides[0], qo);
  put_strides(r.d.out_strides[1], ko);
  const c10::DeviceIndex dev = tensor_device(q);
  core::DeviceScope scope(dev);
  TWG_TORCH_CHECK(twg_qk_norm_rotary(&r.d, q.const_data_ptr(), k.const_data_ptr(), ptr_or_null(qw), ptr_or_null(kw),
                                     r.positions.const_data_ptr(), r.inv_freq.const_data_ptr(), qo.data_ptr(), ko.data_ptr(),
                                     core::current_stream(dev)));
  return {qo, ko};
}

// The gradients of absent weights are empty tensors.
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> qk_norm_rotary_backward(
    const at::Tensor& dq_out, const at::Tensor& dk_out, const at::Tensor& q, const at::Tensor& k, const OptTensor& q_weight,
    const OptTensor& k_weight, const at::Tensor& positions, const at::Tensor& inv_freq, c10::IntArrayRef axis_of, double eps, bool adjacent) {
  const char* name = "qk_norm_rotary_backward";
  if (symbolic(q) || symbolic(k) || symbolic(positions)) {
    auto like = [&](const OptTensor& w) { return given(w) ? at::empty_like(*w) : at::empty({0}, q.options()); };
    return {at::empty_like(q), at::empty_like(k), like(q_weight), like(k_weight)};
  }
  Rotary r = describe_rotary(name, q, &k, positions, inv_freq, axis_of, adjacent);
  TORCH_CHECK(eps >= 0, "torch_webgpu: qk_norm_rotary_backward: eps must not be negative");
  check_weight(name, q, q_weight);
  check_weight(name, q, k_weight);
  set_weight_dtype(name, r.d, q_weight, k_weight);
  for (const auto& [g, x] : {std::tie(dq_out, q), std::tie(dk_out, k)}) {
    same_device(name, x, g);
    TORCH_CHECK(g.sizes() == x.sizes() && g.scalar_type() == x.scalar_type(), "torch_webgpu: ", name, ": a gradient of ", g.sizes(), " ",
                g.scalar_type(), " does not belong to ", x.sizes(), " ", x.scalar_type());
  }
  at::Tensor dq = at::empty_like(q), dk = at::empty_like(k);
  const at::Tensor qw = weight_or_none(q_weight), kw = weight_or_none(k_weight);
  at::Tensor dqw = qw.defined() ? at::empty_like(qw) : at::empty({0}, q.options());
  at::Tensor dkw = kw.defined() ? at::empty_like(kw) : at::empty({0}, q.options());
  if (q.is_meta()) return {dq, dk, dqw, dkw};
  r.d.eps = static_cast<float>(eps);
  put_strides(r.d.out_strides[0], dq);
  put_strides(r.d.out_strides[1], dk);
  put_strides(r.d.grad_strides[0], dq_out);
  put_strides(r.d.grad_strides[1], dk_out);
  const c10::DeviceIndex dev = tensor_device(q);
  core::DeviceScope scope(dev);
  const size_t bytes = twg_qk_norm_rotary_workspace_bytes(&r.d);
  TORCH_CHECK(bytes != 0, "torch_webgpu: ", twg_last_error());
  at::Tensor ws = at::empty({static_cast<int64_t>(bytes)}, q.options().dtype(at::kByte));
  TWG_TORCH_CHECK(twg_qk_norm_rotary_backward(
      &r.d, q.const_data_ptr(), k.const_data_ptr(), ptr_or_null(qw), ptr_or_null(kw), r.positions.const_data_ptr(), r.inv_freq.const_data_ptr(),
      dq_out.const_data_ptr(), dk_out.const_data_ptr(), dq.data_ptr(), dk.data_ptr(), qw.defined() ? dqw.data_ptr() : nullptr,
      kw.defined() ? dkw.data_ptr() : nullptr, ws.data_ptr(), bytes, core::current_stream(dev)));
  return {dq, dk, dqw, dkw};
}

// ---- dropout -----------------------------------------------------------------------------------
static at::Tensor run_dropout(const at::Tensor& x, double p, uint64_t seed, int64_t offset, const at::Tensor* state, const OptTensor& residual) {
  if (symbolic(x)) return at::empty_like(x);
  const int dtype = dtype_of("dropout", x);
  TORCH_CHECK(p >= 0 && p <= 1, "dropout probability has to be between 0 and 1, but got ", p);
  TORCH_CHECK(x.dim() <= TWG_MAX_DIMS, "torch_webgpu: dropout supports at most ", TWG_MAX_DIMS, " dimensions, got ", x.dim());
  if (given(residual)) {
    same_device("dropout", x, *residual);
    TORCH_CHECK(residual->sizes() == x.sizes() && residual->scalar_type() == x.scalar_type(), "torch_webgpu: dropout: the residual must have x's shape and type, got ",
                residual->sizes(), " ", residual->scalar_type(), " beside ", x.sizes(), " ", x.scalar_type());
  }
  if (state) {
    same_device("dropout", x, *state);
    TORCH_CHECK(state->scalar_type() == at::kLong && state->dim() == 1 && state->size(0) == 2 && state->is_contiguous(),
                "torch_webgpu: dropout: state must be a contiguous int64 tensor {seed, offset}");
  }
  at::Tensor out = at::empty_like(x);
  if (x.is_meta() || x.numel() == 0) return out;
  TwgIterDesc d;
  std::memset(&d, 0, sizeof(d));
  d.ndim = static_cast<int32_t>(x.dim());
  d.ntensors = given(residual) ? 3 : 2;
  d.numel = x.numel();
  const at::Tensor* operands[3] = {&out, &x, given(residual) ? &*residual : nullptr};
  for (int k = 0; k < d.ndim; ++k) {  // dimension 0 of the descriptor is the last logical one
    const int64_t dim = d.ndim - 1 - k;
    d.shape[k] = x.size(dim);
    for (int t = 0; t < d.ntensors; ++t) d.strides[t][k] = x.size(dim) == 1 ? 0 : operands[t]->stride(dim);
  }
  const c10::DeviceIndex dev = tensor_device(x);
  core::DeviceScope scope(dev);
  TWG_TORCH_CHECK(twg_dropout(&d, dtype, x.const_data_ptr(), given(residual) ? residual->const_data_ptr() : nullptr, out.data_ptr(), p, seed,
                              static_cast<uint64_t>(offset), state ? static_cast<const uint64_t*>(state->const_data_ptr()) : nullptr,
                              core::current_stream(dev)));
  return out;
}
at::Tensor dropout(const at::Tensor& x, double p, int64_t seed, int64_t offset, const OptTensor& residual) {
  return run_dropout(x, p, static_cast<uint64_t>(seed), offset, nullptr, residual);
}
at::Tensor dropout_state(const at::Tensor& x, double p, const at::Tensor& state, int64_t offset, const OptTensor& residual) {
  return run_dropout(x, p, 0, offset, &state, residual);
}

// ---- token log probabilities ---------------------------------------------------------------------
struct Logprobs {
  TwgLogprobsDesc d;
  at::Tensor logits, tokens;            // [rows, vocab], [rows, tokens per row]
  std::vector<int64_t> lead;            // logits' leading dimensions
};
static Logprobs describe_logprobs(const char* name, const at::Tensor& logits, const at::Tensor& tokens, int64_t top, double scale) {
  Logprobs r;
  std::memset(&r.d, 0, sizeof(r.d));
  r.d.dtype = dtype_of(name, logits);
  TORCH_CHECK(logits.dim() >= 1, "torch_webgpu: ", name, " expects logits of at least one dimension");
  same_device(name, logits, tokens);
  r.d.token_dtype = index_dtype_of(name, "tokens", tokens);
  const int64_t n = logits.dim();
  r.lead.assign(logits.sizes().begin(), logits.sizes().end() - 1);
  TORCH_CHECK(tokens.dim() == n - 1 || tokens.dim() == n, "torch_webgpu: ", name, ": tokens of ", tokens.sizes(), " do not belong to logits of ", logits.sizes());
  int64_t rows = 1;
  for (int64_t i = 0; i < n - 1; ++i) {
    TORCH_CHECK(tokens.size(i) == logits.size(i), "torch_webgpu: ", name, ": tokens of ", tokens.sizes(), " do not belong to logits of ", logits.sizes());
    rows *= logits.size(i);
  }
  const int64_t m = tokens.dim() == n ? tokens.size(n - 1) : 1, vocab = logits.size(n - 1);
  TORCH_CHECK(vocab >= 1 && vocab <= (int64_t(1) << 30), "torch_webgpu: ", name, " supports a vocabulary of 1 to 2^30 tokens, got ", vocab);
  TORCH_CHECK(rows <= (int64_t(1) << 27), "torch_webgpu: ", name, " supports at most 2^27 rows, got ", rows);
  TORCH_CHECK(m <= TWG_LOGPROBS_MAX_TOKENS, "torch_webgpu: ", name, " supports at most ", TWG_LOGPROBS_MAX_TOKENS, " tokens a row, got ", m);
  TORCH_CHECK(top >= 0 && top <= 32 && top <= vocab, "torch_webgpu: ", name, " supports 0 to 32 alternatives out of the vocabulary, got ", top);
  TORCH_CHECK(scale > 0 && scale <= 1e38, "torch_webgpu: ", name, ": scale must be positive and finite, got ", scale);
  r.logits = logits.reshape({rows, vocab});
  if ((vocab > 1 && r.logits.stride(1) != 1) || (rows > 1 && r.logits.stride(0) < vocab)) r.logits = r.logits.contiguous();
  r.tokens = tokens.reshape({rows, m});
  r.d.tokens_per_row = static_cast<int32_t>(m);
  r.d.top = static_cast<int32_t>(top);
  r.d.rows = rows;
  r.d.vocab = vocab;
  r.d.row_stride = rows > 1 ? r.logits.stride(0) : vocab;
  r.d.token_strides[0] = r.tokens.stride(0);
  r.d.token_strides[1] = r.tokens.stride(1);
  r.d.scale = static_cast<float>(scale);
  return r;
}

using LogprobsOut = std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor>;

LogprobsOut token_logprobs(const at::Tensor& logits, const at::Tensor& tokens, int64_t top, double scale) {
  const auto numbers = logits.options().dtype(at::kFloat);
  if (symbolic(logits) || symbolic(tokens)) {
    const auto lead = logits.sym_sizes().slice(0, logits.dim() - 1);
    std::vector<c10::SymInt> tops(lead.begin(), lead.end());
    tops.emplace_back(top);
    return {at::empty_symint(tokens.sym_sizes(), numbers), at::empty_symint(lead, numbers), at::empty_symint(lead, numbers),
            at::empty_symint(tops, numbers), at::empty_symint(tops, logits.options().dtype(at::kLong))};
  }
  Logprobs r = describe_logprobs("token_logprobs", logits, tokens, top, scale);
  at::Tensor logp = at::empty(tokens.sizes(), numbers), entropy = at::empty(r.lead, numbers), lse = at::empty(r.lead, numbers);
  std::vector<int64_t> tops = r.lead;
  tops.push_back(top);
  at::Tensor top_logp = at::empty(tops, numbers), top_ids = at::empty(tops, logits.options().dtype(at::kLong));
  if (logits.is_meta() || r.d.rows == 0) return {logp, entropy, lse, top_logp, top_ids};
  const c10::DeviceIndex dev = tensor_device(logits);
  core::DeviceScope scope(dev);
  TWG_TORCH_CHECK(twg_token_logprobs(&r.d, r.logits.const_data_ptr(), r.tokens.const_data_ptr(), static_cast<float*>(logp.data_ptr()),
                                     static_cast<float*>(entropy.data_ptr()), static_cast<float*>(lse.data_ptr()),
                                     top ? static_cast<float*>(top_logp.data_ptr()) : nullptr,
                                     top ? static_cast<int64_t*>(top_ids.data_ptr()) : nullptr, core::current_stream(dev)));
  return {logp, entropy, lse, top_logp, top_ids};
}

at::Tensor token_logprobs_backward(const OptTensor& dlogp, const OptTensor& dentropy, const OptTensor& dlse, const at::Tensor& logits,
                                   const at::Tensor& tokens, const at::Tensor& entropy, const at::Tensor& lse, double scale) {
  const char* name = "token_logprobs_backward";
  if (symbolic(logits) || symbolic(tokens)) return at::empty_symint(logits.sym_sizes(), logits.options());
  Logprobs r = describe_logprobs(name, logits, tokens, 0, scale);
  auto dense = [&](const OptTensor& g, c10::IntArrayRef shape) -> at::Tensor {
    if (!given(g)) return at::Tensor();
    same_device(name, logits, *g);
    TORCH_CHECK(g->scalar_type() == at::kFloat && g->sizes() == shape, "torch_webgpu: ", name, ": a float32 tensor of ", shape, " is expected, got ",
                g->sizes(), " ", g->scalar_type());
    return g->contiguous();
  };
  const at::Tensor glogp = dense(dlogp, tokens.sizes()), gent = dense(dentropy, r.lead), glse = dense(dlse, r.lead);
  const at::Tensor ent = dense(entropy, r.lead), norm = dense(lse, r.lead);
  at::Tensor out = at::empty(logits.sizes(), logits.options());
  if (logits.is_meta() || r.d.rows == 0) return out;
  const c10::DeviceIndex dev = tensor_device(logits);
  core::DeviceScope scope(dev);
  auto p = [](const at::Tensor& t) { return t.defined() ? static_cast<const float*>(t.const_data_ptr()) : nullptr; };
  TWG_TORCH_CHECK(twg_token_logprobs_backward(&r.d, r.logits.const_data_ptr(), r.tokens.const_data_ptr(), p(ent), p(norm), p(glogp), p(gent),
                                              p(glse), out.data_ptr(), r.d.vocab, core::current_stream(dev)));
  return out;
}

// ------------------------------------------------------------------------------------------
// gradients
// ------------------------------------------------------------------------------------------
template <class F>
static c10::TypedOperatorHandle<F> op(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}
#define TWG_OP(fn, name)                                               \
  ([]() -> auto& {                                                     \
    static const auto handle = op<decltype(fn)>("webgpu::" name);      \
    return handle;                                                     \
  }())

// Calls the kernel behind an op without recording a gradient of its own.
template <class H, class... A>
static auto below_autograd(const H& handle, A&&... args) {
  at::AutoDispatchBelowADInplaceOrView guard;
  return handle.call(std::forward<A>(args)...);
}
static OptTensor optional(const at::Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }

// The gradient of a rotation is the rotation back: its own op again, so it can be differentiated on.
struct RotaryGrad : public Function<RotaryGrad> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& positions, const at::Tensor& inv_freq,
                            std::vector<int64_t> axis_of, bool adjacent, bool inverse) {
    ctx->save_for_backward({positions, inv_freq});
    ctx->saved_data["axis_of"] = axis_of;
    ctx->saved_data["adjacent"] = adjacent;
    ctx->saved_data["inverse"] = inverse;
    return below_autograd(TWG_OP(rotary, "rotary"), x, positions, inv_freq, axis_of, adjacent, inverse);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto saved = ctx->get_saved_variables();
    at::Tensor dx = TWG_OP(rotary, "rotary").call(g[0], saved[0], saved[1], ctx->saved_data["axis_of"].toIntVector(),
                                                  ctx->saved_data["adjacent"].toBool(), !ctx->saved_data["inverse"].toBool());
    return {dx, {}, {}, {}, {}, {}};
  }
};
struct RotaryQkGrad : public Function<RotaryQkGrad> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& positions,
                               const at::Tensor& inv_freq, std::vector<int64_t> axis_of, bool adjacent, bool inverse) {
    ctx->save_for_backward({positions, inv_freq});
    ctx->saved_data["axis_of"] = axis_of;
    ctx->saved_data["adjacent"] = adjacent;
    ctx->saved_data["inverse"] = inverse;
    auto [qo, ko] = below_autograd(TWG_OP(rotary_qk, "rotary_qk"), q, k, positions, inv_freq, axis_of, adjacent, inverse);
    return {qo, ko};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto saved = ctx->get_saved_variables();
    auto [dq, dk] = TWG_OP(rotary_qk, "rotary_qk").call(g[0], g[1], saved[0], saved[1], ctx->saved_data["axis_of"].toIntVector(),
                                                        ctx->saved_data["adjacent"].toBool(), !ctx->saved_data["inverse"].toBool());
    return {dq, dk, {}, {}, {}, {}, {}};
  }
};
static void no_gradient(const char* name, const at::Tensor& inv_freq) {
  TORCH_CHECK(!(at::GradMode::is_enabled() && inv_freq.requires_grad()), "torch_webgpu: ", name, " has no gradient for inv_freq");
}
at::Tensor rotary_autograd(const at::Tensor& x, const at::Tensor& positions, const at::Tensor& inv_freq, c10::IntArrayRef axis_of, bool adjacent,
                           bool inverse) {
  no_gradient("rotary", inv_freq);
  return RotaryGrad::apply(x, positions, inv_freq, axis_of.vec(), adjacent, inverse);
}
std::tuple<at::Tensor, at::Tensor> rotary_qk_autograd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& positions,
                                                      const at::Tensor& inv_freq, c10::IntArrayRef axis_of, bool adjacent, bool inverse) {
  no_gradient("rotary_qk", inv_freq);
  auto out = RotaryQkGrad::apply(q, k, positions, inv_freq, axis_of.vec(), adjacent, inverse);
  return {out[0], out[1]};
}

struct QkNormGrad : public Function<QkNormGrad> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const OptTensor& qw, const OptTensor& kw,
                               const at::Tensor& positions, const at::Tensor& inv_freq, std::vector<int64_t> axis_of, double eps, bool adjacent) {
    ctx->save_for_backward({q, k, given(qw) ? *qw : at::Tensor(), given(kw) ? *kw : at::Tensor(), positions, inv_freq});
    ctx->saved_data["axis_of"] = axis_of;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["adjacent"] = adjacent;
    auto [qo, ko] = below_autograd(TWG_OP(qk_norm_rotary, "qk_norm_rotary"), q, k, qw, kw, positions, inv_freq, axis_of, eps, adjacent);
    return {qo, ko};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto s = ctx->get_saved_variables();
    auto [dq, dk, dqw, dkw] = TWG_OP(qk_norm_rotary_backward, "qk_norm_rotary_backward")
                                  .call(g[0], g[1], s[0], s[1], optional(s[2]), optional(s[3]), s[4], s[5],
                                        ctx->saved_data["axis_of"].toIntVector(), ctx->saved_data["eps"].toDouble(),
                                        ctx->saved_data["adjacent"].toBool());
    return {dq, dk, s[2].defined() ? dqw : at::Tensor(), s[3].defined() ? dkw : at::Tensor(), {}, {}, {}, {}, {}};
  }
};
std::tuple<at::Tensor, at::Tensor> qk_norm_rotary_autograd(const at::Tensor& q, const at::Tensor& k, const OptTensor& qw, const OptTensor& kw,
                                                           const at::Tensor& positions, const at::Tensor& inv_freq, c10::IntArrayRef axis_of,
                                                           double eps, bool adjacent) {
  no_gradient("qk_norm_rotary", inv_freq);
  auto out = QkNormGrad::apply(q, k, qw, kw, positions, inv_freq, axis_of.vec(), eps, adjacent);
  return {out[0], out[1]};
}

// The two gradient ops have no gradient of their own: asking for one is an error, not a zero.
struct QkNormGradTwice : public Function<QkNormGradTwice> {
  static variable_list forward(AutogradContext*, const at::Tensor& gq, const at::Tensor& gk, const at::Tensor& q, const at::Tensor& k,
                               const OptTensor& qw, const OptTensor& kw, const at::Tensor& positions, const at::Tensor& inv_freq,
                               std::vector<int64_t> axis_of, double eps, bool adjacent) {
    auto [a, b, c, d] = below_autograd(TWG_OP(qk_norm_rotary_backward, "qk_norm_rotary_backward"), gq, gk, q, k, qw, kw, positions, inv_freq,
                                       axis_of, eps, adjacent);
    return {a, b, c, d};
  }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK(false, "torch_webgpu: qk_norm_rotary can be differentiated once only");
  }
};
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> qk_norm_rotary_backward_autograd(
    const at::Tensor& gq, const at::Tensor& gk, const at::Tensor& q, const at::Tensor& k, const OptTensor& qw, const OptTensor& kw,
    const at::Tensor& positions, const at::Tensor& inv_freq, c10::IntArrayRef axis_of, double eps, bool adjacent) {
  auto out = QkNormGradTwice::apply(gq, gk, q, k, qw, kw, positions, inv_freq, axis_of.vec(), eps, adjacent);
  return {out[0], out[1], out[2], out[3]};
}

// Dropout is linear in x: its gradient is the same dropout of the gradient.
struct DropoutGrad : public Function<DropoutGrad> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, double p, int64_t seed, int64_t offset, const OptTensor& residual) {
    ctx->saved_data["p"] = p;
    ctx->saved_data["seed"] = seed;
    ctx->saved_data["offset"] = offset;
    ctx->saved_data["residual"] = given(residual);
    return below_autograd(TWG_OP(dropout, "dropout"), x, p, seed, offset, residual);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    at::Tensor dx;
    if (ctx->needs_input_grad(0))
      dx = TWG_OP(dropout, "dropout").call(g[0], ctx->saved_data["p"].toDouble(), ctx->saved_data["seed"].toInt(),
                                           ctx->saved_data["offset"].toInt(), OptTensor());
    return {dx, {}, {}, {}, ctx->saved_data["residual"].toBool() ? g[0] : at::Tensor()};
  }
};
// The state is saved: autograd refuses the backward pass if it was changed in place since.
struct DropoutStateGrad : public Function<DropoutStateGrad> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, double p, const at::Tensor& state, int64_t offset, const OptTensor& residual) {
    ctx->save_for_backward({state});
    ctx->saved_data["p"] = p;
    ctx->saved_data["offset"] = offset;
    ctx->saved_data["residual"] = given(residual);
    return below_autograd(TWG_OP(dropout_state, "dropout_state"), x, p, state, offset, residual);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    at::Tensor dx;
    const auto saved = ctx->get_saved_variables();
    if (ctx->needs_input_grad(0))
      dx = TWG_OP(dropout_state, "dropout_state").call(g[0], ctx->saved_data["p"].toDouble(), saved[0], ctx->saved_data["offset"].toInt(),
                                                          OptTensor());
    return {dx, {}, {}, {}, ctx->saved_data["residual"].toBool() ? g[0] : at::Tensor()};
  }
};
at::Tensor dropout_autograd(const at::Tensor& x, double p, int64_t seed, int64_t offset, const OptTensor& residual) {
  return DropoutGrad::apply(x, p, seed, offset, residual);
}
at::Tensor dropout_state_autograd(const at::Tensor& x, double p, const at::Tensor& state, int64_t offset, const OptTensor& residual) {
  return DropoutStateGrad::apply(x, p, state, offset, residual);
}

struct LogprobsGrad : public Function<LogprobsGrad> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& logits, const at::Tensor& tokens, int64_t top, double scale) {
    auto [logp, entropy, lse, top_logp, top_ids] = below_autograd(TWG_OP(token_logprobs, "token_logprobs"), logits, tokens, top, scale);
    ctx->save_for_backward({logits, tokens, entropy, lse});
    ctx->saved_data["scale"] = scale;
    ctx->mark_non_differentiable({top_logp, top_ids});
    ctx->set_materialize_grads(false);
    return {logp, entropy, lse, top_logp, top_ids};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    if (!g[0].defined() && !g[1].defined() && !g[2].defined()) return {{}, {}, {}, {}};
    const auto s = ctx->get_saved_variables();
    at::Tensor dx = TWG_OP(token_logprobs_backward, "token_logprobs_backward")
                        .call(optional(g[0]), optional(g[1]), optional(g[2]), s[0], s[1], s[2], s[3], ctx->saved_data["scale"].toDouble());
    return {dx, {}, {}, {}};
  }
};
LogprobsOut token_logprobs_autograd(const at::Tensor& logits, const at::Tensor& tokens, int64_t top, double scale) {
  auto out = LogprobsGrad::apply(logits, tokens, top, scale);
  return {out[0], out[1], out[2], out[3], out[4]};
}
struct LogprobsGradTwice : public Function<LogprobsGradTwice> {
  static at::Tensor forward(AutogradContext*, const OptTensor& dlogp, const OptTensor& dentropy, const OptTensor& dlse, const at::Tensor& logits,
                            const at::Tensor& tokens, const at::Tensor& entropy, const at::Tensor& lse, double scale) {
    return below_autograd(TWG_OP(token_logprobs_backward, "token_logprobs_backward"), dlogp, dentropy, dlse, logits, tokens, entropy, lse, scale);
  }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK(false, "torch_webgpu: token_logprobs can be differentiated once only");
  }
};
at::Tensor token_logprobs_backward_autograd(const OptTensor& dlogp, const OptTensor& dentropy, const OptTensor& dlse, const at::Tensor& logits,
                                            const at::Tensor& tokens, const at::Tensor& entropy, const at::Tensor& lse, double scale) {
  return LogprobsGradTwice::apply(dlogp, dentropy, dlse, logits, tokens, entropy, lse, scale);
}

// ------------------------------------------------------------------------------------------
// aten::dropout (torch.nn.Dropout, torch.nn.functional.dropout)
// ------------------------------------------------------------------------------------------
// One seed and one running offset for the backend; every call draws from an offset of its own.
static std::mutex rng_mu;
static uint64_t rng_seed = 0, rng_offset = 0;

at::Tensor aten_dropout(const at::Tensor& input, double p, bool train) {
  TORCH_CHECK(p >= 0 && p <= 1, "dropout probability has to be between 0 and 1, but got ", p);
  if (p == 0 || !train || input.numel() == 0) return input;
  // A traced graph would keep this call's seed and offset and drop the same elements every time.
  TORCH_CHECK(!input.key_set().has(c10::DispatchKey::Python) && !input.key_set().has(c10::DispatchKey::Functionalize),
              "torch_webgpu: dropout with the backend's own generator cannot be compiled; call torch.ops.webgpu.dropout_state with a state tensor");
  uint64_t seed, offset;
  {
    std::lock_guard<std::mutex> lock(rng_mu);
    seed = rng_seed;
    offset = rng_offset++;
  }
  return TWG_OP(dropout, "dropout").call(input, p, static_cast<int64_t>(seed), static_cast<int64_t>(offset), OptTensor());
}

}  // namespace ops

namespace core {
void set_rng_state(uint64_t seed, uint64_t offset) {
  std::lock_guard<std::mutex> lock(ops::rng_mu);
  ops::rng_seed = seed;
  ops::rng_offset = offset;
}
std::pair<uint64_t, uint64_t> get_rng_state() {
  std::lock_guard<std::mutex> lock(ops::rng_mu);
  return {ops::rng_seed, ops::rng_offset};
}
}  // namespace core

TORCH_LIBRARY_FRAGMENT(webgpu, m) {
  m.def("rotary(Tensor x, Tensor positions, Tensor inv_freq, *, int[] axis_of=[], bool adjacent=False, bool inverse=False) -> Tensor");
  m.def("rotary_qk(Tensor q, Tensor k, Tensor positions, Tensor inv_freq, *, int[] axis_of=[], bool adjacent=False, bool inverse=False) -> (Tensor, Tensor)");
  m.def("qk_norm_rotary(Tensor q, Tensor k, Tensor? q_weight, Tensor? k_weight, Tensor positions, Tensor inv_freq, *, int[] axis_of=[], "
        "float eps=1e-06, bool adjacent=False) -> (Tensor, Tensor)");
  m.def("qk_norm_rotary_backward(Tensor dq_out, Tensor dk_out, Tensor q, Tensor k, Tensor? q_weight, Tensor? k_weight, Tensor positions, "
        "Tensor inv_freq, *, int[] axis_of=[], float eps=1e-06, bool adjacent=False) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("dropout(Tensor x, float p, int seed, int offset=0, *, Tensor? residual=None) -> Tensor");
  m.def("dropout_state(Tensor x, float p, Tensor state, int offset=0, *, Tensor? residual=None) -> Tensor");
  m.def("token_logprobs(Tensor logits, Tensor tokens, *, int top=0, float scale=1.0) -> (Tensor logp, Tensor entropy, Tensor lse, "
        "Tensor top_logp, Tensor top_ids)");
  m.def("token_logprobs_backward(Tensor? dlogp, Tensor? dentropy, Tensor? dlse, Tensor logits, Tensor tokens, Tensor entropy, Tensor lse, *, "
        "float scale=1.0) -> Tensor");
}
#define TWG_TRANSFORMER_OPS(m)                                                     \
  m.impl("rotary", TORCH_FN(ops::rotary));                                         \
  m.impl("rotary_qk", TORCH_FN(ops::rotary_qk));                                   \
  m.impl("qk_norm_rotary", TORCH_FN(ops::qk_norm_rotary));                         \
  m.impl("qk_norm_rotary_backward", TORCH_FN(ops::qk_norm_rotary_backward));       \
  m.impl("dropout", TORCH_FN(ops::dropout));                                       \
  m.impl("dropout_state", TORCH_FN(ops::dropout_state));                           \
  m.impl("token_logprobs", TORCH_FN(ops::token_logprobs));                         \
  m.impl("token_logprobs_backward", TORCH_FN(ops::token_logprobs_backward));
TORCH_LIBRARY_IMPL(webgpu, PrivateUse1, m) { TWG_TRANSFORMER_OPS(m) }
TORCH_LIBRARY_IMPL(webgpu, Meta, m) { TWG_TRANSFORMER_OPS(m) }
#undef TWG_TRANSFORMER_OPS
TORCH_LIBRARY_IMPL(webgpu, AutogradPrivateUse1, m) {
  m.impl("rotary", TORCH_FN(ops::rotary_autograd));
  m.impl("rotary_qk", TORCH_FN(ops::rotary_qk_autograd));
  m.impl("qk_norm_rotary", TORCH_FN(ops::qk_norm_rotary_autograd));
  m.impl("qk_norm_rotary_backward", TORCH_FN(ops::qk_norm_rotary_backward_autograd));
  m.impl("dropout", TORCH_FN(ops::dropout_autograd));
  m.impl("dropout_state", TORCH_FN(ops::dropout_state_autograd));
  m.impl("token_logprobs", TORCH_FN(ops::token_logprobs_autograd));
  m.impl("token_logprobs_backward", TORCH_FN(ops::token_logprobs_backward_autograd));
}
TORCH_LIBRARY_IMPL(aten, PrivateUse1, m) { m.impl("dropout", TORCH_FN(ops::aten_dropout)); }
TORCH_LIBRARY_IMPL(aten, AutogradPrivateUse1, m) { m.impl("dropout", TORCH_FN(ops::aten_dropout)); }

}  // namespace torch_webgpu
