// ffa_torch_gen.cpp — the torch-facing host path of general attention (ffa_gen_* of
// include/ffa.h), beside ffa_torch.cpp and in its manner:
//
//   ffa_b200::general(q, k, v, <mask>)            -> o          (no LSE, no grad)
//   ffa_b200::general_lse(q, k, v, <mask>, with_lo) -> (o, o_lo, lse)
//   ffa_b200::general_backward(q, k, v, o, o_lo, do, lse, <mask>, want_dq, want_dkdv,
//                              want_dbias)        -> (dq, dk, dv, dbias)
//   ffa_b200::general_attention(q, k, v, <mask>)  -> o, differentiable (C++ autograd node)
//
// <mask> is (bias, key_lengths, query_offsets, query_offset, borders, both, causal, scale).
// q is [B, Hq, Sq, D] and k, v are [B, Hkv, Sk, D] bf16 CUDA tensors of any strides that a
// tensor map can describe; others are copied.  Outputs, gradients and workspaces come from
// the torch caching allocator on the inputs' device, once a call: two calls, or two captured
// graphs, share none.  Every launch goes on the current stream.
#include <ATen/cuda/CUDAContext.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/autograd.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include <cmath>

#include "../../include/ffa.h"

namespace {

using at::Tensor;
using OptTensor = c10::optional<Tensor>;

void check(int rc, const char* fn) {
  if (rc != FFA_OK) {
    char buf[256];
    ffa_last_error(buf, sizeof(buf));
    TORCH_CHECK(false, fn, " failed with status ", rc, ": ", buf);
  }
}

// Whether a tensor map can describe `t` as it lies.
bool describable(const Tensor& t) {
  if (t.numel() == 0) return true;
  if (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) return false;
  if (t.size(3) > 1 && t.stride(3) != 1) return false;
  for (int d = 0; d < 3; ++d)
    if (t.size(d) > 1 && (t.stride(d) <= 0 || t.stride(d) % 8 != 0 || t.stride(d) >= (int64_t{1} << 39))) return false;
  return true;
}

// `t`, or a contiguous copy (a contiguous tensor that starts off a 16-byte border too).
Tensor prep(const Tensor& t) { return describable(t) ? t : t.clone(at::MemoryFormat::Contiguous); }

// An output in the layout of `like` where the kernels can write it, else contiguous.
Tensor output_like(const Tensor& like) {
  Tensor r = at::empty_like(like);
  return describable(r) ? r : at::empty(like.sizes(), like.options());
}

ffa_gen_tensor tensor(const Tensor& t) {
  auto stride = [&](int d) -> long long { return t.size(d) > 1 && t.numel() > 0 ? t.stride(d) : 8; };
  return {t.data_ptr(), stride(0), stride(1), stride(2)};
}

struct Mask {
  OptTensor bias, key_lengths, query_offsets;
  int64_t query_offset;
  std::vector<int64_t> borders;
  bool both, causal;
  c10::optional<double> scale;
};

// The C ABI's problem.  It points into the mask's tensors and into `borders`.
struct Args {
  ffa_gen_problem p{};
  std::vector<int> borders;
  Tensor bias;
};

void fill(Args& a, const Tensor& q, const Tensor& k, const Tensor& v, const Mask& m) {
  TORCH_CHECK(q.is_cuda(), "q must be a CUDA tensor");
  for (const Tensor* t : {&q, &k, &v}) {
    TORCH_CHECK(t->device() == q.device(), "all tensors must be on one device");
    TORCH_CHECK(t->scalar_type() == at::kBFloat16 && t->dim() == 4, "q, k and v must be bf16 [B, H, S, D]");
  }
  TORCH_CHECK(k.sizes() == v.sizes() && q.size(0) == k.size(0) && q.size(3) == k.size(3),
              "q, k and v must share batch and head dim, k and v their shape");
  auto ints = [&](const OptTensor& t, const char* name) -> const int* {
    if (!t.has_value()) return nullptr;
    TORCH_CHECK(t->device() == q.device() && t->scalar_type() == at::kInt && t->dim() == 1 && t->size(0) == q.size(0) &&
                    t->is_contiguous(),
                name, " must be a contiguous int32 [B] tensor on the device of q");
    return t->data_ptr<int>();
  };
  for (int64_t n : {q.size(0), q.size(1), q.size(2), k.size(1), k.size(2)})
    TORCH_CHECK(n <= INT_MAX, "sizes must fit in 32 bits");
  TORCH_CHECK(std::abs(m.query_offset) <= INT_MAX, "query_offset must fit in 32 bits");
  ffa_gen_problem& p = a.p;
  p.batch = static_cast<int>(q.size(0));
  p.q_heads = static_cast<int>(q.size(1));
  p.kv_heads = static_cast<int>(k.size(1));
  p.q_len = static_cast<int>(q.size(2));
  p.k_len = static_cast<int>(k.size(2));
  p.head_dim = static_cast<int>(q.size(3));
  p.causal = m.causal ? 1 : 0;
  p.scale = m.scale.has_value() ? *m.scale : 1.0 / std::sqrt(static_cast<double>(q.size(3)));
  p.key_lengths = ints(m.key_lengths, "key_lengths");
  p.query_offsets = ints(m.query_offsets, "query_offsets");
  p.query_offset = static_cast<int>(m.query_offset);
  if (m.bias.has_value()) {
    const Tensor& b = *m.bias;
    const int64_t side = static_cast<int64_t>(m.borders.size());
    TORCH_CHECK(b.device() == q.device() && b.scalar_type() == at::kBFloat16 && b.dim() == 2 &&
                    b.size(0) == (m.both ? 2 * side : side) && b.size(1) == q.size(1),
                "bias must be bf16 [buckets, q heads] on the device of q");
    a.bias = b.contiguous();
    a.borders.assign(m.borders.begin(), m.borders.end());
    p.bias = a.bias.data_ptr();
    p.buckets = static_cast<int>(b.size(0));
    p.both = m.both ? 1 : 0;
    p.borders = a.borders.data();
  }
}

// Workspace of one call; freed to the caching allocator on return, which hands it out again
// only behind the kernels queued on this stream.
Tensor workspace(long long bytes, const char* fn, const Tensor& like) {
  if (bytes < 0) check(FFA_ERR_INVALID, fn);
  return bytes > 0 ? at::empty({bytes}, like.options().dtype(at::kByte)) : Tensor();
}
void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

void* stream_of(const Tensor& t) { return at::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

// -> o, its remainder (for the bias's gradient, see ffa_gen_fwd), lse
std::tuple<Tensor, Tensor, Tensor> forward_impl(const Tensor& q0, const Tensor& k0, const Tensor& v0, const Mask& m,
                                                bool with_lse, bool with_lo) {
  Args a;
  fill(a, q0, k0, v0, m);
  const c10::cuda::CUDAGuard guard(q0.device());
  const Tensor q = prep(q0), k = prep(k0), v = prep(v0);
  Tensor o = output_like(q), o_lo, lse;
  if (with_lo) o_lo = at::empty_like(o);
  if (with_lse) lse = at::empty({q.size(0), q.size(1), q.size(2)}, q.options().dtype(at::kFloat));
  const long long bytes = ffa_gen_fwd_workspace(&a.p, with_lo ? 1 : 0);
  const Tensor ws = workspace(bytes, "ffa_gen_fwd_workspace", q);
  const ffa_gen_tensor tq = tensor(q), tk = tensor(k), tv = tensor(v), to = tensor(o);
  const ffa_gen_tensor tlo = with_lo ? tensor(o_lo) : ffa_gen_tensor{};
  check(ffa_gen_fwd(&a.p, &tq, &tk, &tv, &to, with_lo ? &tlo : nullptr, with_lse ? lse.data_ptr<float>() : nullptr, data(ws), bytes,
                    stream_of(q)),
        "ffa_gen_fwd");
  return {o, o_lo, lse};
}

// want: dq, dk and dv, dbias
std::tuple<Tensor, Tensor, Tensor, Tensor> backward_impl(const Tensor& q0, const Tensor& k0, const Tensor& v0,
                                                         const Tensor& o0, const Tensor& lo0, const Tensor& do0,
                                                         const Tensor& lse0, const Mask& m, bool want_dq, bool want_dkdv,
                                                         bool want_dbias) {
  Args a;
  fill(a, q0, k0, v0, m);
  TORCH_CHECK(o0.sizes() == q0.sizes() && do0.sizes() == q0.sizes() && o0.scalar_type() == at::kBFloat16 &&
                  do0.scalar_type() == at::kBFloat16 && o0.device() == q0.device() && do0.device() == q0.device(),
              "o and do must be bf16 tensors like q");
  TORCH_CHECK(!lo0.defined() || (lo0.sizes() == q0.sizes() && lo0.scalar_type() == at::kBFloat16 &&
                                 lo0.device() == q0.device()),
              "o_lo must be a bf16 tensor like q");
  TORCH_CHECK(lse0.scalar_type() == at::kFloat && lse0.numel() == q0.size(0) * q0.size(1) * q0.size(2) &&
                  lse0.device() == q0.device(),
              "lse must be the fp32 [B, H, S] of the forward");
  const c10::cuda::CUDAGuard guard(q0.device());
  const Tensor q = prep(q0), k = prep(k0), v = prep(v0), o = prep(o0), dout = prep(do0), lse = lse0.contiguous();
  const Tensor o_lo = lo0.defined() ? prep(lo0) : Tensor();
  Tensor dq, dk, dv, dbias;
  if (want_dq || want_dbias) dq = output_like(q);  // the kernel of dbias computes dq too
  if (want_dkdv) {
    dk = output_like(k);
    dv = output_like(v);
  }
  if (want_dbias) dbias = at::empty_like(a.bias, at::MemoryFormat::Contiguous);
  const long long bytes = ffa_gen_bwd_workspace(&a.p);
  const Tensor ws = workspace(bytes, "ffa_gen_bwd_workspace", q);
  auto maybe = [](const Tensor& t) { return t.defined() ? tensor(t) : ffa_gen_tensor{}; };
  const ffa_gen_tensor tq = tensor(q), tk = tensor(k), tv = tensor(v), to = tensor(o), tdo = tensor(dout);
  const ffa_gen_tensor tlo = maybe(o_lo), tdq = maybe(dq), tdk = maybe(dk), tdv = maybe(dv);
  check(ffa_gen_bwd(&a.p, &tq, &tk, &tv, &to, o_lo.defined() ? &tlo : nullptr, &tdo, lse.data_ptr<float>(), dq.defined() ? &tdq : nullptr,
                    dk.defined() ? &tdk : nullptr, dk.defined() ? &tdv : nullptr, data(dbias), data(ws), bytes,
                    stream_of(q)),
        "ffa_gen_bwd");
  return {dq, dk, dv, dbias};
}

Tensor general_op(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& bias,
                  const OptTensor& key_lengths, const OptTensor& query_offsets, int64_t query_offset,
                  at::IntArrayRef borders, bool both, bool causal, c10::optional<double> scale) {
  const Mask m{bias, key_lengths, query_offsets, query_offset, borders.vec(), both, causal, scale};
  return std::get<0>(forward_impl(q, k, v, m, false, false));
}

Tensor some(const Tensor& t, const Tensor& like) { return t.defined() ? t : at::empty({0}, like.options()); }

std::tuple<Tensor, Tensor, Tensor> general_lse_op(const Tensor& q, const Tensor& k, const Tensor& v,
                                                  const OptTensor& bias, const OptTensor& key_lengths,
                                                  const OptTensor& query_offsets, int64_t query_offset,
                                                  at::IntArrayRef borders, bool both, bool causal,
                                                  c10::optional<double> scale, bool with_lo) {
  const Mask m{bias, key_lengths, query_offsets, query_offset, borders.vec(), both, causal, scale};
  auto [o, lo, lse] = forward_impl(q, k, v, m, true, with_lo);
  return {o, some(lo, q), lse};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> general_backward_op(
    const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& o, const OptTensor& o_lo, const Tensor& dout,
    const Tensor& lse, const OptTensor& bias, const OptTensor& key_lengths, const OptTensor& query_offsets, int64_t query_offset,
    at::IntArrayRef borders, bool both, bool causal, c10::optional<double> scale, bool want_dq, bool want_dkdv,
    bool want_dbias) {
  const Mask m{bias, key_lengths, query_offsets, query_offset, borders.vec(), both, causal, scale};
  auto [dq, dk, dv, db] =
      backward_impl(q, k, v, o, o_lo.value_or(Tensor()), dout, lse, m, want_dq, want_dkdv, want_dbias);
  return {some(dq, q), some(dk, q), some(dv, q), some(db, q)};
}

// The autograd node of ffa_b200::general_attention.  It saves q, k, v, o (and its remainder,
// where the bias wants a gradient), the LSE and the
// mask's tensors, and computes the gradients that are wanted.
class GeneralAttention : public torch::autograd::Function<GeneralAttention> {
 public:
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                        const OptTensor& bias, const OptTensor& key_lengths, const OptTensor& query_offsets,
                        int64_t query_offset, std::vector<int64_t> borders, bool both, bool causal,
                        c10::optional<double> scale) {
    const Mask m{bias, key_lengths, query_offsets, query_offset, borders, both, causal, scale};
    auto [o, lo, lse] = forward_impl(q, k, v, m, true, bias.has_value() && bias->requires_grad());
    ctx->save_for_backward({q, k, v, o, lo, lse, bias.value_or(Tensor()), key_lengths.value_or(Tensor()),
                            query_offsets.value_or(Tensor())});
    ctx->saved_data["query_offset"] = query_offset;
    ctx->saved_data["borders"] = borders;
    ctx->saved_data["both"] = both;
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["has_scale"] = scale.has_value();
    ctx->saved_data["scale"] = scale.value_or(0.0);
    return o;
  }

  static torch::autograd::tensor_list backward(torch::autograd::AutogradContext* ctx,
                                               torch::autograd::tensor_list grads) {
    TORCH_CHECK(!c10::AutogradState::get_tls_state().get_fw_grad_mode() || !grads[0]._fw_grad(0).defined(),
                "the backward of general attention does not support forward-mode derivatives of the output's gradient");
    const auto s = ctx->get_saved_variables();
    auto opt = [](const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
    auto& d = ctx->saved_data;
    Mask m{opt(s[6]),
           opt(s[7]),
           opt(s[8]),
           d["query_offset"].toInt(),
           d["borders"].toIntVector(),
           d["both"].toBool(),
           d["causal"].toBool(),
           d["has_scale"].toBool() ? c10::optional<double>(d["scale"].toDouble()) : c10::nullopt};
    const bool want_dq = ctx->needs_input_grad(0), want_dkdv = ctx->needs_input_grad(1) || ctx->needs_input_grad(2);
    const bool want_dbias = m.bias.has_value() && ctx->needs_input_grad(3);
    torch::autograd::tensor_list r(11);
    {
      const at::AutoGradMode off(false);
      auto [dq, dk, dv, db] = backward_impl(s[0], s[1], s[2], s[3], s[4], grads[0], s[5], m, want_dq, want_dkdv, want_dbias);
      if (want_dq) r[0] = dq;
      r[1] = dk;
      r[2] = dv;
      r[3] = db;
    }
    if (at::GradMode::is_enabled()) {  // create_graph: an error where someone differentiates these
      for (int i = 0; i < 4; ++i)
        if (r[i].defined()) r[i].set_requires_grad(true);
      torch::autograd::tensor_list in(r.begin(), r.begin() + 4);
      auto error = std::make_shared<torch::autograd::DelayedError>(
          "the backward of general attention cannot be differentiated", 4);
      auto out = (*error)(std::move(in));
      for (int i = 0; i < 4; ++i) r[i] = out[i];
    }
    return r;
  }
};

Tensor general_attention_op(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& bias,
                            const OptTensor& key_lengths, const OptTensor& query_offsets, int64_t query_offset,
                            at::IntArrayRef borders, bool both, bool causal, c10::optional<double> scale) {
  return GeneralAttention::apply(q, k, v, bias, key_lengths, query_offsets, query_offset, borders.vec(), both, causal,
                                 scale);
}

}  // namespace

#define FFA_MASK_ARGS                                                                                          \
  "Tensor? bias, Tensor? key_lengths, Tensor? query_offsets, int query_offset, int[] borders, bool both, "      \
  "bool causal, float? scale"

TORCH_LIBRARY_FRAGMENT(ffa_b200, m) {
  m.def("general(Tensor q, Tensor k, Tensor v, " FFA_MASK_ARGS ") -> Tensor");
  m.def("general_lse(Tensor q, Tensor k, Tensor v, " FFA_MASK_ARGS ", bool with_lo) -> (Tensor, Tensor, Tensor)");
  m.def("general_backward(Tensor q, Tensor k, Tensor v, Tensor o, Tensor? o_lo, Tensor dout, Tensor lse, " FFA_MASK_ARGS
        ", bool want_dq, bool want_dkdv, bool want_dbias) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("general_attention(Tensor q, Tensor k, Tensor v, " FFA_MASK_ARGS ") -> Tensor");
}

TORCH_LIBRARY_IMPL(ffa_b200, CUDA, m) {
  m.impl("general", general_op);
  m.impl("general_lse", general_lse_op);
  m.impl("general_backward", general_backward_op);
  m.impl("general_attention", general_op);  // reached only where autograd is off (inference mode)
}

// Without a kernel of their own the other operators would drop tangents (forward-mode
// derivatives) without a word; this one refuses them, and a backward through their outputs.
TORCH_LIBRARY_IMPL(ffa_b200, Autograd, m) {
  m.impl("general_attention", general_attention_op);
  for (const char* name : {"general", "general_lse", "general_backward"})
    m.impl(name, torch::autograd::autogradNotImplementedFallback());
}
