// The autograd nodes of the embedding, dropout and policy loss over the C ABI, in C++.
//
// The kernels of a small call take a few microseconds; what it costs is the host: as
// Python autograd Functions over ctypes a forward and backward took 95 to 135 us, as nodes
// here 55 to 85 (the engine's own hand-over to its device thread and back is 40). Argument
// checks raise ValueError; a status other than FH_OK raises FlashHogError, from the forward
// and from the engine's threads alike.
//
// The library is the one that _capi.py loads: bind() receives its functions' addresses.

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <cmath>
#include <limits>
#include <vector>

#include "flash_hog_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;
using OptTensor = c10::optional<Tensor>;

struct Api {
  decltype(&fh_embed_scratch_bytes) embed_scratch_bytes = nullptr;
  decltype(&fh_embed_fwd) embed_fwd = nullptr;
  decltype(&fh_embed_bwd) embed_bwd = nullptr;
  decltype(&fh_embed_bwd_bwd) embed_bwd_bwd = nullptr;
  decltype(&fh_dropout) dropout = nullptr;
  decltype(&fh_policy_stats_floats) policy_stats_floats = nullptr;
  decltype(&fh_policy_scratch_floats) policy_scratch_floats = nullptr;
  decltype(&fh_policy_fwd) policy_fwd = nullptr;
  decltype(&fh_policy_bwd) policy_bwd = nullptr;
  decltype(&fh_policy_bwd_bwd) policy_bwd_bwd = nullptr;
} api;

// Raises what _capi._check(entry, rc) raises, in this thread (the detail message is the thread's).
void check(const char* entry, int rc) {
  if (rc == FH_OK) return;
  py::gil_scoped_acquire gil;
  py::module_::import("flash_hog_b200._capi").attr("_check")(entry, rc);
}

int dtype_code(const Tensor& t) { return t.scalar_type() == at::kBFloat16 ? 1 : 0; }

bool fp32_or_bf16(const Tensor& t) { return t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16; }

// Every tensor on the first's CUDA device, with storage (not the wrapper of a torch.func transform).
void same_device(const Tensor& t, std::initializer_list<const Tensor*> others) {
  TORCH_CHECK_VALUE(t.is_cuda(), "flash_hog_b200 runs on CUDA tensors only");
  TORCH_CHECK_NOT_IMPLEMENTED(t.has_storage(), "the fused ops do not run under torch.func transforms");
  for (const Tensor* x : others) {
    if (!x->defined()) continue;
    TORCH_CHECK_VALUE(x->device() == t.device(), "tensors must be on one CUDA device, got ", t.device(), " and ",
                      x->device());
    TORCH_CHECK_NOT_IMPLEMENTED(x->has_storage(), "the fused ops do not run under torch.func transforms");
  }
}

void* stream_of(const Tensor& t) { return at::cuda::getCurrentCUDAStream(t.get_device()).stream(); }
float* floats(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }
const long long* longs(const Tensor& t) { return reinterpret_cast<const long long*>(t.data_ptr<int64_t>()); }

// Whether a backward's result will itself be differentiated by something it depends on.
bool tracked(const Tensor& t) { return at::GradMode::is_enabled() && t.requires_grad(); }

// ------------------------------------------------------------------------------------
// Embedding
// ------------------------------------------------------------------------------------

// scale w[t]; `adjoint`: the derivative of the gradient (zero rows for padding and tokens outside).
Tensor embed_lookup(const Tensor& w, const Tensor& tokens, double scale, int64_t padding, bool adjoint) {
  same_device(w, {&tokens});
  c10::cuda::CUDAGuard guard(w.device());
  std::vector<int64_t> shape(tokens.sizes().begin(), tokens.sizes().end());
  shape.push_back(w.size(1));
  Tensor y = at::empty(shape, w.options());
  const int n = static_cast<int>(tokens.numel()), vocab = static_cast<int>(w.size(0)), dim = static_cast<int>(w.size(1));
  if (adjoint)
    check("fh_embed_bwd_bwd", api.embed_bwd_bwd(stream_of(w), dtype_code(w), n, vocab, dim, w.data_ptr(), longs(tokens),
                                                static_cast<float>(scale), padding, y.data_ptr()));
  else
    check("fh_embed_fwd", api.embed_fwd(stream_of(w), dtype_code(w), n, vocab, dim, w.data_ptr(), longs(tokens),
                                        static_cast<float>(scale), y.data_ptr()));
  return y;
}

// dw[v] = scale sum_{t_i = v} dy_i, every row written.
Tensor embed_gradient(const Tensor& dy, const Tensor& tokens, int64_t vocab, double scale, int64_t padding) {
  same_device(dy, {&tokens});
  c10::cuda::CUDAGuard guard(dy.device());
  const int n = static_cast<int>(tokens.numel()), dim = static_cast<int>(dy.size(-1));
  Tensor dw = at::empty({vocab, dim}, dy.options());
  Tensor scratch = at::empty({static_cast<int64_t>(api.embed_scratch_bytes(n, dim))}, dy.options().dtype(at::kByte));
  check("fh_embed_bwd", api.embed_bwd(stream_of(dy), dtype_code(dy), n, static_cast<int>(vocab), dim, dy.data_ptr(),
                                      longs(tokens), static_cast<float>(scale), padding, dw.data_ptr(),
                                      scratch.data_ptr()));
  return dw;
}

// Lookup and gradient are linear and each other's derivatives: one node each, any order.
struct EmbedGradient;
struct EmbedLookup : Function<EmbedLookup> {
  static Tensor forward(AutogradContext* ctx, const Tensor& w, const Tensor& tokens, double scale, int64_t padding,
                        bool adjoint) {
    ctx->save_for_backward({tokens});
    ctx->saved_data["vocab"] = w.size(0);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    return embed_lookup(w, tokens, scale, padding, adjoint);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads);
};

struct EmbedGradient : Function<EmbedGradient> {
  static Tensor forward(AutogradContext* ctx, const Tensor& dy, const Tensor& tokens, int64_t vocab, double scale,
                        int64_t padding) {
    ctx->save_for_backward({tokens});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    return embed_gradient(dy, tokens, vocab, scale, padding);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor tokens = ctx->get_saved_variables()[0], ddw = grads[0].contiguous();
    const double scale = ctx->saved_data["scale"].toDouble();
    const int64_t padding = ctx->saved_data["padding"].toInt();
    return {tracked(ddw) ? EmbedLookup::apply(ddw, tokens, scale, padding, true)
                         : embed_lookup(ddw, tokens, scale, padding, true),
            {}, {}, {}, {}};
  }
};

variable_list EmbedLookup::backward(AutogradContext* ctx, variable_list grads) {
  const Tensor tokens = ctx->get_saved_variables()[0], dy = grads[0].contiguous();
  const int64_t vocab = ctx->saved_data["vocab"].toInt(), padding = ctx->saved_data["padding"].toInt();
  const double scale = ctx->saved_data["scale"].toDouble();
  return {tracked(dy) ? EmbedGradient::apply(dy, tokens, vocab, scale, padding)
                      : embed_gradient(dy, tokens, vocab, scale, padding),
          {}, {}, {}, {}};
}

Tensor embedding(const Tensor& tokens, const Tensor& weight, double scale, c10::optional<int64_t> padding_idx) {
  TORCH_CHECK_VALUE(tokens.scalar_type() == at::kLong || tokens.scalar_type() == at::kInt,
                    "embedding tokens are int64 or int32, got ", tokens.scalar_type());
  TORCH_CHECK_VALUE(weight.dim() == 2 && fp32_or_bf16(weight) && weight.numel() > 0,
                    "the embedding weight is a non-empty (vocab, dim) fp32 or bf16 tensor");
  const int64_t vocab = weight.size(0), padding = padding_idx.value_or(-1);
  TORCH_CHECK_VALUE(!padding_idx || (padding >= 0 && padding < vocab), "padding_idx must be in [0, ", vocab, "), got ",
                    padding);
  TORCH_CHECK_VALUE(tokens.numel() < (1ll << 31) && vocab < (1ll << 31) - 1 && weight.size(1) <= (1 << 20),
                    "embedding: fewer than 2^31 tokens and 2^31 - 1 table rows of at most 2^20 elements");
  same_device(weight, {&tokens});
  return EmbedLookup::apply(weight.contiguous(), tokens.to(at::kLong).contiguous(), scale, padding, false);
}

// ------------------------------------------------------------------------------------
// Dropout
// ------------------------------------------------------------------------------------

Tensor dropout_run(const Tensor& x, const Tensor& residual, const Tensor& seed, int64_t subsequence, int64_t limit,
                   at::ScalarType dtype) {
  same_device(x, {&residual, &seed});
  c10::cuda::CUDAGuard guard(x.device());
  Tensor y = at::empty(x.sizes(), x.options().dtype(dtype).memory_format(at::MemoryFormat::Contiguous));
  check("fh_dropout",
        api.dropout(stream_of(x), x.numel(), dtype_code(x), x.data_ptr(),
                    residual.defined() ? dtype_code(residual) : 0, residual.defined() ? residual.data_ptr() : nullptr,
                    dtype_code(y), y.data_ptr(), longs(seed), static_cast<unsigned>(subsequence),
                    static_cast<int>(limit)));
  return y;
}

// Linear in x: its backward is itself on dy, the mask drawn again from the saved seed.
struct Dropout : Function<Dropout> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& residual, const Tensor& seed,
                        int64_t subsequence, int64_t limit, int64_t dtype) {
    ctx->save_for_backward({seed});
    ctx->saved_data["subsequence"] = subsequence;
    ctx->saved_data["limit"] = limit;
    ctx->saved_data["x"] = static_cast<int64_t>(x.scalar_type());
    ctx->saved_data["residual"] = residual ? static_cast<int64_t>(residual->scalar_type()) : int64_t{-1};
    return dropout_run(x, residual.value_or(Tensor()), seed, subsequence, limit, static_cast<at::ScalarType>(dtype));
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor seed = ctx->get_saved_variables()[0];
    const int64_t subsequence = ctx->saved_data["subsequence"].toInt(), limit = ctx->saved_data["limit"].toInt();
    const int64_t x = ctx->saved_data["x"].toInt(), residual = ctx->saved_data["residual"].toInt();
    Tensor dx, dres;
    if (ctx->needs_input_grad(0)) {
      const Tensor dy = grads[0].contiguous();
      dx = tracked(dy) ? Dropout::apply(dy, c10::nullopt, seed, subsequence, limit, x)
                       : dropout_run(dy, Tensor(), seed, subsequence, limit, static_cast<at::ScalarType>(x));
    }
    if (residual >= 0 && ctx->needs_input_grad(1)) dres = grads[0].to(static_cast<at::ScalarType>(residual));
    return {dx, dres, {}, {}, {}, {}};
  }
};

Tensor dropout(const Tensor& x, double p, const Tensor& seed, int64_t subsequence, const OptTensor& residual) {
  TORCH_CHECK_VALUE(p >= 0.0 && p <= 1.0, "dropout p must be in [0, 1], got ", p);
  TORCH_CHECK_VALUE(subsequence >= 0 && subsequence < (1ll << 32), "subsequence must be in [0, 2^32), got ",
                    subsequence);
  TORCH_CHECK_VALUE(fp32_or_bf16(x) && (!residual || fp32_or_bf16(*residual)), "dropout takes fp32 or bf16 tensors");
  TORCH_CHECK_VALUE(!residual || residual->sizes() == x.sizes(), "the residual must have x's shape");
  same_device(x, {&seed});
  if (residual) same_device(x, {&*residual});
  TORCH_CHECK_VALUE(seed.scalar_type() == at::kLong && seed.numel() == 1,
                    "the dropout seed is an int64 tensor of one element");
  const at::ScalarType dtype = residual ? at::promote_types(x.scalar_type(), residual->scalar_type()) : x.scalar_type();
  return Dropout::apply(x.contiguous(), residual ? OptTensor(residual->contiguous()) : OptTensor(), seed, subsequence,
                        static_cast<int64_t>(std::nearbyint(p * 65536.0)), static_cast<int64_t>(dtype));
}

// ------------------------------------------------------------------------------------
// Policy loss
// ------------------------------------------------------------------------------------

long long row_stride(const Tensor& z) { return z.size(0) > 1 ? z.stride(0) : z.size(1); }

Tensor policy_gradient(const Tensor& z, const Tensor& actions, const Tensor& stats, const Tensor& g) {
  same_device(z, {&g});
  c10::cuda::CUDAGuard guard(z.device());
  Tensor dz = at::empty(z.sizes(), z.options().memory_format(at::MemoryFormat::Contiguous));
  check("fh_policy_bwd",
        api.policy_bwd(stream_of(z), dtype_code(z), static_cast<int>(z.size(0)), static_cast<int>(z.size(1)),
                       row_stride(z), z.data_ptr(), longs(actions), floats(stats), floats(g), dz.data_ptr()));
  return dz;
}

// dz = g dloss/dz; its backward is the double backward.
struct PolicyGradient : Function<PolicyGradient> {
  static Tensor forward(AutogradContext* ctx, const Tensor& z, const Tensor& actions, const Tensor& stats,
                        const Tensor& g) {
    const Tensor g32 = g.to(at::kFloat).contiguous();
    ctx->save_for_backward({z, actions, stats, g32});
    ctx->saved_data["g"] = static_cast<int64_t>(g.scalar_type());
    return policy_gradient(z, actions, stats, g32);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &z = saved[0], &actions = saved[1], &stats = saved[2], &g = saved[3];
    TORCH_CHECK_NOT_IMPLEMENTED(!at::GradMode::is_enabled(),
                                "third-order derivatives of the fused policy loss are not supported");
    same_device(z, {&grads[0]});
    c10::cuda::CUDAGuard guard(z.device());
    const Tensor u = grads[0].to(z.scalar_type()).contiguous();
    const int rows = static_cast<int>(z.size(0)), vocab = static_cast<int>(z.size(1));
    Tensor gz = at::empty(z.sizes(), z.options().memory_format(at::MemoryFormat::Contiguous));
    Tensor gg = at::empty({rows}, z.options().dtype(at::kFloat)), scratch;
    if (const long long n = api.policy_scratch_floats(rows, vocab); n > 0) scratch = at::empty({n}, gg.options());
    check("fh_policy_bwd_bwd",
          api.policy_bwd_bwd(stream_of(z), dtype_code(z), rows, vocab, row_stride(z), z.data_ptr(), longs(actions),
                             floats(stats), floats(g), u.data_ptr(), gz.data_ptr(), floats(gg), floats(scratch)));
    Tensor dg;
    if (ctx->needs_input_grad(3))
      dg = gg.sum().to(static_cast<at::ScalarType>(ctx->saved_data["g"].toInt())).reshape(g.sizes());
    return {gz, {}, {}, dg};
  }
};

struct PolicyLoss : Function<PolicyLoss> {
  static variable_list forward(AutogradContext* ctx, const Tensor& z, const Tensor& actions, const Tensor& old,
                               const Tensor& adv, const OptTensor& ref, const OptTensor& weights, double clip_low,
                               double clip_high, double kl_coef, double normalizer) {
    c10::cuda::CUDAGuard guard(z.device());
    const int rows = static_cast<int>(z.size(0)), vocab = static_cast<int>(z.size(1));
    const auto f32 = z.options().dtype(at::kFloat);
    Tensor lp = at::empty({rows}, f32), loss = at::empty({}, f32);
    Tensor stats = at::empty({static_cast<int64_t>(api.policy_stats_floats(rows, vocab))}, f32);
    check("fh_policy_fwd",
          api.policy_fwd(stream_of(z), dtype_code(z), rows, vocab, row_stride(z), z.data_ptr(), longs(actions),
                         floats(old), floats(adv), floats(ref.value_or(Tensor())), floats(weights.value_or(Tensor())),
                         static_cast<float>(clip_low), static_cast<float>(clip_high), static_cast<float>(kl_coef),
                         static_cast<float>(normalizer), floats(lp), floats(loss), floats(stats)));
    ctx->save_for_backward({z, actions, stats});
    ctx->mark_non_differentiable({lp});
    return {loss, lp};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    // Under create_graph dz depends on z, whether or not the upstream scalar is tracked.
    const Tensor dz = at::GradMode::is_enabled()
                          ? PolicyGradient::apply(saved[0], saved[1], saved[2], grads[0])
                          : policy_gradient(saved[0], saved[1], saved[2], grads[0].to(at::kFloat).contiguous());
    return {dz, {}, {}, {}, {}, {}, {}, {}, {}, {}};
  }
};

std::tuple<Tensor, Tensor> policy_loss(const Tensor& logits, const Tensor& actions, const Tensor& old_logprobs,
                                       const Tensor& advantages, const OptTensor& ref_logprobs,
                                       const OptTensor& weights, double clip_low, double clip_high, double kl_coef,
                                       c10::optional<double> normalizer) {
  TORCH_CHECK_VALUE(logits.dim() == 2 && fp32_or_bf16(logits) && logits.size(1) > 0,
                    "policy_loss takes (rows, vocab) fp32 or bf16 logits");
  TORCH_CHECK_VALUE(clip_low >= 0.0 && clip_high >= 0.0, "clip_low and clip_high must be >= 0");
  TORCH_CHECK_VALUE(kl_coef >= 0.0 && kl_coef < std::numeric_limits<double>::infinity(),
                    "kl_coef must be finite and >= 0");
  TORCH_CHECK_VALUE(kl_coef == 0.0 || ref_logprobs, "kl_coef > 0 needs ref_logprobs");
  TORCH_CHECK_VALUE(!normalizer || (*normalizer >= std::numeric_limits<float>::min() &&
                                    *normalizer <= std::numeric_limits<float>::max()),
                    "normalizer must be positive and finite (a normal fp32 number)");
  const int64_t rows = logits.size(0);
  TORCH_CHECK_VALUE(rows < (1ll << 31) && logits.size(1) < (1ll << 31), "policy_loss: fewer than 2^31 rows and columns");
  TORCH_CHECK_VALUE(!actions.is_floating_point() && actions.dim() == 1 && actions.size(0) == rows,
                    "policy actions are an integer vector of one entry per row");
  same_device(logits, {&actions, &old_logprobs, &advantages});
  // A constant per row, in fp32.
  auto vec = [&](const Tensor& t) {
    TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == rows, "the policy's per-row inputs are vectors of one entry per row");
    same_device(logits, {&t});
    return t.detach().to(at::kFloat).contiguous();
  };
  const bool strided = logits.stride(1) == 1 && (rows <= 1 || logits.stride(0) >= logits.size(1));
  const bool kl = static_cast<float>(kl_coef) > 0.f;
  auto out = PolicyLoss::apply(strided ? logits : logits.contiguous(), actions.to(at::kLong).contiguous(),
                               vec(old_logprobs), vec(advantages), kl ? OptTensor(vec(*ref_logprobs)) : OptTensor(),
                               weights ? OptTensor(vec(*weights)) : OptTensor(), clip_low, clip_high, kl_coef,
                               normalizer.value_or(0.0));
  return {out[0], out[1]};
}

void bind(const py::dict& addresses) {
  auto set = [&](auto& f, const char* name) {
    f = reinterpret_cast<std::remove_reference_t<decltype(f)>>(addresses[name].cast<uintptr_t>());
  };
  set(api.embed_scratch_bytes, "fh_embed_scratch_bytes");
  set(api.embed_fwd, "fh_embed_fwd");
  set(api.embed_bwd, "fh_embed_bwd");
  set(api.embed_bwd_bwd, "fh_embed_bwd_bwd");
  set(api.dropout, "fh_dropout");
  set(api.policy_stats_floats, "fh_policy_stats_floats");
  set(api.policy_scratch_floats, "fh_policy_scratch_floats");
  set(api.policy_fwd, "fh_policy_fwd");
  set(api.policy_bwd, "fh_policy_bwd");
  set(api.policy_bwd_bwd, "fh_policy_bwd_bwd");
}

}  // namespace

PYBIND11_MODULE(_torch_ops, m) {
  m.def("bind", &bind);
  m.def("embedding", &embedding);
  m.def("dropout", &dropout);
  m.def("policy_loss", &policy_loss);
}
