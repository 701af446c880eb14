// The autograd nodes of dense attention, the embedding, dropout and the policy loss over the
// C ABI, in C++.
//
// The kernels of a small call take a few microseconds; what it costs is the host: as
// Python autograd Functions over ctypes a forward and backward took 98 (dropout) to 177 us
// (attention), as nodes here 58 to 91 (the engine's own hand-over to its device thread and
// back is 40). Argument checks raise ValueError; a status other than FH_OK raises FlashHogError, from the forward
// and from the engine's threads alike.
//
// Forward mode and torch.func transforms stay with the Functions of attention.py, which
// have their rules: its entry point sends transformed calls there, and a transformed
// cotangent goes back to them from here.
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
  decltype(&fh_attn_sink_scratch_floats) sink_scratch_floats = nullptr;
  decltype(&fh_attn_fwd) attn_fwd = nullptr;
  decltype(&fh_attn_bwd) attn_bwd = nullptr;
  decltype(&fh_attn_bwdbwd_o) attn_bwdbwd = nullptr;
  decltype(&fh_attn_fwd_f32) attn_fwd_f32 = nullptr;
  decltype(&fh_attn_bwd_f32) attn_bwd_f32 = nullptr;
  decltype(&fh_attn_bwdbwd_f32) attn_bwdbwd_f32 = nullptr;
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

// Whether a torch.func transform is at work: tensors may then be wrappers without storage, and
// under grad new ones are.
bool transforms_active() {
  return c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode);
}

// Every tensor on the first's CUDA device, outside torch.func transforms.
void same_device(const Tensor& t, std::initializer_list<const Tensor*> others) {
  TORCH_CHECK_VALUE(t.is_cuda(), "flash_hog_b200 runs on CUDA tensors only");
  TORCH_CHECK_NOT_IMPLEMENTED(!transforms_active(), "this op does not run under torch.func transforms");
  for (const Tensor* x : others) {
    if (!x->defined()) continue;
    TORCH_CHECK_VALUE(x->device() == t.device(), "tensors must be on one CUDA device, got ", t.device(), " and ",
                      x->device());
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
  const int n = static_cast<int>(tokens.numel()), vocab = static_cast<int>(w.size(0));
  const int dim = static_cast<int>(w.size(1));
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
  TORCH_CHECK_VALUE(tokens.numel() < (1ll << 31) - 1024 && vocab < (1ll << 31) - 1 && weight.size(1) <= (1 << 20),
                    "embedding: fewer than 2^31 - 1024 tokens and 2^31 - 1 table rows of at most 2^20 elements");
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
  TORCH_CHECK_VALUE(rows < (1ll << 31) - 1024 && logits.size(1) < (1ll << 31) - 1024,
                    "policy_loss: fewer than 2^31 - 1024 rows and columns");
  TORCH_CHECK_VALUE(!actions.is_floating_point() && actions.dim() == 1 && actions.size(0) == rows,
                    "policy actions are an integer vector of one entry per row");
  same_device(logits, {&actions, &old_logprobs, &advantages});
  // A constant per row, in fp32.
  auto vec = [&](const Tensor& t) {
    TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == rows,
                      "the policy's per-row inputs are vectors of one entry per row");
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

// ------------------------------------------------------------------------------------
// Dense attention
// ------------------------------------------------------------------------------------

// What a call is besides its tensors.
struct Attn {
  int causal, window, sinks;
  double scale;
  bool f32;  // fp32 kernels; otherwise bf16 operands
  void save(AutogradContext* ctx) const {
    ctx->saved_data["mask"] = c10::IValue(std::vector<int64_t>{causal, window, sinks, f32});
    ctx->saved_data["scale"] = scale;
  }
  static Attn load(AutogradContext* ctx) {
    const auto m = ctx->saved_data["mask"].toIntVector();
    return Attn{static_cast<int>(m[0]), static_cast<int>(m[1]), static_cast<int>(m[2]),
                ctx->saved_data["scale"].toDouble(), m[3] != 0};
  }
  Tensor operand(const Tensor& t) const { return t.to(f32 ? at::kFloat : at::kBFloat16).contiguous(); }
  // Contiguous (batch, tokens, heads, head_dim) tensors; a dimension of size 1 is never stepped over.
  static fh_strides strides(const Tensor& t) {
    const int64_t d = t.size(3), h = t.size(2), n = t.size(1);
    return fh_strides{t.size(0) > 1 ? n * h * d : 0, n > 1 ? h * d : 8, h > 1 ? d : 0};
  }
  fh_attn_dims dims(const Tensor& q, const Tensor& k) const {
    fh_attn_dims d{};
    d.batch = static_cast<int32_t>(q.size(0));
    d.heads = static_cast<int32_t>(q.size(2));
    d.seq_q = static_cast<int32_t>(q.size(1));
    d.seq_k = static_cast<int32_t>(k.size(1));
    d.head_dim = static_cast<int32_t>(q.size(3));
    d.q = strides(q);
    d.k = strides(k);
    d.kv_heads = static_cast<int32_t>(k.size(2));
    d.window = window;
    d.sinks = sinks;
    return d;
  }
  // The scratch that lets the key passes split the sinks' tiles; the result keeps it alive.
  Tensor sink_scratch(fh_attn_dims& d, const Tensor& q) const {
    if (sinks == 0 || f32) return Tensor();
    const long long n = api.sink_scratch_floats(&d, causal);
    if (n <= 0) return Tensor();  // not used, or dims that the call itself refuses
    Tensor t = at::empty({n}, q.options().dtype(at::kFloat));
    d.sink_scratch = t.data_ptr();
    return t;
  }
};

// (out in q's dtype, log-sum-exp)
variable_list attn_forward(const Attn& a, const Tensor& query, const Tensor& key, const Tensor& value) {
  c10::cuda::CUDAGuard guard(query.device());
  const Tensor q = a.operand(query), k = a.operand(key), v = a.operand(value);
  Tensor out = at::empty_like(q), lse = at::empty({q.size(0), q.size(2), q.size(1)}, q.options().dtype(at::kFloat));
  const fh_attn_dims d = a.dims(q, k);
  const float scale = static_cast<float>(a.scale);
  if (a.f32)
    check("fh_attn_fwd_f32", api.attn_fwd_f32(stream_of(q), &d, floats(q), floats(k), floats(v), floats(out),
                                              floats(lse), scale, a.causal));
  else
    check("fh_attn_fwd", api.attn_fwd(stream_of(q), &d, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                                      floats(lse), scale, a.causal));
  return {out.to(query.scalar_type()), lse};
}

// (dq, dk, dv) in the dtypes of q, k, v.
variable_list attn_backward(const Attn& a, const Tensor& query, const Tensor& key, const Tensor& value,
                            const Tensor& lse, const Tensor& out, const Tensor& g) {
  c10::cuda::CUDAGuard guard(query.device());
  const Tensor q = a.operand(query), k = a.operand(key), v = a.operand(value), o = a.operand(out), dO = a.operand(g);
  Tensor dq = at::empty_like(q), dk = at::empty_like(k), dv = at::empty_like(v), delta = at::empty_like(lse);
  fh_attn_dims d = a.dims(q, k);
  const Tensor scratch = a.sink_scratch(d, q);
  const float scale = static_cast<float>(a.scale);
  if (a.f32)
    check("fh_attn_bwd_f32",
          api.attn_bwd_f32(stream_of(q), &d, floats(q), floats(k), floats(v), floats(o), floats(dO), floats(lse),
                           floats(dq), floats(dk), floats(dv), floats(delta), scale, a.causal));
  else
    check("fh_attn_bwd", api.attn_bwd(stream_of(q), &d, q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
                                      dO.data_ptr(), floats(lse), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                                      floats(delta), scale, a.causal));
  return {dq.to(query.scalar_type()), dk.to(key.scalar_type()), dv.to(value.scalar_type())};
}

// (dq2, dk2, dv2, ddo) in the dtypes of q, k, v, dO.
variable_list attn_double(const Attn& a, const Tensor& query, const Tensor& key, const Tensor& value,
                          const Tensor& lse, const Tensor& out, const Tensor& g, const Tensor& ddQ, const Tensor& ddK,
                          const Tensor& ddV) {
  c10::cuda::CUDAGuard guard(query.device());
  const Tensor q = a.operand(query), k = a.operand(key), v = a.operand(value), o = a.operand(out), dO = a.operand(g);
  const Tensor ddq = a.operand(ddQ), ddk = a.operand(ddK), ddv = a.operand(ddV);
  Tensor dq2 = at::empty_like(q), ddo = at::empty_like(q), dk2 = at::empty_like(k), dv2 = at::empty_like(k);
  Tensor stats = at::empty({3, lse.numel()}, lse.options());
  float *delta = floats(stats), *dd = delta + lse.numel(), *bvec = dd + lse.numel();
  fh_attn_dims d = a.dims(q, k);
  const Tensor scratch = a.sink_scratch(d, q);
  const float scale = static_cast<float>(a.scale);
  constexpr int kBoth = FH_PASS_QUERY | FH_PASS_KEY;
  if (a.f32)
    check("fh_attn_bwdbwd_f32",
          api.attn_bwdbwd_f32(stream_of(q), &d, floats(q), floats(k), floats(v), floats(o), floats(dO), floats(ddq),
                              floats(ddk), floats(ddv), floats(lse), floats(dq2), floats(ddo), floats(dk2), floats(dv2),
                              delta, dd, bvec, scale, a.causal, kBoth));
  else
    check("fh_attn_bwdbwd_o",
          api.attn_bwdbwd(stream_of(q), &d, q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), dO.data_ptr(),
                          ddq.data_ptr(), ddk.data_ptr(), ddv.data_ptr(), floats(lse), dq2.data_ptr(), ddo.data_ptr(),
                          dk2.data_ptr(), dv2.data_ptr(), delta, dd, bvec, scale, a.causal, kBoth));
  return {dq2.to(query.scalar_type()), dk2.to(key.scalar_type()), dv2.to(value.scalar_type()), ddo.to(g.scalar_type())};
}

// Whether a backward is being batched or differentiated by a torch.func transform or forward
// mode: it is then the Python Functions' (which have those rules), on this node's saved tensors.
bool transformed(const variable_list& grads) {
  if (transforms_active()) return true;
  for (const Tensor& g : grads)
    if (g.defined() && g._fw_grad(0).defined()) return true;
  return false;
}

// flash_hog_b200.attention's `rule` on the tensors and the mask, scale and precision of `a`.
variable_list python_rule(const char* rule, const variable_list& ts, const Attn& a) {
  py::gil_scoped_acquire gil;
  return py::module_::import("flash_hog_b200.attention")
      .attr(rule)(ts, a.causal, a.window, a.sinks, a.scale, a.f32)
      .cast<variable_list>();
}

bool any_tracked(const variable_list& ts) {
  for (const Tensor& t : ts)
    if (tracked(t)) return true;
  return false;
}

Tensor or_zeros(const Tensor& t, const Tensor& like) { return t.defined() ? t : at::zeros_like(like); }

// The last derivative there is: its own raises.
struct AttnDouble : Function<AttnDouble> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                               const Tensor& lse, const Tensor& out, const Tensor& g, const Tensor& ddq,
                               const Tensor& ddk, const Tensor& ddv, const Attn& a) {
    return attn_double(a, q, k, v, lse, out, g, ddq, ddk, ddv);
  }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK_NOT_IMPLEMENTED(false,
                                "flash_bwdbwd has no derivative: third-order derivatives of attention are not "
                                "supported (the reference's double-backward rule is the last one it defines, "
                                "flash_hog/jax/attention.py:100-130)");
  }
};

struct AttnBackward : Function<AttnBackward> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                               const Tensor& lse, const Tensor& out, const Tensor& g, const Attn& a) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({q, k, v, lse, out, g});
    a.save(ctx);
    return attn_backward(a, q, k, v, lse, out, g);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    const Attn a = Attn::load(ctx);
    const Tensor ddq = or_zeros(grads[0], s[0]), ddk = or_zeros(grads[1], s[1]), ddv = or_zeros(grads[2], s[2]);
    variable_list r;
    if (transformed(grads))
      r = python_rule("_transformed_double", {s[0], s[1], s[2], s[3], s[4], s[5], ddq, ddk, ddv}, a);
    else if (any_tracked({s[0], s[1], s[2], s[5], ddq, ddk, ddv}))
      r = AttnDouble::apply(s[0], s[1], s[2], s[3], s[4], s[5], ddq, ddk, ddv, a);
    else
      r = attn_double(a, s[0], s[1], s[2], s[3], s[4], s[5], ddq, ddk, ddv);
    // The formulas carry the dependence of L and O on (Q, K, V): none for them.
    return {r[0], r[1], r[2], {}, {}, r[3], {}};
  }
};

struct AttnForward : Function<AttnForward> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Attn& a) {
    const variable_list r = attn_forward(a, q, k, v);
    // A second backward reaches this node with no cotangent of the output (AttnBackward's
    // formulas carry that path): none instead of zeros spares a pass on them.
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({r[1]});
    ctx->save_for_backward({q, k, v, r[1], r[0]});
    a.save(ctx);
    return r;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor& g = grads[0];
    if (!g.defined()) return {{}, {}, {}, {}};
    const variable_list s = ctx->get_saved_variables();
    const Attn a = Attn::load(ctx);
    variable_list r;
    if (transformed(grads))
      r = python_rule("_transformed_backward", {s[0], s[1], s[2], s[3], s[4], g}, a);
    else if (at::GradMode::is_enabled())
      r = AttnBackward::apply(s[0], s[1], s[2], s[3], s[4], g, a);
    else
      r = attn_backward(a, s[0], s[1], s[2], s[3], s[4], g);
    return {r[0], r[1], r[2], {}};
  }
};

Tensor attention(const Tensor& query, const Tensor& key, const Tensor& value, int64_t causal, int64_t window,
                 int64_t sinks, double scale, bool f32) {
  TORCH_CHECK_VALUE(query.dim() == 4 && key.dim() == 4 && value.dim() == 4, "expected BTNH tensors");
  same_device(query, {&key, &value});
  TORCH_CHECK_VALUE(key.sizes() == value.sizes() && query.size(0) == key.size(0) && query.size(3) == key.size(3),
                    "incompatible shapes q", query.sizes(), " k", key.sizes(), " v", value.sizes());
  TORCH_CHECK_VALUE(key.size(2) > 0 && query.size(2) % key.size(2) == 0, "q_heads (", query.size(2),
                    ") must be a multiple of kv_heads (", key.size(2), ")");
  for (const int64_t n : {query.size(0), query.size(1), query.size(2), key.size(1)})
    TORCH_CHECK_VALUE(n < (1ll << 31), "attention sizes must be below 2^31");
  const Attn a{static_cast<int>(causal), static_cast<int>(window), static_cast<int>(sinks), scale, f32};
  return AttnForward::apply(query, key, value, a)[0];
}

void bind(const py::dict& addresses) {
  auto set = [&](auto& f, const char* name) {
    f = reinterpret_cast<std::remove_reference_t<decltype(f)>>(addresses[name].cast<uintptr_t>());
  };
  set(api.sink_scratch_floats, "fh_attn_sink_scratch_floats");
  set(api.attn_fwd, "fh_attn_fwd");
  set(api.attn_bwd, "fh_attn_bwd");
  set(api.attn_bwdbwd, "fh_attn_bwdbwd_o");
  set(api.attn_fwd_f32, "fh_attn_fwd_f32");
  set(api.attn_bwd_f32, "fh_attn_bwd_f32");
  set(api.attn_bwdbwd_f32, "fh_attn_bwdbwd_f32");
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
  // Without the interpreter's lock, as ctypes calls the library: a launch waits where the GPU's
  // queue is full, and the allocator where it has to free memory.
  using Unlocked = py::call_guard<py::gil_scoped_release>;
  m.def("attention", &attention, Unlocked());
  m.def("embedding", &embedding, Unlocked());
  m.def("dropout", &dropout, Unlocked());
  m.def("policy_loss", &policy_loss, Unlocked());
}
