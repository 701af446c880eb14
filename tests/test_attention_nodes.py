"""The autograd nodes of the public attention op: what reaches them and what they hand on.

Plain dense calls run as C++ nodes; transforms, forward mode and packed batches as the Python
Functions, whose rules a plain graph also needs when its backward is transformed.
"""

import pytest
import torch

MASKS = [dict(), dict(is_causal=True), dict(is_causal=True, causal_alignment="bottom_right", sliding_window_length=40),
         dict(is_causal=True, sliding_window_length=40, sink_tokens=5)]


def _qkv(dtype=torch.bfloat16, b=2, t=200, s=200, h=4, hk=2, d=64, seed=5, grad=True):
    gen = torch.Generator("cuda").manual_seed(seed)
    make = lambda n, heads: torch.randn(b, n, heads, d, device="cuda", generator=gen).to(dtype)
    return [x.requires_grad_(grad) for x in (make(t, h), make(s, hk), make(s, hk))]


def _call(q, k, v, **kw):
    from flash_hog_b200 import dot_product_attention

    return dot_product_attention(q, k, v, **kw)


def _functions(q, k, v, **kw):
    """The same call as the Python Functions make it."""
    from flash_hog_b200 import attention as A

    mask = A._mask_of(kw.get("is_causal", False), kw.get("causal_alignment", "top_left"),
                      kw.get("sliding_window_length"), kw.get("sink_tokens", 0))
    return A._DotProductAttention.apply(q, k, v, mask, q.shape[-1] ** -0.5, "fp32")[0]


def _hvp(f, xs, kw, vs, w):
    out = f(*xs, **kw)
    first = torch.autograd.grad((out * w).sum(), xs, create_graph=True)
    second = torch.autograd.grad(sum((a * b).sum() for a, b in zip(first, vs)), [*xs, w])
    return [out, *first, *second]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("kw", MASKS)
def test_same_values_as_the_functions(kw, dtype):
    """Both call the same kernels on the same operands: every value is the same, bit for bit."""
    xs, vs = _qkv(dtype), _qkv(dtype, seed=6, grad=False)
    w = torch.randn_like(xs[0]).requires_grad_()
    for got, want in zip(_hvp(_call, xs, kw, vs, w), _hvp(_functions, xs, kw, vs, w)):
        assert got.dtype == want.dtype == dtype and torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", MASKS)
def test_batched_cotangents_of_both_backwards(kw):
    """``vmap`` over the backwards runs the batching rules: each slice is the plain one's. (The key
    pass with sinks splits by the batch, so its bf16 sums may round to the other neighbour:
    half a step on each side, 2 * 2^-8 of the value.)"""
    xs = _qkv()
    out = _call(*xs, **kw)
    gs = torch.randn(3, *out.shape, device="cuda").bfloat16()
    batched = torch.func.vmap(lambda g: torch.autograd.grad(out, xs, g, retain_graph=True))(gs)
    for i in range(3):
        for got, want in zip(batched, torch.autograd.grad(out, xs, gs[i], retain_graph=True)):
            torch.testing.assert_close(got[i], want, rtol=2.0 ** -7, atol=1e-3)
    first = torch.autograd.grad((out * gs[0]).sum(), xs, create_graph=True)
    dd = [torch.randn(3, *x.shape, device="cuda").bfloat16() for x in xs]
    batched = torch.func.vmap(lambda *c: torch.autograd.grad(first, xs, c, retain_graph=True))(*dd)
    for i in range(3):
        want = torch.autograd.grad(first, xs, [x[i] for x in dd], retain_graph=True)
        for got, ref in zip(batched, want):
            # Second derivatives are sums of several bf16-product terms that cancel; the split
            # changes the order of their fp32 sums alone, 2^-24 a term, below the last rounding.
            torch.testing.assert_close(got[i], ref, rtol=2.0 ** -7, atol=1e-3 * ref.abs().max().item())


@pytest.mark.gpu
def test_inside_a_transform_of_something_else():
    """A transform that does not wrap q, k, v: the op runs as it does outside."""
    from flash_hog_b200 import dot_product_attention_varlen

    q, k, v = _qkv(grad=False)
    w = torch.randn_like(q)
    want = _call(q, k, v, is_causal=True)
    got, out = torch.func.grad_and_value(lambda w: (_call(q, k, v, is_causal=True).float() * w.float()).sum())(w)
    assert torch.equal(got, want) and torch.isfinite(out)
    cu = torch.tensor([0, 120, 200], dtype=torch.int32, device="cuda")
    run = lambda: dot_product_attention_varlen(q[0], k[0], v[0], cu, cu, 120, 120, is_causal=True)
    want = run()
    got = torch.func.grad(lambda w: (run().float() * w.float()).sum())(w[0])
    assert torch.equal(got, want)
    got = torch.func.vmap(lambda u: (_call(q, k, v) * u).float().sum())(torch.ones(2, 1, device="cuda"))
    assert torch.equal(got[0], got[1])


@pytest.mark.gpu
def test_backward_inside_a_transform():
    """A graph built outside, differentiated while a transform of something else is at work."""
    q, k, v = _qkv()
    out = _call(q, k, v, is_causal=True)
    g = torch.randn_like(out)
    want = torch.autograd.grad(out, (q, k, v), g, retain_graph=True)
    seen = []

    def f(u):
        seen.extend(torch.autograd.grad(out, (q, k, v), g, retain_graph=True))
        return u.sum()

    torch.func.vmap(f)(torch.ones(2, 3, device="cuda"))
    for got, ref in zip(seen, want):
        assert torch.equal(got, ref)


@pytest.mark.gpu
def test_forward_mode_over_a_plain_graph():
    """A cotangent with a tangent, of a graph that was built before forward mode began."""
    import torch.autograd.forward_ad as fwAD

    q, k, v = _qkv(torch.float32)
    out = _call(q, k, v, is_causal=True)
    g, t = torch.randn_like(out), torch.randn_like(out)
    want = torch.autograd.grad(out, (q, k, v), t, retain_graph=True)  # the backward is linear in g
    with fwAD.dual_level():
        grads = torch.autograd.grad(out, (q, k, v), fwAD.make_dual(g, t))
        tangents = [fwAD.unpack_dual(x).tangent for x in grads]
    for got, ref in zip(tangents, want):
        # tdQ of the fp32 kernels also holds the Hessian product of zero tangents: exact zeros.
        torch.testing.assert_close(got, ref, rtol=2e-5, atol=2e-5)


@pytest.mark.gpu
def test_third_order_is_refused():
    q, k, v = _qkv(torch.float32)
    first = torch.autograd.grad(_call(q, k, v).square().sum(), q, create_graph=True)[0]
    second = torch.autograd.grad(first.square().sum(), q, create_graph=True)[0]
    with pytest.raises(NotImplementedError, match="third-order"):
        second.sum().backward()


@pytest.mark.gpu
def test_some_inputs_without_gradient_hooks_and_checkpoint():
    from torch.utils.checkpoint import checkpoint

    q, k, v = _qkv()
    want = torch.autograd.grad(_call(q, k, v, is_causal=True).float().sum(), (q, k, v))
    for x, ref in zip((q, k, v), want):
        args = [y if y is x else y.detach() for y in (q, k, v)]
        assert torch.equal(torch.autograd.grad(_call(*args, is_causal=True).float().sum(), x)[0], ref)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.cuda()):
        out = _call(q, k, v, is_causal=True)
    for got, ref in zip(torch.autograd.grad(out.float().sum(), (q, k, v)), want):
        assert torch.equal(got, ref)
    out = checkpoint(lambda *a: _call(*a, is_causal=True), q, k, v, use_reentrant=False)
    for got, ref in zip(torch.autograd.grad(out.float().sum(), (q, k, v)), want):
        assert torch.equal(got, ref)


@pytest.mark.gpu
def test_one_tensor_as_all_three():
    x = _qkv(torch.float32, hk=4)[0]
    got = torch.autograd.grad(_call(x, x, x, is_causal=True).square().sum(), x)[0]
    parts = [x.detach().clone().requires_grad_() for _ in range(3)]
    want = sum(torch.autograd.grad(_call(*parts, is_causal=True).square().sum(), parts))
    # Three fp32 terms added in another order: 2 * 2^-24 of the largest each.
    assert (got - want).abs().max() <= 2.0 ** -22 * want.abs().max()


@pytest.mark.gpu
def test_inference_mode():
    from flash_hog_b200 import fused

    q, k, v = _qkv()
    w = torch.randn(50, 16, device="cuda", requires_grad=True)
    t = torch.arange(7, device="cuda")
    z = torch.randn(7, 50, device="cuda", requires_grad=True)
    zero, seed = torch.zeros(7, device="cuda"), torch.tensor([5], device="cuda")
    calls = [lambda: _call(q, k, v, is_causal=True), lambda: fused.embedding(t, w, 2.0),
             lambda: fused.dropout(q, 0.5, seed, residual=q), lambda: fused.policy_loss(z, t, zero, zero + 1)[0]]
    for call in calls:
        want = call()
        assert want.requires_grad
        with torch.inference_mode():
            got = call()
        assert got.is_inference() and not got.requires_grad and torch.equal(got, want)
        with torch.no_grad():
            got = call()
        assert not got.requires_grad and torch.equal(got, want)


@pytest.mark.gpu
def test_a_changed_input_is_noticed_and_graphs_are_freed():
    q, k, v = _qkv()
    out = _call(q, k, v)
    out.float().sum().backward()
    with pytest.raises(RuntimeError, match="second time"):
        out.float().sum().backward()
    out = _call(q, k, v)
    with torch.no_grad():
        q.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out.float().sum().backward()


@pytest.mark.gpu
def test_library_errors_and_refusals(monkeypatch):
    from flash_hog_b200._capi import FlashHogError

    q, k, v = _qkv()
    with pytest.raises(ValueError):
        _call(q, k[:1], v[:1])
    with pytest.raises(ValueError, match="multiple"):
        _call(q[:, :, :3], k, v)
    with pytest.raises(ValueError):
        _call(q, k.detach().cpu(), v)
    with pytest.raises(ValueError):
        _call(q[None], k[None], v[None])
    with pytest.raises(FlashHogError):
        _call(q[..., :24], k[..., :24], v[..., :24])
    monkeypatch.setenv("FLASH_HOG_B200_INJECT_ERROR", "fh_attn_bwd")
    out = _call(q, k, v)
    with pytest.raises(FlashHogError, match="fh_attn_bwd"):
        out.float().sum().backward()
    monkeypatch.setenv("FLASH_HOG_B200_INJECT_ERROR", "fh_attn_fwd")
    with pytest.raises(FlashHogError, match="FH_ERR_INJECTED"):
        _call(q, k, v)


@pytest.mark.gpu
@pytest.mark.parametrize("b,t,s", [(0, 4, 4), (1, 0, 4), (1, 4, 0)])
def test_empty_sizes_as_the_functions_take_them(b, t, s):
    xs = _qkv(b=b, t=t, s=s)
    results = []
    for f in (_call, _functions):
        try:
            out = f(*xs)
            results.append([out, *torch.autograd.grad(out.float().sum(), xs)])
        except Exception as e:  # noqa: BLE001 - the same refusal is the point
            results.append(type(e))
    if isinstance(results[0], list):
        for got, want in zip(*results):
            assert torch.equal(got, want)
    else:
        assert results[0] is results[1]
