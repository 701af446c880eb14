"""Windows and sinks of the C ABI up to the largest int32: past the sequences' lengths they
hide, and add, nothing."""

import pytest
import torch

from flash_hog_b200 import _capi

BIG = 2 ** 31 - 1


def _inputs(tq, tk, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    make = lambda t, h: torch.randn(1, t, h, 64, generator=g).to(dtype).cuda()
    return dict(q=make(tq, 4), k=make(tk, 2), v=make(tk, 2), do=make(tq, 4), ddq=make(tq, 4), ddk=make(tk, 2),
                ddv=make(tk, 2))


def _all_passes(x, causal, window, sinks, f32):
    q, k, v, do = (x[n] for n in ("q", "k", "v", "do"))
    sfx = "_f32" if f32 else ""
    kw = dict(window=window, sinks=sinks)
    stat = lambda: torch.full((1, 4, q.shape[1]), float("nan"), device="cuda")
    out, lse = torch.empty_like(q), stat()
    getattr(_capi, "attn_fwd" + sfx)(q, k, v, out, lse, 0.125, causal, **kw)
    dq, dk, dv, delta = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v), stat()
    getattr(_capi, "attn_bwd" + sfx)(q, k, v, out, do, lse, dq, dk, dv, delta, 0.125, causal, **kw)
    dq2, ddo, dk2, dv2 = torch.empty_like(q), torch.empty_like(q), torch.empty_like(k), torch.empty_like(k)
    entry = _capi.attn_bwdbwd_f32 if f32 else _capi.attn_bwdbwd_o
    entry(q, k, v, out, do, x["ddq"], x["ddk"], x["ddv"], lse, dq2, ddo, dk2, dv2, delta, stat(), stat(), 0.125,
          causal, **kw)
    return out, lse, dq, dk, dv, dq2, ddo, dk2, dv2


@pytest.mark.gpu
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("causal,tq,tk", [(1, 200, 200), (1, 300, 130), (2, 300, 130), (2, 130, 300)])
def test_a_window_past_every_length_is_the_causal_mask(causal, tq, tk, f32):
    x = _inputs(tq, tk, torch.float32 if f32 else torch.bfloat16)
    want = _all_passes(x, causal, 0, 0, f32)
    for window, sinks in ((BIG, 0), (BIG - 100, 0), (BIG, BIG)):
        for a, b in zip(_all_passes(x, causal, window, sinks, f32), want):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("tq,tk", [(300, 300), (1, 300), (300, 130)])
def test_sinks_past_every_key_are_all_keys(tq, tk, f32):
    x = _inputs(tq, tk, torch.float32 if f32 else torch.bfloat16, seed=1)
    want = _all_passes(x, 2, 40, tk, f32)
    for a, b in zip(_all_passes(x, 2, 40, BIG, f32), want):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_packed_batch_with_the_largest_window():
    x = _inputs(400, 400, torch.bfloat16, seed=2)
    cu = torch.tensor([0, 150, 150, 400], dtype=torch.int32, device="cuda")
    vl = _capi.Varlen(cu, cu, 250, 250)
    res = []
    for window, sinks in ((0, 0), (BIG, 0), (BIG, BIG)):
        out, lse = torch.empty_like(x["q"]), torch.empty(1, 4, 400, device="cuda")
        _capi.attn_fwd(x["q"], x["k"], x["v"], out, lse, 0.125, 2, window=window, varlen=vl, sinks=sinks)
        dq, dk, dv = torch.empty_like(x["q"]), torch.empty_like(x["k"]), torch.empty_like(x["v"])
        _capi.attn_bwd(x["q"], x["k"], x["v"], out, x["do"], lse, dq, dk, dv, torch.empty_like(lse), 0.125, 2,
                       window=window, varlen=vl, sinks=sinks)
        res.append((out, lse, dq, dk, dv))
    for other in res[1:]:
        for a, b in zip(other, res[0]):
            torch.testing.assert_close(a, b, rtol=2 * 2.0 ** -7, atol=2.0 ** -7)  # sinks: other kernels, a bf16 step
