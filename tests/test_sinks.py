"""Sliding windows with sinks: the first S keys stay visible behind the window.

Query i sees key j iff j <= d_i and (d_i - j < W or j < S), d_i the query's diagonal key.
Every kernel of the attention op takes the mask: forward, backward, double backward and
the forward-mode passes, in bf16 and fp32, dense and packed.
"""

import ctypes

import numpy as np
import pytest
import torch

from oracle import attention_oracle as ora
from tests.parity_util import assert_close, assert_elementwise, np64
from tests.test_varlen import _packed_inputs, _seq

# fp32 products and sums: a row's longest chain here is head_dim + 1000 keys, twice in a row
# for the double backward: 2 * 1128 * 2^-24 = 1.3e-4 of the largest value at the very worst.
F32_TOL = 1.4e-4


def _loop(nq, nk, causal, window, sinks):
    keep = np.zeros((nq, nk), dtype=bool)
    for i in range(nq):
        d = i + (nk - nq if causal == 2 else 0)
        for j in range(nk):
            keep[i, j] = j <= d and (d - j < window or j < sinks)
    return keep


@pytest.mark.parametrize("nq,nk,causal,window,sinks", [(10, 20, 2, 5, 3), (20, 10, 1, 4, 2), (16, 16, 1, 1, 1),
                                                       (13, 7, 2, 3, 9), (6, 40, 2, 4, 30)])
def test_mask_statement(nq, nk, causal, window, sinks):
    assert np.array_equal(ora.causal_mask(nq, nk, causal, (window, sinks)), _loop(nq, nk, causal, window, sinks))


def _tiles(tq, tk, diag, window, sinks, r0, rows, bn):
    """The kernels' list of key tiles of a block of query rows (attn_common.cuh), restated."""
    r1 = min(r0 + rows, tq) - 1
    if r1 < r0:
        return []
    lo, hi = max(0, r0 + diag - window + 1), min(tk - 1, r1 + diag)
    if hi < 0:
        return []
    front, first, end = -(-min(sinks, hi + 1) // bn), lo // bn, hi // bn + 1
    if hi < lo:
        return list(range(front))
    if first <= front:
        return list(range(end))
    return list(range(front)) + list(range(first, end))


@pytest.mark.parametrize("causal", [1, 2])
@pytest.mark.parametrize("tq,tk,window,sinks", [(300, 300, 40, 4), (257, 700, 64, 130), (500, 130, 33, 7),
                                                (1, 900, 128, 64), (300, 260, 70, 300), (200, 200, 1, 1)])
def test_key_tiles_cover_the_mask_once(tq, tk, window, sinks, causal):
    keep = _loop(tq, tk, causal, window, sinks)
    diag = tk - tq if causal == 2 else 0
    for rows, bn in ((128, 64), (128, 32), (256, 128), (64, 64)):
        for r0 in range(0, tq, rows):
            tiles = _tiles(tq, tk, diag, window, sinks, r0, rows, bn)
            assert len(tiles) == len(set(tiles))
            seen = {int(j) // bn for j in np.nonzero(keep[r0:r0 + rows].any(0))[0]}
            assert seen <= set(tiles)


CASES = [  # b, h, hk, tq, tk, causal, window, sinks, d
    (1, 2, 2, 600, 600, 1, 64, 4, 64),       # a few sinks behind a short window
    (1, 2, 1, 700, 900, 2, 100, 130, 64),    # sinks past a tile, grouped heads, bottom-right
    (1, 4, 2, 513, 513, 1, 17, 1, 128),      # one sink, ragged, head_dim 128
    (1, 2, 2, 300, 260, 2, 70, 5, 64),       # queries that see no key
    (1, 2, 2, 300, 260, 2, 70, 5, 128),
    (2, 2, 2, 1, 777, 2, 128, 4, 64),        # single tokens
    (2, 4, 1, 1, 777, 2, 128, 4, 128),
    (1, 2, 2, 400, 900, 2, 1, 200, 128),     # a window of the diagonal alone
    (1, 2, 2, 800, 130, 1, 40, 6, 64),       # queries past the last key's window see the sinks alone
    (1, 2, 2, 800, 130, 1, 40, 6, 128),
    (1, 1, 1, 260, 260, 1, 300, 16, 64),     # a window that hides nothing
    (1, 2, 2, 520, 520, 1, 128, 512, 128),   # sinks that overlap most windows
    (1, 2, 2, 384, 384, 1, 64, 64, 64),      # sinks and window at tile edges
    (1, 3, 3, 129, 129, 1, 1, 128, 64),      # sinks that end with the last tile's first key
    (1, 1, 1, 1, 1, 1, 1, 1, 64),
]


def _inputs(b, h, hk, tq, tk, d, dtype, seed=3):
    x = ora.make_inputs(b, h, tq, tk, d, seed=seed, kv_heads=hk, dtype=dtype)
    x["tdo"] = torch.randn(x["do"].shape, generator=torch.Generator().manual_seed(seed + 1)).to(dtype)
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("b,h,hk,tq,tk,causal,window,sinks,d", CASES)
def test_all_passes_match_the_oracle(b, h, hk, tq, tk, causal, window, sinks, d, dtype):
    from flash_hog_b200 import _attention_impl as impl
    from flash_hog_b200 import _capi
    from flash_hog_b200._attention_impl import MaskType, SlidingWindow
    from flash_hog_b200.bwdbwd import flash_bwdbwd

    x = _inputs(b, h, hk, tq, tk, d, dtype)
    c = {n: t.cuda() for n, t in x.items()}
    mask = SlidingWindow(MaskType(causal), window, sinks)
    sc = d ** -0.5
    a = {n: t.double().numpy() for n, t in x.items()}
    kw = dict(scale=sc, causal=causal, window=(window, sinks))
    bf16 = dtype == torch.bfloat16

    def close(name, got, want):
        got = got.double().cpu().numpy()
        if np.abs(want).max(initial=0) < 1e-3:
            # One visible key: softmax is constant and terms up to 1e3 cancel. What is left of the
            # statement is the fp32 L's rounding, 2^-23 of them: 1e-4; of bf16 products 2^-9: 2.
            assert np.abs(got).max() < (2.0 if bf16 else 1e-3)
        elif bf16:
            assert_close(name, got, want)
            assert_elementwise(name, got, want)
        else:
            assert_close(name, got, want, F32_TOL)

    o, lse = impl.cuda_dot_product_attention(c["q"], c["k"], c["v"], mask, sc, return_residual=True)
    o_r, lse_r = ora.attention_fwd(a["q"], a["k"], a["v"], **kw)
    close("O", o, o_r)
    lse_np = lse.cpu().numpy()
    assert np.array_equal(np.isneginf(lse_np), np.isneginf(lse_r))
    fin = np.isfinite(lse_r)
    assert np.abs(lse_np[fin] - lse_r[fin]).max(initial=0) < (2e-2 if bf16 else 1e-4)
    a["o"], a["lse"] = o.double().cpu().numpy(), lse.double().cpu().numpy()
    res = (c["q"], c["k"], c["v"], lse, o)
    first = impl.dot_product_attention_bwd_rule(mask, sc, res, c["do"])
    for name, got, want in zip(("dQ", "dK", "dV"), first,
                               ora.attention_bwd(a["q"], a["k"], a["v"], a["o"], a["lse"], a["do"], **kw)):
        close(name, got, want)
    outs = flash_bwdbwd(c["q"], c["k"], c["v"], o, c["do"], c["ddq"], c["ddk"], c["ddv"], lse, mask_type=mask, scale=sc)
    ref = ora.bwdbwd_stats(a["q"], a["k"], a["v"], a["o"], a["lse"], a["do"], a["ddq"], a["ddk"], a["ddv"], **kw)
    for name, got, want in zip(("dQ'", "dK'", "dV'", "ddO"), outs, ref):
        close(name, got, want)
    to, _ = impl.dot_product_attention_fwd_jvp(mask, sc, res, (c["ddq"], c["ddk"], c["ddv"]))
    close("tO", to, ora.jvp_fwd(a["q"], a["k"], a["v"], a["o"], a["lse"], a["ddq"], a["ddk"], a["ddv"], **kw)[0])
    jvp = impl.dot_product_attention_bwd_jvp(mask, sc, res, c["do"], (c["ddq"], c["ddk"], c["ddv"], c["tdo"]))
    ref = ora.jvp_bwd(a["q"], a["k"], a["v"], a["o"], a["lse"], a["do"], a["ddq"], a["ddk"], a["ddv"], a["tdo"], **kw)
    for name, got, want in zip(("tdQ", "tdK", "tdV"), jvp, ref):
        close(name, got, want)
    assert _capi.device_status() == 0


FEW = [  # b, h, hk, tq, tk, causal, window, sinks
    (3, 4, 4, 1, 2000, 2, 300, 4), (2, 8, 2, 1, 5000, 2, 1024, 4), (1, 8, 1, 1, 8192, 2, 4096, 64),
    (2, 2, 2, 5, 900, 2, 100, 3), (1, 4, 2, 4, 333, 2, 17, 40), (1, 8, 1, 1, 40, 2, 7, 9), (300, 1, 1, 1, 90, 2, 16, 1),
    (1, 2, 2, 3, 64, 1, 2, 1), (2, 2, 1, 4, 3, 2, 1, 1), (1, 1, 1, 8, 500, 2, 1, 1), (2, 3, 3, 7, 300, 2, 64, 255),
    (2, 4, 2, 8, 700, 2, 99, 5), (1, 16, 1, 1, 1000, 2, 2000, 4), (3, 5, 1, 3, 129, 2, 128, 1),
]


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("b,h,hk,tq,tk,causal,window,sinks", FEW)
def test_few_query_rows(b, h, hk, tq, tk, causal, window, sinks, packed, d):
    """Single tokens and a handful: fp32 sums, probabilities to 2^-17, so within the output's
    rounding (half a step of bf16, 2^-8: it has 8 significant bits) and 2^-13 of the largest
    value (sums of up to 4160 terms near 1e-5 off)."""
    from flash_hog_b200 import _capi

    x = {n: t.cuda() for n, t in _inputs(b, h, hk, tq, tk, d, torch.bfloat16).items()}
    q, k, v = x["q"], x["k"], x["v"]
    o, lse = torch.full_like(q, float("nan")), torch.full((b, h, tq), float("nan"), device="cuda")
    if packed:
        fold = lambda t: t.reshape(1, -1, *t.shape[2:])
        cu = lambda t: torch.arange(0, b * t + 1, t, dtype=torch.int32, device="cuda")
        vl = _capi.Varlen(cu(tq), cu(tk), tq, tk)
        _capi.attn_fwd(fold(q), fold(k), fold(v), fold(o), lse, d ** -0.5, causal, window, vl, sinks)
        lse = lse.reshape(h, b, tq).transpose(0, 1)
    else:
        _capi.attn_fwd(q, k, v, o, lse, d ** -0.5, causal, window, None, sinks)
    keep = torch.from_numpy(ora.causal_mask(tq, tk, causal, (window, sinks))).cuda()
    kk, vv = (t.double().repeat_interleave(h // hk, 2) for t in (k, v))
    s = torch.einsum("bqhd,bkhd->bhqk", q.double(), kk) * d ** -0.5
    s = s.masked_fill(~keep, float("-inf"))
    blind = ~keep.any(1)
    p = torch.where(blind[:, None], 0.0, s.softmax(-1))
    want = torch.einsum("bhqk,bkhd->bqhd", p, vv)
    assert ((o.double() - want).abs() <= torch.finfo(torch.bfloat16).eps / 2 * want.abs() + 2.0 ** -13 * vv.abs().max()).all()
    ref = torch.logsumexp(s, -1)
    assert torch.equal(lse.isneginf(), blind.expand(b, h, tq))
    assert (lse[..., ~blind].double() - ref[..., ~blind]).abs().max() <= 1e-4 if (~blind).any() else True
    assert _capi.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
def test_no_sinks_and_all_sinks_are_the_masks_there_are(d):
    """Sinks of 0: the window's kernels, bit for bit. As many sinks as keys: causal attention."""
    import flash_hog_b200 as fhb

    x = {n: t.cuda() for n, t in _inputs(1, 2, 2, 400, 400, d, torch.bfloat16).items()}
    kw = dict(is_causal=True, sliding_window_length=100)
    a = fhb.dot_product_attention(x["q"], x["k"], x["v"], **kw)
    assert torch.equal(fhb.dot_product_attention(x["q"], x["k"], x["v"], sink_tokens=0, **kw), a)
    full = fhb.dot_product_attention(x["q"], x["k"], x["v"], is_causal=True)
    for s in (400, 2 ** 40):
        got = fhb.dot_product_attention(x["q"], x["k"], x["v"], sink_tokens=s, **kw)
        assert_close("O", np64(got), np64(full))
    got = fhb.dot_product_attention(x["q"], x["k"], x["v"], is_causal=True, sliding_window_length=2 ** 40, sink_tokens=3)
    assert torch.equal(got, full)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_public_op_twice_differentiated(dtype):
    import flash_hog_b200 as fhb

    x = ora.make_inputs(1, 4, 333, 400, 64, seed=6, kv_heads=2, dtype=dtype)
    ref = ora.autograd_all(*(x[n].double() for n in ("q", "k", "v", "do", "ddq", "ddk", "ddv")), causal=2, window=(60, 9))
    c = {n: t.cuda() for n, t in x.items()}
    q, k, v, do = (c[n].clone().requires_grad_(True) for n in ("q", "k", "v", "do"))
    o = fhb.dot_product_attention(q, k, v, is_causal=True, causal_alignment="bottom_right", sliding_window_length=60,
                                  sink_tokens=9)
    first = torch.autograd.grad(o, (q, k, v), do, create_graph=True)
    second = torch.autograd.grad(first, (q, k, v, do), (c["ddq"], c["ddk"], c["ddv"]))
    tol = 2e-2 if dtype == torch.bfloat16 else F32_TOL
    for n, t in zip(("o", "dq", "dk", "dv", "dq2", "dk2", "dv2", "ddo"), (o, *first, *second)):
        assert_close(n, np64(t), ref[n].numpy(), tol)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["btnh", "bhtd", "padded"])
def test_strided_inputs(layout):
    """Heads outermost, or rows of a wider buffer: the same values, the same result."""
    import flash_hog_b200 as fhb

    x = {n: t.cuda() for n, t in _inputs(2, 2, 2, 300, 300, 64, torch.bfloat16).items()}
    kw = dict(is_causal=True, sliding_window_length=50, sink_tokens=7)
    want = fhb.dot_product_attention(x["q"], x["k"], x["v"], **kw)

    def relay(t):
        if layout == "bhtd":
            return t.transpose(1, 2).contiguous().transpose(1, 2)
        if layout == "padded":
            wide = torch.randn(*t.shape[:3], 2 * t.shape[3], device="cuda").to(t.dtype)
            wide[..., :t.shape[3]] = t
            return wide[..., :t.shape[3]]
        return t

    assert torch.equal(fhb.dot_product_attention(*(relay(x[n]) for n in ("q", "k", "v")), **kw), want)


@pytest.mark.gpu
@pytest.mark.parametrize("causal,h,hk,d", [(1, 2, 2, 64), (2, 4, 2, 128), (2, 2, 1, 64)])
def test_packed_batch_equals_per_sequence_calls(causal, h, hk, d):
    """The sinks are each sequence's own first keys; sequences without queries or keys included."""
    from flash_hog_b200 import _capi

    lq, lk, window, sinks = [200, 0, 333, 5, 64], [350, 40, 333, 0, 500], 48, 20
    x, cq, ck = _packed_inputs(lq, lk, h, hk, d, seed=7)
    g = {n: t.cuda() for n, t in x.items()}
    scale = d ** -0.5

    def passes(s, vl):
        kw = dict(window=window, sinks=sinks, varlen=vl)
        o, lse = torch.empty_like(s["q"]), torch.empty((1, h, s["q"].shape[1]), dtype=torch.float32, device="cuda")
        _capi.attn_fwd(s["q"], s["k"], s["v"], o, lse, scale, causal, **kw)
        dq, dk, dv = torch.empty_like(s["q"]), torch.empty_like(s["k"]), torch.empty_like(s["v"])
        _capi.attn_bwd(s["q"], s["k"], s["v"], o, s["do"], lse, dq, dk, dv, torch.empty_like(lse), scale, causal, **kw)
        dq2, ddo, dk2, dv2 = (torch.empty_like(s[n]) for n in ("q", "q", "k", "k"))
        _capi.attn_bwdbwd_o(s["q"], s["k"], s["v"], o, s["do"], s["ddq"], s["ddk"], s["ddv"], lse, dq2, ddo, dk2, dv2,
                            *[torch.empty_like(lse) for _ in range(3)], scale, causal, **kw)
        return {"q": (o, dq, dq2, ddo), "k": (dk, dv, dk2, dv2), "lse": lse}

    got = passes(g, _capi.Varlen(cq.cuda(), ck.cuda(), max(lq), max(lk)))
    for b in range(len(lq)):
        if lk[b] == 0:
            assert all((_seq(t, cq, b) == 0).all() for t in got["q"])
            continue
        if lq[b] == 0:
            assert all((_seq(t, ck, b) == 0).all() for t in got["k"])
            continue
        s = {n: _seq(g[n], cq if n in ("q", "do", "ddq") else ck, b).contiguous() for n in g}
        want = passes(s, None)
        for t, w in zip(got["q"], want["q"]):
            assert torch.equal(_seq(t, cq, b), w)
        for t, w in zip(got["k"], want["k"]):
            assert_close("key side", np64(_seq(t, ck, b)), np64(w))
        assert torch.equal(got["lse"][:, :, int(cq[b]):int(cq[b + 1])], want["lse"])
    assert _capi.device_status() == 0


@pytest.mark.gpu
def test_public_varlen_op():
    import flash_hog_b200 as fhb

    lq, lk = [150, 256, 1], [200, 256, 90]
    x, cq, ck = _packed_inputs(lq, lk, 2, 2, 64, seed=5)
    q, k, v, do = (x[n][0].cuda().requires_grad_(True) for n in ("q", "k", "v", "do"))
    kw = dict(is_causal=True, causal_alignment="bottom_right", sliding_window_length=32, sink_tokens=5)
    out = fhb.dot_product_attention_varlen(q, k, v, cq.cuda(), ck.cuda(), max(lq), max(lk), **kw)
    first = torch.autograd.grad(out, (q, k, v), do, create_graph=True)
    second = torch.autograd.grad(first[0].float().square().sum(), (q, k, v, do))
    assert all(t.isfinite().all() for t in second)
    for b in range(len(lq)):
        sq, sk = slice(int(cq[b]), int(cq[b + 1])), slice(int(ck[b]), int(ck[b + 1]))
        one = fhb.dot_product_attention(q[sq][None], k[sk][None], v[sk][None], **kw)[0]
        if lq[b] > 16:
            assert torch.equal(out[sq], one)
        else:
            # Alone, few rows run a kernel with finer probabilities; the packed batch's rounds them
            # to bf16 (2^-8 of each), and both round their output (2^-8).
            bound = 2.0 ** -8 * (v[sk].float().abs().amax(0) + 2 * one.float().abs())
            assert ((out[sq].float() - one.float()).abs() <= bound).all()


@pytest.mark.gpu
def test_vmap_folds_the_sinks_too():
    import flash_hog_b200 as fhb

    x = {n: t.cuda() for n, t in _inputs(4, 2, 2, 200, 200, 64, torch.bfloat16).items()}
    kw = dict(is_causal=True, sliding_window_length=30, sink_tokens=5)
    fold = {n: x[n].view(2, 2, *x[n].shape[1:]) for n in ("q", "k", "v", "do", "ddq", "ddk", "ddv")}

    def hvp(q, k, v, do, *tangents):
        def grads(*a):
            return torch.func.vjp(lambda *b: fhb.dot_product_attention(*b, **kw), *a)[1](do)
        return torch.func.vjp(grads, q, k, v)[1](tangents)

    names = ("q", "k", "v", "do", "ddq", "ddk", "ddv")
    got = torch.func.vmap(hvp)(*(fold[n] for n in names))
    for i in range(2):
        for a, b in zip(got, hvp(*(fold[n][i] for n in names))):
            assert_close("vmap", np64(a[i]), np64(b))


@pytest.mark.gpu
def test_captured_and_replayed():
    import flash_hog_b200 as fhb

    x = {n: t.cuda() for n, t in _inputs(1, 2, 2, 500, 500, 64, torch.bfloat16).items()}
    kw = dict(is_causal=True, sliding_window_length=64, sink_tokens=4)

    def step():
        q, k, v = (x[n].detach().requires_grad_(True) for n in ("q", "k", "v"))
        o = fhb.dot_product_attention(q, k, v, **kw)
        first = torch.autograd.grad(o, (q, k, v), x["do"], create_graph=True)
        return (o, *first, *torch.autograd.grad(first, (q, k, v), (x["ddq"], x["ddk"], x["ddv"])))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (21, 22):
        for n, t in _inputs(1, 2, 2, 500, 500, 64, torch.bfloat16, seed=seed).items():
            x[n].copy_(t)
        graph.replay()
        got = [t.clone() for t in captured]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_token_step_captured_and_replayed_on_other_contents():
    """A server's captured step: keys and values that grow in place, one query."""
    import flash_hog_b200 as fhb

    x = {n: t.cuda() for n, t in _inputs(3, 8, 2, 1, 600, 64, torch.bfloat16).items()}
    kw = dict(is_causal=True, causal_alignment="bottom_right", sliding_window_length=128, sink_tokens=4)
    run = lambda: fhb.dot_product_attention(x["q"], x["k"], x["v"], **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for seed in (31, 32):
        for n, t in _inputs(3, 8, 2, 1, 600, 64, torch.bfloat16, seed=seed).items():
            x[n].copy_(t)
        graph.replay()
        got = out.clone()
        assert torch.equal(got, run())


@pytest.mark.gpu
def test_hidden_keys_are_not_read_by_tokens():
    """What lies between the sinks and the window (an evicted cache) may hold anything."""
    import flash_hog_b200 as fhb

    x = {n: t.cuda() for n, t in _inputs(2, 4, 2, 1, 900, 64, torch.bfloat16).items()}
    kw = dict(is_causal=True, causal_alignment="bottom_right", sliding_window_length=100, sink_tokens=6)
    want = fhb.dot_product_attention(x["q"], x["k"], x["v"], **kw)
    x["k"][:, 6:800] = float("nan")
    x["v"][:, 6:800] = float("inf")
    assert torch.equal(fhb.dot_product_attention(x["q"], x["k"], x["v"], **kw), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tq", [1, 3, 40])
def test_nan_is_not_hidden(tq, dtype):
    """NaN in a query reaches its own row alone; in a visible key, the rows that see it."""
    import flash_hog_b200 as fhb

    x = {n: t.cuda() for n, t in _inputs(2, 4, 2, tq, 300, 64, dtype).items()}
    kw = dict(is_causal=True, causal_alignment="bottom_right", sliding_window_length=100, sink_tokens=6)
    want = fhb.dot_product_attention(x["q"], x["k"], x["v"], **kw)
    q = x["q"].clone()
    q[1, -1, 2] = float("nan")
    got = fhb.dot_product_attention(q, x["k"], x["v"], **kw)
    assert got[1, -1, 2].isnan().all()
    got[1, -1, 2] = want[1, -1, 2]
    # When a warp rescales may change with a row of it: half a step of the result on each side.
    near = dict(rtol=2 * torch.finfo(dtype).eps, atol=2 * torch.finfo(dtype).eps * want.abs().max().item())
    torch.testing.assert_close(got, want, **near)
    for t in ("k", "v"):
        bad = {**x, t: x[t].clone()}
        bad[t][0, 3, 1] = float("nan")  # a sink of heads 2 and 3
        got = fhb.dot_product_attention(bad["q"], bad["k"], bad["v"], **kw)
        hit = got[0, :, 2:].isnan()
        assert hit.all() if t == "k" else hit.any(-1).all()
        torch.testing.assert_close(got[1], want[1], **near)
        torch.testing.assert_close(got[0, :, :2], want[0, :, :2], **near)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
def test_long_sequences_with_few_heads(d):
    """Most of the sink tiles' work lies on few CTAs: 40 query tiles for one key tile of sinks."""
    import flash_hog_b200 as fhb

    x = {n: t.cuda() for n, t in _inputs(1, 2, 1, 5001, 5001, d, torch.bfloat16).items()}
    q, k, v, do = (x[n].requires_grad_(True) for n in ("q", "k", "v", "do"))
    o = fhb.dot_product_attention(q, k, v, is_causal=True, sliding_window_length=200, sink_tokens=140)
    first = torch.autograd.grad(o, (q, k, v), do, create_graph=True)
    second = torch.autograd.grad(first, (q, k, v, do), (x["ddq"], x["ddk"], x["ddv"]))
    t = [z.detach().double() for z in (q, k, v, do)]
    for z in t:
        z.requires_grad_(True)
    i = torch.arange(5001, device="cuda")
    keep = (i[None] <= i[:, None]) & ((i[:, None] - i[None] < 200) | (i[None] < 140))
    s = torch.einsum("bqhd,bkd->bhqk", t[0], t[1][:, :, 0]) * d ** -0.5
    p = s.masked_fill(~keep, float("-inf")).softmax(-1)
    want = [torch.einsum("bhqk,bkd->bqhd", p, t[2][:, :, 0])]
    want += torch.autograd.grad(want[0], t[:3], t[3], create_graph=True)
    want += torch.autograd.grad(want[1:], t, [x[n].double() for n in ("ddq", "ddk", "ddv")])
    for n, a, b in zip(("o", "dq", "dk", "dv", "dq2", "dk2", "dv2", "ddo"), (o, *first, *second), want):
        assert_close(n, np64(a), b.detach().cpu().numpy())


def test_refusals():
    import flash_hog_b200 as fhb
    from flash_hog_b200._attention_impl import MaskType, SlidingWindow, _mask_args, _mask_kw

    q = torch.zeros(1, 128, 2, 64)
    with pytest.raises(ValueError):
        fhb.dot_product_attention(q, q, q, is_causal=True, sink_tokens=4)
    with pytest.raises(ValueError):
        fhb.dot_product_attention(q, q, q, sink_tokens=4)
    with pytest.raises(ValueError):
        fhb.dot_product_attention(q, q, q, is_causal=True, sliding_window_length=8, sink_tokens=-1)
    with pytest.raises(ValueError):
        fhb.dot_product_attention_varlen(q[0], q[0], q[0], None, None, 1, 1, is_causal=True, sink_tokens=1)
    with pytest.raises(ValueError):
        _mask_args(SlidingWindow(MaskType.NO_MASK, 8, 2))
    assert _mask_args(SlidingWindow(MaskType.CAUSAL, 8, 2)) == (1, 8)
    assert _mask_kw(SlidingWindow(MaskType.CAUSAL, 8, 2)) == {"sinks": 2}
    assert _mask_kw(SlidingWindow(MaskType.CAUSAL, 8)) == {} and _mask_kw(MaskType.CAUSAL) == {}


def test_c_abi_refusals():
    from flash_hog_b200._capi import FhAttnDims, FhStrides, lib

    st, p = FhStrides(128 * 2 * 64, 2 * 64, 64), ctypes.c_void_p(64)

    def fwd(window, sinks, causal=1):
        d = FhAttnDims(1, 2, 128, 128, 64, st, st, 0, window)
        d.sinks = sinks
        return lib().fh_attn_fwd(None, ctypes.byref(d), p, p, p, ctypes.c_void_p(8), p, 0.125, causal)

    assert fwd(8, -1) == 1 and b"sinks" in lib().fh_last_error()
    assert fwd(0, 4) == 1 and b"sliding window" in lib().fh_last_error()
    assert fwd(8, 4) == 1 and b"aligned" in lib().fh_last_error()  # past the mask's checks
