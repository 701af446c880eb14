"""The embedding lookup with scaling and its gradient by sorted tokens.

fp64 statements: y_i = s W[t_i]; dW[v] = s sum_{t_i = v} dy_i. The lookup rounds twice at
most (the product in fp32, then the type): one half-step of the type plus one of fp32. The
gradient adds a run of c rows in fp32 (at most c roundings of half a step on partial sums
bounded by sum |dy|), scales (one more) and rounds to the type (half a step).
"""

import numpy as np
import pytest
import torch

F32 = torch.finfo(torch.float32).eps / 2


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _inputs(n, vocab, dim, dtype, seed, skew=0.0, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(vocab, dim, generator=g).to(dtype)
    dy = torch.randn(n, dim, generator=g).to(dtype)
    t = (torch.rand(n, generator=g).pow(1 + skew) * vocab).long().clamp_(max=vocab - 1)
    return w.to(device), t.to(device), dy.to(device)


def _check_lookup(y, w, t, scale):
    ref = w.double()[t] * float(np.float32(scale))
    bound = (_half_step(w.dtype) + 2 * F32) * ref.abs()
    assert ((y.double() - ref).abs() <= bound).all()


def _check_grad(dw, t, dy, vocab, scale, padding=None):
    t, dy = t.flatten(), dy.reshape(t.numel(), -1)
    keep = (t >= 0) & (t < vocab)
    if padding is not None:
        keep &= t != padding
    t, dy = t[keep], dy[keep].double()
    zeros = torch.zeros(vocab, dy.shape[1], dtype=torch.float64, device=dy.device)
    ref = zeros.index_add(0, t, dy) * float(np.float32(scale))
    mass = zeros.index_add(0, t, dy.abs()) * abs(scale)
    count = torch.bincount(t, minlength=vocab)[:, None]
    bound = F32 * (count + 1) * mass + _half_step(dw.dtype) * (ref.abs() + F32 * (count + 1) * mass)
    assert ((dw.double() - ref).abs() <= bound).all()
    assert (dw[(count == 0).flatten()] == 0).all()


CASES = [  # n, vocab, dim, skew
    (1, 1, 1, 0), (1, 1000, 64, 0), (31, 7, 3, 0), (32, 33, 8, 0), (33, 1000, 129, 1), (257, 2, 768, 0),
    (1000, 1023, 65, 2), (1001, 1024, 16, 0), (4099, 32000, 72, 3), (5000, 50, 24, 8), (70001, 300, 4, 0),
    (66000, 131072, 12, 4), (300, 1100000, 4, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,vocab,dim,skew", CASES)
def test_lookup_and_gradient(n, vocab, dim, skew, dtype):
    from flash_hog_b200 import fused

    w, t, dy = _inputs(n, vocab, dim, dtype, seed=n + dim, skew=skew)
    w.requires_grad_(True)
    y = fused.embedding(t, w, 1.7)
    assert y.dtype == dtype and y.shape == (n, dim)
    _check_lookup(y.detach(), w.detach(), t, 1.7)
    (dw,) = torch.autograd.grad(y, w, dy)
    _check_grad(dw, t, dy, vocab, 1.7)
    y2 = fused.embedding(t, w, 1.7)
    assert torch.equal(dw, torch.autograd.grad(y2, w, dy)[0])  # no run-to-run differences


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 9, 40, 4096, 20000])
def test_one_token_takes_every_row(n):
    """A single run through every chunk; its neighbours stay zero."""
    from flash_hog_b200 import fused

    w, _, dy = _inputs(n, 5, 130, torch.float32, seed=3)
    w.requires_grad_(True)
    t = torch.full((n,), 3, device="cuda")
    (dw,) = torch.autograd.grad(fused.embedding(t, w), w, dy)
    _check_grad(dw, t, dy, 5, 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("run", [7, 8, 9, 16, 31, 33, 64])
def test_runs_that_end_at_and_around_chunk_borders(run):
    from flash_hog_b200 import fused

    n = 640
    t = (torch.arange(n, device="cuda") // run)[torch.randperm(n, device="cuda")]
    w, _, dy = _inputs(n, n, 20, torch.float32, seed=run)
    w.requires_grad_(True)
    (dw,) = torch.autograd.grad(fused.embedding(t, w), w, dy)
    _check_grad(dw, t, dy, n, 1.0)


@pytest.mark.gpu
def test_no_tokens():
    from flash_hog_b200 import fused

    w = torch.randn(10, 6, device="cuda", requires_grad=True)
    y = fused.embedding(torch.zeros((2, 0), dtype=torch.long, device="cuda"), w)
    assert y.shape == (2, 0, 6)
    (dw,) = torch.autograd.grad(y, w, torch.zeros_like(y))
    assert torch.equal(dw, torch.zeros_like(w))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_padding_and_tokens_outside(dtype):
    from flash_hog_b200 import fused

    w, t, dy = _inputs(500, 40, 24, dtype, seed=1)
    t[::7] = 5
    t[3], t[4], t[5] = -1, 40, 2 ** 40
    w.requires_grad_(True)
    y = fused.embedding(t, w, 2.0, padding_idx=5)
    outside = (t < 0) | (t >= 40)
    assert y[outside].isnan().all()
    _check_lookup(y[~outside].detach(), w.detach(), t[~outside], 2.0)  # padding is looked up like any token
    dy.requires_grad_(True)
    (dw,) = torch.autograd.grad(y, w, dy, create_graph=True)
    _check_grad(dw.detach(), t, dy.detach(), 40, 2.0, padding=5)
    u = torch.randn_like(dw)
    (ddy,) = torch.autograd.grad(dw, dy, u)
    want = 2.0 * u.double()[t.clamp(0, 39)]
    want[outside | (t == 5)] = 0
    assert ((ddy.double() - want).abs() <= (_half_step(dtype) + 2 * F32) * want.abs()).all()


@pytest.mark.gpu
def test_third_order_and_adjoint_identity():
    """<dW, U> = <dy, lookup(U)>, and the derivative of the double backward is the gradient again."""
    from flash_hog_b200 import fused

    w, t, dy = _inputs(300, 37, 12, torch.float32, seed=4)
    w.requires_grad_(True)
    dy.requires_grad_(True)
    u = torch.randn_like(w).requires_grad_(True)
    (dw,) = torch.autograd.grad(fused.embedding(t, w, 0.5), w, dy, create_graph=True)
    (ddy,) = torch.autograd.grad(dw, dy, u, create_graph=True)
    torch.testing.assert_close((dw.double() * u).sum(), (dy.double() * ddy).sum(), rtol=1e-6, atol=1e-4)
    v = torch.randn_like(dy)
    (du,) = torch.autograd.grad(ddy, u, v)
    _check_grad(du, t, v, 37, 0.5)


@pytest.mark.gpu
def test_shapes_strides_and_index_types():
    from flash_hog_b200 import fused

    w = torch.randn(50, 48, device="cuda")[:, ::2].requires_grad_(True)  # not contiguous
    t = torch.randint(0, 50, (6, 4), device="cuda").t()
    y = fused.embedding(t.int(), w, 3.0)
    assert y.shape == (4, 6, 24)
    _check_lookup(y.detach().reshape(24, 24), w.detach(), t.flatten(), 3.0)
    (dw,) = torch.autograd.grad(y.sum(), w)  # an expanded cotangent
    _check_grad(dw, t.flatten(), torch.ones(24, 24, device="cuda"), 50, 3.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tables_and_gradients_off_the_vector_alignment(dtype):
    from flash_hog_b200 import fused

    w = torch.randn(40 * 16 + 1, device="cuda").to(dtype)[1:].view(40, 16).requires_grad_(True)
    dy = torch.randn(100 * 16 + 1, device="cuda").to(dtype)[1:].view(100, 16)
    t = torch.randint(0, 40, (100,), device="cuda")
    y = fused.embedding(t, w, 0.7)
    _check_lookup(y.detach(), w.detach(), t, 0.7)
    (dw,) = torch.autograd.grad(y, w, dy)
    _check_grad(dw, t, dy, 40, 0.7)


@pytest.mark.gpu
def test_module_matches_nn_embedding():
    from flash_hog_b200 import fused

    torch.manual_seed(0)
    ref = torch.nn.Embedding(100, 32, padding_idx=-2).cuda()
    ours = fused.Embedding(100, 32, padding_idx=-2).cuda()
    ours.load_state_dict(ref.state_dict())
    t = torch.randint(0, 100, (3, 50), device="cuda")
    assert torch.equal(ours(t), ref(t))
    g = torch.randn(3, 50, 32, device="cuda")
    ref(t).backward(g)
    ours(t).backward(g)
    torch.testing.assert_close(ours.weight.grad, ref.weight.grad, rtol=1e-5, atol=1e-5)


@pytest.mark.gpu
def test_captured_and_replayed_with_other_tokens():
    from flash_hog_b200 import fused

    w, t, dy = _inputs(777, 90, 40, torch.float32, seed=6)

    def step():
        v = w.detach().requires_grad_(True)
        y = fused.embedding(t, v, 1.5)
        return y, torch.autograd.grad(y, v, dy)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, dw = step()
    for seed in (1, 2):
        _, t2, dy2 = _inputs(777, 90, 40, torch.float32, seed=seed, skew=seed)
        t.copy_(t2)
        dy.copy_(dy2)
        graph.replay()
        _check_lookup(y, w, t2, 1.5)
        _check_grad(dw, t2, dy2, 90, 1.5)


@pytest.mark.gpu
def test_two_streams_at_once():
    from flash_hog_b200 import fused

    data = [_inputs(4000, 3000, 64, torch.float32, seed=s, skew=s) for s in range(2)]
    streams = [torch.cuda.Stream() for _ in data]
    torch.cuda.synchronize()
    outs = []
    for _ in range(3):
        for (w, t, dy), s in zip(data, streams):
            with torch.cuda.stream(s):
                v = w.detach().requires_grad_(True)
                outs.append(torch.autograd.grad(fused.embedding(t, v), v, dy)[0])
    torch.cuda.synchronize()
    for i, dw in enumerate(outs):
        _check_grad(dw, data[i % 2][1], data[i % 2][2], 3000, 1.0)


def test_refusals():
    from flash_hog_b200 import fused

    w, t = torch.zeros(10, 4), torch.zeros(3, dtype=torch.long)
    with pytest.raises(ValueError):
        fused.embedding(t, w)  # CPU tensors
    with pytest.raises(ValueError):
        fused.embedding(t.float(), w)
    with pytest.raises(ValueError):
        fused.embedding(t, w.half())
    with pytest.raises(ValueError):
        fused.embedding(t, w[0])
    with pytest.raises(ValueError):
        fused.embedding(t, w[:0])
    for bad in (-1, 10):
        with pytest.raises(ValueError):
            fused.embedding(t, w, padding_idx=bad)
    with pytest.raises(ValueError):
        fused.Embedding(10, 4, max_norm=1.0)


def test_c_abi_refusals():
    import ctypes

    from flash_hog_b200._capi import lib

    h, p, odd = lib(), ctypes.c_void_p(64), ctypes.c_void_p(72)
    assert h.fh_embed_scratch_bytes(-1, 4) == -1 and h.fh_embed_scratch_bytes(0, 4) == 0
    assert h.fh_embed_scratch_bytes(100, 4) >= 16 * 100
    assert h.fh_embed_scratch_bytes(2 ** 31 - 1, 4) == -1             # 32-bit positions, a block past the end
    assert h.fh_embed_scratch_bytes(2 ** 31 - 1025, 4) >= 16 * (2 ** 31 - 1025)
    assert h.fh_embed_bwd(None, 0, 2 ** 31 - 1024, 1, 1, p, p, 1.0, -1, p, p) == 1
    assert h.fh_embed_fwd(None, 2, 1, 1, 1, p, p, 1.0, p) == 1        # dtype
    assert h.fh_embed_fwd(None, 0, 1, 0, 1, p, p, 1.0, p) == 1        # empty table
    assert h.fh_embed_fwd(None, 0, 1, 1, 1, None, p, 1.0, p) == 1
    assert h.fh_embed_fwd(None, 0, 0, 1, 1, None, None, 1.0, None) == 0  # no tokens
    assert h.fh_embed_bwd(None, 0, 1, 1, 1, p, p, 1.0, -1, odd, p) == 1  # dw not aligned
    assert h.fh_embed_bwd(None, 0, 1, 1, 1, p, p, 1.0, -1, p, None) == 1
    assert h.fh_embed_bwd_bwd(None, 0, -1, 1, 1, p, p, 1.0, -1, p) == 1


# Lists long enough for the chunks of 64 (from 151584 tokens on) and of 128 (303168).
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [160000, 163841, 320000, 327681])
@pytest.mark.parametrize("vocab,skew", [(300000, 0), (5000, 8), (1, 0)])
def test_long_lists(vocab, skew, n, dtype):
    from flash_hog_b200 import fused

    w, t, dy = _inputs(n, vocab, 8, dtype, n + vocab, skew)
    w.requires_grad_(True)
    (dw,) = torch.autograd.grad(fused.embedding(t, w, 0.5), w, dy)
    _check_grad(dw, t, dy, vocab, 0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [160000, 320000])
@pytest.mark.parametrize("run", [63, 64, 65, 127, 128, 129, 191, 256, 1151])
def test_runs_around_the_borders_of_long_chunks(run, n):
    """Runs that end at, one before and one after multiples of 64 and 128, up to those that a
    block joins together."""
    from flash_hog_b200 import fused

    vocab = (n + run - 1) // run
    w, _, dy = _inputs(n, vocab, 4, torch.float32, run)
    t = (torch.arange(n) // run)[torch.randperm(n, generator=torch.Generator().manual_seed(run))].cuda()
    w.requires_grad_(True)
    (dw,) = torch.autograd.grad(fused.embedding(t, w), w, dy)
    _check_grad(dw, t, dy, vocab, 1.0)
