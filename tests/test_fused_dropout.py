"""Dropout from a counter-based generator, with the residual addition.

The mask is restated here in numpy: Philox4x32-10 (Salmon et al., 2011), pinned to its
published known answers. y = r + keep x / (1 - limit / 65536): the factor and the fused
multiply-add round once each in fp32, then once to the type.
"""

import numpy as np
import pytest
import torch

F32 = torch.finfo(torch.float32).eps / 2


def _philox(counter, key):
    """(n, 4) uint32 words of counters (n, 4) under a 64-bit key."""
    c = [counter[:, i].astype(np.uint64) for i in range(4)]
    lo, k = np.uint64(0xFFFFFFFF), [key & 0xFFFFFFFF, (key >> 32) & 0xFFFFFFFF]
    for r in range(10):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        k0, k1 = np.uint64((k[0] + r * 0x9E3779B9) & 0xFFFFFFFF), np.uint64((k[1] + r * 0xBB67AE85) & 0xFFFFFFFF)
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ k0, p1 & lo, (p0 >> np.uint64(32)) ^ c[3] ^ k1, p0 & lo]
    return np.stack(c, 1).astype(np.uint32)


def _draws(n, seed, sub, first=0):
    b = np.arange(first // 8, (first + n + 7) // 8, dtype=np.uint64)
    counter = np.stack([b & np.uint64(0xFFFFFFFF), b >> np.uint64(32), np.full_like(b, sub), np.zeros_like(b)], 1)
    return _philox(counter, seed % 2 ** 64).astype("<u4").view("<u2").reshape(-1)[:n]


def _keep(n, seed, sub, p):
    return torch.from_numpy(_draws(n, seed, sub) >= round(p * 65536))


def test_generator_known_answers():
    """The published vectors of Philox4x32-10: all zeros, all ones, digits of pi."""
    zero = _philox(np.zeros((1, 4), np.uint32), 0)[0]
    assert [hex(x) for x in zero] == ["0x6627e8d5", "0xe169c58d", "0xbc57ac4c", "0x9b00dbd8"]
    ones = _philox(np.full((1, 4), 0xFFFFFFFF, np.uint32), 2 ** 64 - 1)[0]
    assert [hex(x) for x in ones] == ["0x408f276d", "0x41c83b0e", "0xa20bc7c6", "0x6d5451fd"]
    pi = _philox(np.array([[0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344]], np.uint32), 0x299F31D0A4093822)[0]
    assert [hex(x) for x in pi] == ["0xd16cfe09", "0x94fdcceb", "0x5001e420", "0x24126ea1"]


def _seed(value):
    return torch.tensor([value], dtype=torch.int64, device="cuda")


TYPES = [(torch.float32, None), (torch.bfloat16, None), (torch.float32, torch.float32),
         (torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float32, torch.bfloat16)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,res", TYPES)
@pytest.mark.parametrize("n,p", [(1, 0.5), (7, 0.1), (8, 0.0), (9, 1.0), (1000, 0.9), (4097 * 33, 0.1)])
def test_matches_the_generator(n, p, dtype, res):
    from flash_hog_b200 import fused

    g = torch.Generator().manual_seed(n)
    x = torch.randn(n, generator=g).to(dtype)
    r = None if res is None else torch.randn(n, generator=g).to(res)
    xc = x.cuda().requires_grad_(True)
    rc = None if r is None else r.cuda().requires_grad_(True)
    seed = -0x123456789ABCDEF if n % 2 else 0x7FEDCBA987654321
    y = fused.dropout(xc, p, _seed(seed), subsequence=n, residual=rc)
    out = dtype if res is None else torch.promote_types(dtype, res)
    assert y.dtype == out
    limit = round(p * 65536)
    gate = _keep(n, seed, n, p).double() * (0.0 if limit == 65536 else 65536 / (65536 - limit))
    want = x.double() * gate + (0 if r is None else r.double())
    # The factor's rounding, and one of the fp32 result; then the type's.
    slack = 2 * F32 * (x.double() * gate).abs() + F32 * want.abs()
    half = torch.finfo(out).eps / 2
    assert ((y.detach().double().cpu() - want).abs() <= slack + half * (want.abs() + slack)).all()
    dy = torch.randn(n, generator=g).to(out)
    grads = torch.autograd.grad(y, [xc] + ([] if rc is None else [rc]), dy.cuda())
    assert grads[0].dtype == dtype
    want = dy.double() * gate
    half = torch.finfo(dtype).eps / 2
    assert ((grads[0].double().cpu() - want).abs() <= (3 * F32 + half * (1 + 3 * F32)) * want.abs()).all()
    assert (grads[0].cpu()[gate == 0] == 0).all()
    if rc is not None:
        assert torch.equal(grads[1].cpu(), dy.to(res))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_views_off_the_vector_alignment_and_strides(dtype):
    """The mask goes by an element's index in x, whatever x's address or strides."""
    from flash_hog_b200 import fused

    base = torch.randn(61 * 40 + 1, device="cuda").to(dtype)
    seed = _seed(5)
    want = fused.dropout(base[1:].clone().view(61, 40), 0.3, seed)
    assert torch.equal(fused.dropout(base[1:].view(61, 40), 0.3, seed), want)
    wide = torch.randn(61, 80, device="cuda").to(dtype)
    wide[:, ::2] = base[1:].view(61, 40)
    assert torch.equal(fused.dropout(wide[:, ::2], 0.3, seed), want)
    res = torch.randn(61 * 40 + 1, device="cuda").to(dtype)
    a = fused.dropout(base[1:].view(61, 40), 0.3, seed, residual=res[1:].view(61, 40))
    assert torch.equal(a, fused.dropout(base[1:].clone().view(61, 40), 0.3, seed, residual=res[1:].clone().view(61, 40)))


@pytest.mark.gpu
def test_seeds_and_subsequences_give_other_masks_at_the_right_rate():
    from flash_hog_b200 import fused

    x = torch.ones(1 << 20, device="cuda")
    masks = [fused.dropout(x, 0.1, _seed(s), subsequence=q) != 0 for s, q in ((1, 0), (2, 0), (1, 1), (1 + 2 ** 32, 0))]
    for i, a in enumerate(masks):
        # 2^20 draws at 0.9: a standard deviation of 2.9e-4; six of them.
        assert abs(a.float().mean().item() - 0.9) < 6 * 2.93e-4
        for b in masks[:i]:  # agreement of independent masks: 0.82 with a deviation of 3.8e-4
            assert abs((a == b).float().mean().item() - 0.82) < 6 * 3.8e-4


@pytest.mark.gpu
def test_double_backward_is_the_same_map():
    from flash_hog_b200 import fused

    x = torch.randn(50, 33, device="cuda", dtype=torch.bfloat16).requires_grad_(True)
    r = torch.randn(50, 33, device="cuda").requires_grad_(True)
    dy = torch.randn(50, 33, device="cuda").requires_grad_(True)
    seed = _seed(9)
    y = fused.dropout(x, 0.25, seed, residual=r)
    dx, dr = torch.autograd.grad(y, (x, r), dy, create_graph=True)
    u = torch.randn_like(dx).requires_grad_(True)
    (ddy,) = torch.autograd.grad((dx, dr), dy, (u, torch.zeros_like(dr)), create_graph=True)
    gate = _keep(50 * 33, 9, 0, 0.25).view(50, 33).cuda().double() / 0.75
    assert ((ddy.double() - u.double() * gate).abs() <= 3 * F32 * (u.double() * gate).abs()).all()
    (du,) = torch.autograd.grad(ddy, u, torch.ones_like(ddy))
    assert ((du.double() - gate).abs() <= (2.0 ** -8 + 3 * F32) * gate).all()


@pytest.mark.gpu
def test_empty_and_default_arguments():
    from flash_hog_b200 import fused

    x = torch.zeros((0, 4), device="cuda", requires_grad=True)
    y = fused.dropout(x, 0.5, _seed(0))
    assert y.shape == (0, 4) and torch.autograd.grad(y.sum(), x)[0].shape == (0, 4)


@pytest.mark.gpu
def test_captured_and_replayed_with_other_seeds():
    from flash_hog_b200 import fused

    x, seed = torch.randn(999, device="cuda"), _seed(1)
    dy = torch.randn(999, device="cuda")

    def step():
        v = x.detach().requires_grad_(True)
        y = fused.dropout(v, 0.4, seed, subsequence=2)
        return y, torch.autograd.grad(y, v, dy)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, dx = step()
    for s in (11, 12):
        seed.fill_(s)
        graph.replay()
        keep = _keep(999, s, 2, 0.4).cuda()
        assert torch.equal(y != 0, keep & (x != 0)) and torch.equal(dx != 0, keep & (dy != 0))


@pytest.mark.gpu
def test_a_seed_changed_before_the_backward_is_refused():
    from flash_hog_b200 import fused

    x, seed = torch.randn(64, device="cuda", requires_grad=True), _seed(1)
    y = fused.dropout(x, 0.5, seed)
    seed += 1
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()


@pytest.mark.gpu
def test_refusals_on_the_device():
    from flash_hog_b200 import fused

    x = torch.zeros(8, device="cuda")
    for seed in (torch.zeros(1, dtype=torch.long), torch.zeros(2, dtype=torch.long, device="cuda"),
                 torch.zeros(1, device="cuda")):
        with pytest.raises(ValueError):
            fused.dropout(x, 0.5, seed)


@pytest.mark.gpu
def test_library_errors_reach_the_caller_from_both_passes(monkeypatch):
    """A status from the library (injected on the host) is a FlashHogError with its name, in the
    forward and out of the engine's threads."""
    from flash_hog_b200 import fused
    from flash_hog_b200._capi import FlashHogError

    x = torch.randn(8, device="cuda", requires_grad=True)
    w = torch.randn(4, 4, device="cuda", requires_grad=True)
    t = torch.zeros(2, dtype=torch.long, device="cuda")
    monkeypatch.setenv("FLASH_HOG_B200_INJECT_ERROR", "fh_dropout,fh_embed_bwd")
    with pytest.raises(FlashHogError, match="FH_ERR_INJECTED") as e:
        fused.dropout(x, 0.5, _seed(1))
    assert e.value.entry == "fh_dropout" and e.value.status == 5
    y = fused.embedding(t, w)
    with pytest.raises(FlashHogError, match="fh_embed_bwd"):
        y.sum().backward()
    monkeypatch.delenv("FLASH_HOG_B200_INJECT_ERROR")
    y = fused.embedding(t, w)
    y.sum().backward()
    assert w.grad[0].tolist() == [2.0] * 4


@pytest.mark.gpu
def test_transforms_are_refused():
    from flash_hog_b200 import fused

    x, seed = torch.randn(3, 8, device="cuda"), _seed(1)
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.vmap(lambda v: fused.dropout(v, 0.5, seed))(x)
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.grad(lambda v: fused.dropout(v, 0.5, seed).sum())(x)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises((NotImplementedError, RuntimeError)):
            fused.dropout(dual, 0.5, seed)


def test_refusals():
    from flash_hog_b200 import fused

    x, seed = torch.zeros(8), torch.zeros(1, dtype=torch.long)
    with pytest.raises(ValueError):
        fused.dropout(x, 0.5, seed)  # CPU tensors
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError):
            fused.dropout(x, p, seed)
    for q in (-1, 2 ** 32):
        with pytest.raises(ValueError):
            fused.dropout(x, 0.5, seed, subsequence=q)
    with pytest.raises(ValueError):
        fused.dropout(x.half(), 0.5, seed)
    with pytest.raises(ValueError):
        fused.dropout(x, 0.5, seed, residual=torch.zeros(4))
    with pytest.raises(ValueError):
        fused.dropout(x, 0.5, seed, residual=x.half())


def test_c_abi_refusals():
    import ctypes

    from flash_hog_b200._capi import lib

    h, p = lib(), ctypes.c_void_p(64)
    call = lambda n=8, xt=0, rt=0, yt=0, res=None, x=p, limit=100: h.fh_dropout(None, n, xt, x, rt, res, yt, p, p, 0, limit)
    assert call(n=-1) == 1 and call(xt=2) == 1 and call(yt=3) == 1 and call(limit=65537) == 1 and call(limit=-1) == 1
    assert call(x=None) == 1
    assert call(res=p, rt=5) == 1
    assert call(res=p, xt=1, rt=0, yt=1) == 1  # a bf16 result of an fp32 residual
    assert call(n=0, x=None) == 0
