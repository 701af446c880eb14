"""The clipped policy loss with a KL term: forward, backward and the backward's backward.

The statement is the definition in float64, differentiated twice by autograd. Bounds: an
exponential's argument (z - m) log2e is below 32 in size here and rounds three times, by
3 * 32 * 2^-24 * ln 2, the exponential itself by 2^-22: below 4.2e-6 relative; the sum of exponentials likewise, so a
softmax entry is off by at most REL = 8e-6 relative with its products, and a log
probability by 8e-6. Outputs then round to their type.
"""

import math

import pytest
import torch

REL = 8e-6


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _inputs(rows, vocab, dtype, seed, kl=True, masked=0.3, ld=None, offset=0):
    g = torch.Generator().manual_seed(seed)
    ld = vocab if ld is None else ld
    store = (torch.randn(rows * ld + offset, generator=g) * 2.5).to(dtype).cuda()
    z = store[offset:].view(rows, ld)[:, :vocab]
    a = torch.randint(0, vocab, (rows,), generator=g).cuda()
    lp = torch.log_softmax(z.double(), 1).gather(1, a[:, None])[:, 0]
    # Log ratios on both sides of the clip borders (at -0.223 and 0.182), none within 0.05 of one.
    ratio = torch.tensor([-0.6, -0.3, -0.1, 0.05, 0.1, 0.3, 0.7])[torch.randint(0, 7, (rows,), generator=g)].cuda()
    old = (lp - ratio).float()
    adv = torch.randn(rows, generator=g).cuda()
    ref = (lp + torch.randn(rows, generator=g).cuda() * 0.5).float() if kl else None
    w = (torch.rand(rows, generator=g) >= masked).float().cuda() if masked else None
    if w is not None:
        w[0] = 0.5
    return z, a, old, adv, ref, w


def _statement(z, a, old, adv, ref, w, lo=0.2, hi=0.2, beta=0.0, norm=None):
    """(loss, lp, row coefficients dl/dlp w / N) in float64; z may require grad."""
    lp = torch.log_softmax(z, 1).gather(1, a[:, None])[:, 0]
    w = torch.ones_like(lp) if w is None else w.double()
    used = w != 0
    lp = torch.where(used, lp, torch.zeros_like(lp))
    rho = torch.exp(lp - old.double())
    adv = adv.double()
    clipped = ((adv > 0) & (rho > 1 + hi)) | ((adv < 0) & (rho < 1 - lo))
    row = -torch.where(clipped, rho.detach().clamp(1 - lo, 1 + hi), rho) * adv
    if beta:
        d = ref.double() - lp
        row = row + beta * (torch.exp(d) - d - 1)
    n = w.sum() if norm is None else norm
    return (torch.where(used, row, torch.zeros_like(row)) * w).sum() / n, lp


CASES = [  # rows, vocab, ld, offset
    (1, 1, 1, 0), (1, 2, 2, 0), (3, 7, 9, 1), (5, 1000, 1000, 0), (4, 1001, 1001, 0), (6, 1003, 1008, 3),
    (33, 4097, 4097, 0), (2, 131075, 131075, 0), (40, 16391, 16400, 1), (130, 8192, 8192, 0), (300, 513, 520, 0), (1, 40000, 40000, 5),
    # Enough rows for a block each; rows of z and dz that reach 16 bytes at different columns.
    (600, 2500, 2500, 0), (601, 8193, 8193, 0), (593, 16385, 16392, 8), (592, 32801, 32801, 3), (594, 9000, 9001, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("beta", [0.0, 0.1])
@pytest.mark.parametrize("rows,vocab,ld,offset", CASES)
def test_all_passes(rows, vocab, ld, offset, beta, dtype):
    from flash_hog_b200 import fused

    z, a, old, adv, ref, w = _inputs(rows, vocab, dtype, rows + vocab, masked=0.3 if rows > 2 else 0.0, ld=ld,
                                     offset=offset)
    zg = z.requires_grad_(True)
    loss, lp = fused.policy_loss(zg, a, old, adv, ref_logprobs=ref, weights=w, kl_coef=beta)
    assert loss.dtype == torch.float32 and loss.shape == () and lp.dtype == torch.float32
    zd = z.detach().double().requires_grad_(True)
    want, want_lp = _statement(zd, a, old, adv, ref, w, beta=beta)
    scale = (adv.double().abs() * 2.1 + beta).max()  # of |dl/dlp| and |l| (ratios below e^0.7, KL terms below)
    scale = scale + beta * torch.exp((ref.double() - want_lp).max())
    assert ((lp.double() - want_lp).abs() <= 2 * REL + 2.0 ** -23 * want_lp.abs()).all()
    assert abs(loss.item() - want.item()) <= 4 * REL * scale + 2.0 ** -23 * abs(want.item())
    g = torch.tensor(1.5, device="cuda", requires_grad=True)
    (dz,) = torch.autograd.grad(loss, zg, g, create_graph=True)
    gd = torch.tensor(1.5, dtype=torch.float64, device="cuda", requires_grad=True)
    (dzd,) = torch.autograd.grad(want, zd, gd, create_graph=True)
    assert dz.dtype == dtype
    # |dz| <= k (p + e): the softmax's error, the coefficient's (as lp's) and the roundings.
    wn = torch.ones(rows, device="cuda") if w is None else w
    k = (1.5 * scale * wn.double() / wn.double().sum())[:, None]
    p = torch.softmax(zd.detach(), 1)
    e = torch.zeros_like(p).scatter_(1, a[:, None], 1.0)
    err = (dz.detach().double() - dzd.detach()).abs()
    assert (err <= 4 * REL * k * (p + e) + _half(dtype) * dzd.detach().abs() + 1e-37).all()
    if w is not None:
        assert (dz.detach()[w == 0] == 0).all()
    u = torch.randn(rows, vocab, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    gz, gg = torch.autograd.grad(dz, (zg, g), u)
    gzd, ggd = torch.autograd.grad(dzd, (zd, gd), u.double())
    umax = u.double().abs().max()
    # Every term of gz is at most k (p + e) times |u| (twice: u and its mean; c' likewise).
    err = (gz.double() - gzd).abs()
    assert (err <= 24 * REL * umax * k * (p + e) + _half(dtype) * gzd.abs() + 1e-37).all()
    assert abs(gg.item() - ggd.item()) <= 12 * REL * umax * k.sum() / 1.5


@pytest.mark.gpu
def test_gradient_against_differences():
    from flash_hog_b200 import fused

    z, a, old, adv, ref, w = _inputs(6, 50, torch.float32, 3)
    kw = dict(ref_logprobs=ref, weights=w, kl_coef=0.1, normalizer=3.0)
    zg = z.requires_grad_(True)
    (dz,) = torch.autograd.grad(fused.policy_loss(zg, a, old, adv, **kw)[0], zg)
    d = torch.randn_like(z)
    h = 2.0 ** -8
    up = fused.policy_loss(z.detach() + h * d, a, old, adv, **kw)[0].double()
    down = fused.policy_loss(z.detach() - h * d, a, old, adv, **kw)[0].double()
    slope = (dz.double() * d).sum()
    # Third derivatives along d are below 30 |d|^3-ish here: h^2 * 30 / 6 = 8e-5; the losses' rounding 2^-23 / h = 3e-5.
    assert abs((up - down).item() / (2 * h) - slope.item()) <= 5e-3 * max(1.0, abs(slope.item()))


@pytest.mark.gpu
@pytest.mark.parametrize("hi", [0.2, float("inf")])
def test_clip_sides_and_default_weights(hi):
    """Ratios beyond each border with each sign of the advantage: which side carries a gradient."""
    from flash_hog_b200 import fused

    z = torch.randn(4, 10, device="cuda")
    a = torch.tensor([1, 2, 3, 4], device="cuda")
    lp = torch.log_softmax(z.double(), 1).gather(1, a[:, None])[:, 0]
    old = (lp - torch.tensor([0.5, 0.5, -0.5, -0.5], device="cuda")).float()
    adv = torch.tensor([1.0, -1.0, 1.0, -1.0], device="cuda")
    zg = z.requires_grad_(True)
    loss, _ = fused.policy_loss(zg, a, old, adv, clip_low=0.2, clip_high=hi)
    (dz,) = torch.autograd.grad(loss, zg)
    active = (dz != 0).any(1).tolist()
    assert active == [math.isinf(hi), True, True, False]
    up, down = math.exp(0.5), math.exp(-0.5)
    want = [-min(up, 1 + hi), up, -down, 0.8]
    assert abs(loss.item() - sum(want) / 4) <= 1e-5


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masked_rows_are_not_read(dtype):
    from flash_hog_b200 import fused

    z, a, old, adv, ref, _ = _inputs(8, 200, dtype, 5)
    keep = torch.tensor([1, 0, 1, 1, 0, 1, 0, 1], dtype=torch.bool, device="cuda")
    bad = z.clone()
    bad[~keep] = float("nan")
    bad[1] = float("inf")
    for t in (old, adv, ref):
        t[~keep] = float("nan")
    a2 = torch.where(keep, a, torch.full_like(a, -100))
    out = []
    for logits, acts, weights in ((z[keep], a[keep], None), (bad, a2, keep)):
        v = logits.detach().clone().requires_grad_(True)
        sel = keep if weights is not None else slice(None)
        take = (lambda t: t) if weights is not None else (lambda t: t[keep])
        loss, lp = fused.policy_loss(v, acts, take(old), take(adv), ref_logprobs=take(ref), weights=weights, kl_coef=0.1)
        g = torch.tensor(1.0, device="cuda", requires_grad=True)
        (dz,) = torch.autograd.grad(loss, v, g, create_graph=True)
        u = torch.ones_like(dz).cumsum(1)
        gz, gg = torch.autograd.grad(dz, (v, g), u)
        out.append((loss, lp[sel], dz[sel], gz[sel], gg))
        if weights is not None:
            assert (lp[~keep] == 0).all() and (dz[~keep] == 0).all() and (gz[~keep] == 0).all()
    for x, y in zip(out[0][:-1], out[1][:-1]):
        assert torch.equal(x, y)
    # gg adds 5 and 8 row terms in fp32, in another order: at most 7 roundings of 2^-24 each
    # on partial sums below sum |gg_r| <= sum w/N |c| 2 max|u| <= 4 * 400.
    assert abs(out[0][-1].item() - out[1][-1].item()) <= 14 * 2.0 ** -24 * 1600


@pytest.mark.gpu
def test_no_weight_no_rows_and_lowest_logits():
    from flash_hog_b200 import fused

    z = torch.randn(3, 20, device="cuda", requires_grad=True)
    a, v = torch.zeros(3, dtype=torch.long, device="cuda"), torch.zeros(3, device="cuda")
    loss, lp = fused.policy_loss(z, a, v, v + 1, weights=v)
    assert loss.item() == 0 and (lp == 0).all()
    assert (torch.autograd.grad(loss, z)[0] == 0).all()
    e = torch.zeros((0, 20), device="cuda", requires_grad=True)
    loss, lp = fused.policy_loss(e, a[:0], v[:0], v[:0])
    assert loss.item() == 0 and lp.shape == (0,) and torch.autograd.grad(loss, e)[0].shape == (0, 20)
    # Excluded vocabulary entries: -inf and the type's lowest value have probability 0.
    for dtype in (torch.float32, torch.bfloat16):
        for low in (-math.inf, torch.finfo(dtype).min):
            zz = torch.randn(2, 600, device="cuda").to(dtype)
            zz[:, 100:] = low
            zz.requires_grad_(True)
            aa = torch.tensor([3, 99], device="cuda")
            loss, lp = fused.policy_loss(zz, aa, torch.full((2,), -4.0, device="cuda"), torch.ones(2, device="cuda"),
                                         clip_high=float("inf"))
            want = torch.log_softmax(zz.detach()[:, :100].double(), 1).gather(1, aa[:, None])[:, 0]
            assert ((lp.double() - want).abs() <= 2 * REL + 2.0 ** -23 * want.abs()).all()
            (dz,) = torch.autograd.grad(loss, zz)
            assert (dz[:, 100:] == 0).all() and dz.isfinite().all()
            # A row of nothing but the lowest value is uniform, one of -inf undefined.
            zz = torch.full((2, 64), low, dtype=dtype, device="cuda")
            _, lp = fused.policy_loss(zz, aa[:1].expand(2), torch.zeros(2, device="cuda"), torch.ones(2, device="cuda"))
            if math.isinf(low):
                assert lp.isnan().all()
            else:
                assert ((lp + math.log(64)).abs() <= 2 * REL).all()


@pytest.mark.gpu
def test_bad_logits_and_actions_show():
    from flash_hog_b200 import fused

    for spoil in ("nan", "inf", "low_action", "high_action"):
        z = torch.randn(3, 300, device="cuda")
        a = torch.tensor([1, 2, 3], device="cuda")
        if spoil in ("nan", "inf"):
            z[1, 250] = float(spoil)
        else:
            a[1] = -1 if spoil == "low_action" else 300
        z.requires_grad_(True)
        loss, lp = fused.policy_loss(z, a, torch.full((3,), -5.0, device="cuda"), torch.ones(3, device="cuda"))
        assert loss.isnan() and lp[1].isnan() and not lp[[0, 2]].isnan().any()
        (dz,) = torch.autograd.grad(loss, z)
        assert dz[1].isnan().all() and not dz[[0, 2]].isnan().any()


@pytest.mark.gpu
def test_captured_and_replayed():
    from flash_hog_b200 import fused

    z, a, old, adv, ref, w = _inputs(40, 1000, torch.bfloat16, 7)
    z = z.clone()

    def step():
        v = z.detach().requires_grad_(True)
        loss, lp = fused.policy_loss(v, a, old, adv, ref_logprobs=ref, weights=w, kl_coef=0.1)
        return loss, lp, torch.autograd.grad(loss, v)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (8, 9):
        new = _inputs(40, 1000, torch.bfloat16, seed)
        for x, y in zip((z, a, old, adv, ref, w), new):
            x.copy_(y)
        graph.replay()
        got = [t.clone() for t in captured]
        for x, y in zip(got, step()):
            assert torch.equal(x, y)


def test_refusals():
    from flash_hog_b200 import fused

    z, a, v = torch.zeros(2, 5), torch.zeros(2, dtype=torch.long), torch.zeros(2)
    with pytest.raises(ValueError):
        fused.policy_loss(z, a, v, v)  # CPU tensors
    with pytest.raises(ValueError):
        fused.policy_loss(z[0], a, v, v)
    with pytest.raises(ValueError):
        fused.policy_loss(z.half(), a, v, v)
    with pytest.raises(ValueError):
        fused.policy_loss(z[:, :0], a, v, v)
    for kw in (dict(clip_low=-0.1), dict(clip_high=float("nan")), dict(kl_coef=0.1), dict(kl_coef=-1.0),
               dict(normalizer=0.0), dict(normalizer=1e-40), dict(normalizer=float("inf"))):
        with pytest.raises(ValueError):
            fused.policy_loss(z, a, v, v, **kw)


@pytest.mark.gpu
def test_refusals_on_the_device():
    from flash_hog_b200 import fused

    z, a, v = torch.zeros(2, 5, device="cuda"), torch.zeros(2, dtype=torch.long, device="cuda"), torch.zeros(2, device="cuda")
    for args in ((z, a[:1], v, v), (z, a, v[:1], v), (z, a, v, v.cpu()), (z, a, v, v.expand(3, 2))):
        with pytest.raises(ValueError):
            fused.policy_loss(*args)
    with pytest.raises(ValueError):
        fused.policy_loss(z, a, v, v, weights=torch.ones(3, device="cuda"))


@pytest.mark.gpu
def test_third_order_is_refused():
    from flash_hog_b200 import fused

    z, a, old, adv, _, _ = _inputs(3, 20, torch.float32, 1, kl=False, masked=0.0)
    z.requires_grad_(True)
    loss, _ = fused.policy_loss(z, a, old, adv)
    (dz,) = torch.autograd.grad(loss, z, create_graph=True)
    with pytest.raises(NotImplementedError):
        torch.autograd.grad(dz.square().sum(), z, create_graph=True)


def test_c_abi_refusals():
    import ctypes

    from flash_hog_b200._capi import lib

    h, p = lib(), ctypes.c_void_p(64)
    fwd = lambda dt=0, rows=1, vocab=4, ld=4, old=p, ref=p, lo=0.2, kl=0.1, norm=0.0: h.fh_policy_fwd(
        None, dt, rows, vocab, ld, p, p, old, p, ref, None, lo, 0.2, kl, norm, p, p, p)
    assert fwd(dt=2) == 1 and fwd(rows=-1) == 1 and fwd(vocab=0) == 1 and fwd(ld=3) == 1
    assert fwd(old=None) == 1 and fwd(ref=None) == 1 and fwd(lo=-1.0) == 1 and fwd(norm=-1.0) == 1
    assert h.fh_policy_bwd(None, 0, 1, 4, 4, p, p, None, p, p) == 1
    assert h.fh_policy_bwd(None, 0, 0, 4, 4, p, p, p, p, p) == 0
    assert h.fh_policy_bwd_bwd(None, 0, 1, 4, 4, p, p, p, p, None, p, p, None) == 1
    assert h.fh_policy_bwd(None, 0, 1, 4, 4, p, p, ctypes.c_void_p(72), p, p) == 1  # stats not aligned
    assert h.fh_policy_stats_floats(-1, 4) == -1 and h.fh_policy_scratch_floats(1, 0) == -1
    assert fwd(rows=2 ** 31 - 1024) == 1 and fwd(vocab=2 ** 31 - 1024, ld=2 ** 31) == 1
    assert h.fh_policy_stats_floats(2 ** 31 - 1, 1) == -1 and h.fh_policy_stats_floats(2 ** 31 - 1025, 1) > 2 ** 33
    assert h.fh_policy_scratch_floats(1, 100) == 0 and h.fh_policy_scratch_floats(1, 1 << 20) > 0
    assert h.fh_policy_bwd_bwd(None, 0, 1, 1 << 20, 1 << 20, p, p, p, p, p, p, p, None) == 1  # needs scratch


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [10, 1000, 32000, 131075])
def test_the_side_of_a_clip_border(vocab, dtype):
    """Ratios close to the borders fall on the side that they have, down to the bound on the log
    probability (2 * REL and its rounding), and the others' rows carry their whole gradient."""
    from flash_hog_b200 import fused

    steps = [s * d for d in (2e-5, 4e-5, 1e-4, 1e-3) for s in (-1, 1)]
    rows = 4 * len(steps)
    g = torch.Generator().manual_seed(vocab)
    z = (torch.randn(rows, vocab, generator=g) * 2.5).to(dtype).cuda()
    a = torch.randint(0, vocab, (rows,), generator=g).cuda()
    lp = torch.log_softmax(z.double(), 1).gather(1, a[:, None])[:, 0]
    lo, hi = 0.2, 0.25
    low, high = (1 + s * torch.tensor(c, dtype=torch.float32).double().item() for s, c in ((-1, lo), (1, hi)))
    border = torch.tensor([math.log(high), math.log(low)] * 2, dtype=torch.float64).repeat_interleave(len(steps)).cuda()
    adv = torch.tensor([1.0, 1.0, -1.0, -1.0]).repeat_interleave(len(steps)).cuda()
    old = (lp - border - torch.tensor(steps * 4, dtype=torch.float64, device="cuda")).float()
    distance = lp - old.double() - border  # after the rounding of old
    assert (distance.abs() > 2 * REL + 2.0 ** -23 * lp.abs()).all()
    rho = torch.exp(lp - old.double())
    clipped = ((adv > 0) & (rho > high)) | ((adv < 0) & (rho < low))
    assert 0 < clipped.sum() < rows
    z.requires_grad_(True)
    loss, _ = fused.policy_loss(z, a, old, adv, clip_low=lo, clip_high=hi)
    (dz,) = torch.autograd.grad(loss, z)
    assert torch.equal((dz == 0).all(1), clipped)
