"""NaN and infinities in what attention reads: a visible NaN, or a score of +inf, makes the
rows that see it NaN (output and log-sum-exp), a score of -inf counts as 0, and a hidden
key's score does not count -- with every mask, whichever kernel it takes and wherever the key
lies."""

import pytest
import torch

from flash_hog_b200._attention_impl import MaskType, SlidingWindow, cuda_dot_product_attention

TQ, TK, B, H, HK = 200, 300, 1, 4, 2
BR = MaskType.CAUSAL_BOTTOM_RIGHT
MASKS = {
    "none": MaskType.NO_MASK,
    "causal": BR,
    "window": SlidingWindow(BR, 100),
    "sinks": SlidingWindow(BR, 100, 6),
    "sinks, nothing hidden": SlidingWindow(BR, 400, 6),
}


def _visible(mask, tq, tk):
    keep = torch.ones(tq, tk, dtype=torch.bool)
    if mask is MaskType.NO_MASK:
        return keep
    d, j = torch.arange(tq)[:, None] + tk - tq, torch.arange(tk)
    keep &= j <= d
    if isinstance(mask, SlidingWindow):
        keep &= (j > d - mask.length) | (j < mask.sinks)
    return keep


def _inputs(dtype, d, tq=TQ):
    g = torch.Generator().manual_seed(5)
    return [torch.randn(B, t, h, d, generator=g).to(dtype).cuda() for t, h in ((tq, H), (TK, HK), (TK, HK))]


def _run(q, k, v, mask):
    return cuda_dot_product_attention(q, k, v, mask_type=mask, scale=0.125, return_residual=True)


def _check(got, want, hit, dtype):
    """NaN in the rows `hit` of heads 2 and 3 (key head 1) and nowhere else; the others as they were."""
    (o, lse), (o0, lse0) = got, want
    hit = hit.cuda()
    assert o[0, hit, 2:].isnan().all() and lse[0, 2:, hit].isnan().all()
    # When a warp rescales may change with a row of it: half a step of the result on each side.
    eps = torch.finfo(dtype).eps
    near = dict(rtol=2 * eps, atol=2 * eps * o0.abs().max().item())
    torch.testing.assert_close(o[0, ~hit, 2:], o0[0, ~hit, 2:], **near)
    torch.testing.assert_close(o[0, :, :2], o0[0, :, :2], **near)
    for a, b in ((lse[0, 2:, ~hit], lse0[0, 2:, ~hit]), (lse[0, :2], lse0[0, :2])):
        torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-5)


# Key positions in both kinds of columns that the exponentials are split into (0 to 3 of 16 and
# the others), in the first, a middle and the last tile.
@pytest.mark.gpu
@pytest.mark.parametrize("key", [3, 5, 130, 299])
@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float32, 64)])
def test_a_visible_nan_key_reaches_output_and_lse(dtype, d, mask, key):
    q, k, v = _inputs(dtype, d)
    mask = MASKS[mask]
    want = _run(q, k, v, mask)
    k[0, key, 1, 7] = float("nan")
    _check(_run(q, k, v, mask), want, _visible(mask, TQ, TK)[:, key], dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("key", [5, 259])
@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float32, 64)])
def test_infinite_scores(dtype, d, mask, key):
    q, k, v = _inputs(dtype, d)
    mask = MASKS[mask]
    k[0, key, 1] = 0
    q[..., 7] = 1
    want = _run(q, k, v, mask)
    k[0, key, 1, 7] = float("inf")
    _check(_run(q, k, v, mask), want, _visible(mask, TQ, TK)[:, key], dtype)
    # -inf: as a score far below all others. (1e30 / 8 in the exponent gives 0 exactly.)
    k[0, key, 1, 7] = -1e30
    want = _run(q, k, v, mask)
    k[0, key, 1, 7] = -float("inf")
    got = _run(q, k, v, mask)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("tq", [1, 5])
@pytest.mark.parametrize("mask", MASKS)
def test_few_query_rows(mask, tq):
    q, k, v = _inputs(torch.bfloat16, 64, tq)
    mask = MASKS[mask]
    for key in (2, 9, 260, 299):
        for value in ("nan", "inf"):
            bad = k.clone()
            bad[0, key, 1] = 0
            bad[0, key, 1, 7] = float(value)
            _check(_run(q.abs(), bad, v, mask), _run(q.abs(), torch.where(bad.isfinite(), bad, 0), v, mask),
                   _visible(mask, tq, TK)[:, key], torch.bfloat16)


@pytest.mark.gpu
def test_a_nan_query_reaches_its_row_alone():
    q, k, v = _inputs(torch.bfloat16, 128)
    for mask in MASKS.values():
        want = _run(q, k, v, mask)
        bad = q.clone()
        bad[0, 77, 2:] = float("nan")
        _check(_run(bad, k, v, mask), want, torch.arange(TQ) == 77, torch.bfloat16)
