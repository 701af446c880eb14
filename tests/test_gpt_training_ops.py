"""The GPT with its embeddings, windows with sinks, dropout and policy loss together, as a
training run uses them: against the same model in torch math, differentiated twice where the
penalty asks for it, eager and replayed as a CUDA graph."""

import pytest
import torch
import torch.nn.functional as F

from flash_hog_b200.gpt import (GPT, GPTConfig, PenaltyStepGraph, naive_attention, penalty_objective,
                                policy_objective, policy_step, train_step)

# Tolerances: both models compute in fp32; a chain of some 40 products and sums of up to 515
# terms, each off by at most 515 * 2^-24 of its size and mostly by its root, stays below 1e-3
# (twice that through the exponentials of the policy loss).
CFG = dict(n_layer=2, d_model=128, n_head=2, d_mlp=256, vocab=515, seq_len=160, window=48, sinks=3, embed_scale=3.0)


def _tokens(cfg, batch, seed, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, cfg.vocab, (batch, cfg.seq_len + 1), generator=g).to(device)


def _pair(**kw):
    torch.manual_seed(0)
    cfg = GPTConfig(**{**CFG, **kw})
    ref = GPT(cfg, attention="naive").cuda()
    ours = GPT(cfg, attention="flash").cuda()
    ours.load_state_dict(ref.state_dict())
    return cfg, ref, ours


def test_naive_attention_has_the_window():
    torch.manual_seed(1)
    q, k, v = (torch.randn(1, 30, 2, 16) for _ in range(3))
    got = naive_attention(q, k, v, sliding_window_length=5, sink_tokens=2)
    for i in (0, 4, 7, 29):
        seen = [j for j in range(i + 1) if i - j < 5 or j < 2]
        s = torch.einsum("hd,khd->hk", q[0, i], k[0, seen]) * 0.25
        want = torch.einsum("hk,khd->hd", s.softmax(-1), v[0, seen])
        torch.testing.assert_close(got[0, i], want, rtol=1e-5, atol=1e-5)


def test_sinks_need_a_window():
    with pytest.raises(ValueError):
        GPT(GPTConfig(n_layer=1, d_model=64, n_head=1, d_mlp=64, vocab=50, seq_len=16, sinks=2))


def _close(got, want, tol):
    """Relative distance of two lists of gradients, as a whole and each by itself (looser)."""
    num = sum(((a.double() - b.double()) ** 2).sum() for a, b in zip(got, want)).sqrt()
    den = sum((b.double() ** 2).sum() for b in want).sqrt()
    assert (num / den).item() <= tol
    for a, b in zip(got, want):
        assert ((a.double() - b.double()).norm() / b.double().norm().clamp_min(1e-12)).item() <= 5 * tol


@pytest.mark.gpu
def test_penalty_step_with_window_sinks_and_scaled_embeddings():
    """fp32 throughout: loss, penalty and the gradients of L + lam ||dL/dtheta||^2."""
    cfg, ref, ours = _pair()
    tokens = _tokens(cfg, 2, 1)
    out = []
    for model in (ref, ours):
        loss, pen = train_step(model, tokens, 0.5, autocast=False)
        out.append((loss.item(), pen.item(), [p.grad for p in model.parameters()]))
    (l0, p0, g0), (l1, p1, g1) = out
    assert abs(l1 - l0) <= 1e-4 * abs(l0) and abs(p1 - p0) <= 1e-3 * abs(p0)
    _close(g1, g0, 1e-3)


def test_old_configurations_have_the_same_parameters():
    plain = GPT(GPTConfig(n_layer=1, d_model=64, n_head=1, d_mlp=64, vocab=50, seq_len=16))
    assert sorted(plain.state_dict()) == sorted(GPT(GPTConfig(n_layer=1, d_model=64, n_head=1, d_mlp=64, vocab=50,
                                                              seq_len=16, dropout=0.1), attention="naive").state_dict())


@pytest.mark.gpu
def test_dropout_follows_its_seed():
    cfg, _, model = _pair(dropout=0.2)
    tokens = _tokens(cfg, 2, 2)

    def step(seed):
        model.dropout_seed.fill_(seed)
        model.zero_grad(set_to_none=True)
        total, loss, penalty = penalty_objective(model, tokens, 0.1)
        total.backward()
        assert model.dropout_seed.item() == seed + 1
        return loss.item(), penalty.item(), [p.grad.clone() for p in model.parameters()]

    a, b, c = step(5), step(5), step(6)
    assert a[:2] == b[:2] and all(torch.equal(x, y) for x, y in zip(a[2], b[2]))
    assert a[0] != c[0]
    model.eval()
    with torch.no_grad():
        x = model(tokens[:, :-1])
        assert torch.equal(x, model(tokens[:, :-1])) and model.dropout_seed.item() == 7


@pytest.mark.gpu
def test_gradient_with_dropout_against_differences():
    """The masks are those of the forward: the gradient along a direction is the slope of the loss
    with the same seed."""
    cfg, _, model = _pair(dropout=0.3)
    tokens = _tokens(cfg, 1, 3)
    params = list(model.parameters())
    torch.manual_seed(1)
    d = [torch.randn_like(p) * 0.02 for p in params]

    def loss():
        model.dropout_seed.fill_(11)
        return F.cross_entropy(model(tokens[:, :-1]).flatten(0, 1), tokens[:, 1:].flatten())

    slope = sum((g.double() * v).sum() for g, v in zip(torch.autograd.grad(loss(), params), d)).item()
    h = 2.0 ** -5
    with torch.no_grad():
        ends = []
        for s in (h, -h):
            for p, v in zip(params, d):
                p.add_(v, alpha=s)
            ends.append(loss().double().item())
            for p, v in zip(params, d):
                p.add_(v, alpha=-s)
    # The losses are near 6 and round by 6 * 2^-23: 2e-5 of the slope at this step; the third
    # derivative's term is h^2 / 6 = 1.6e-4 of a slope of its own size.
    assert abs((ends[0] - ends[1]) / (2 * h) - slope) <= 2e-2 * max(abs(slope), 0.05)


@pytest.mark.gpu
def test_captured_step_draws_new_masks_and_matches_eager():
    cfg, _, model = _pair(dropout=0.2)
    tokens = [_tokens(cfg, 2, s) for s in (4, 5)]
    graph = PenaltyStepGraph(model, 2, 0.1, autocast=False)
    got = []
    for t, seed in ((tokens[0], 100), (tokens[1], 101), (tokens[0], 100)):
        if seed == 100:
            model.dropout_seed.fill_(100)
        loss, pen = graph.step(t)
        got.append((loss.item(), pen.item(), [p.grad.clone() for p in model.parameters()]))
        assert model.dropout_seed.item() == seed + 1
    assert got[0][:2] == got[2][:2] and got[0][0] != got[1][0]
    del graph
    for (want_loss, want_pen, want), t, seed in zip(got[:2], tokens, (100, 101)):
        model.dropout_seed.fill_(seed)
        model.zero_grad(set_to_none=True)
        loss, pen = train_step(model, t, 0.1, autocast=False)
        assert abs(loss.item() - want_loss) <= 1e-5 * want_loss and abs(pen.item() - want_pen) <= 1e-3 * want_pen
        _close([p.grad for p in model.parameters()], want, 1e-3)


@pytest.mark.gpu
@pytest.mark.parametrize("lam", [0.0, 0.3])
def test_policy_objective_against_torch(lam):
    """Sampled continuations of two prompts, one padded: the loss, the log probabilities and the
    gradients (with lam, of the penalty too) against log_softmax in torch."""
    cfg, ref, ours = _pair()
    tokens = _tokens(cfg, 2, 6)
    g = torch.Generator().manual_seed(7)
    weights = torch.zeros(2, cfg.seq_len)
    weights[0, 30:], weights[1, 40:120] = 1, 1
    adv = torch.randn(2, cfg.seq_len, generator=g)
    with torch.no_grad():
        lp = F.log_softmax(ref(tokens[:, :-1]), -1).gather(2, tokens[:, 1:, None])[..., 0].cpu()
    # Ratios of 0.61 to 1.65: on both sides of the borders 0.8 and 1.25, none within 0.05 of one.
    old = lp - torch.tensor([-0.5, -0.1, 0.1, 0.5])[torch.randint(0, 4, lp.shape, generator=g)]
    refp = lp + 0.3 * torch.randn(lp.shape, generator=g)
    weights, adv, old, refp = (t.cuda() for t in (weights, adv, old, refp))

    logits = ref(tokens[:, :-1])
    l = F.log_softmax(logits, -1).gather(2, tokens[:, 1:, None])[..., 0]
    rho = torch.exp(l - old)
    d = refp - l
    rows = -torch.minimum(rho * adv, rho.clamp(0.8, 1.25) * adv) + 0.05 * (torch.exp(d) - d - 1)
    want = (rows * weights).sum() / weights.sum()
    total = want
    if lam:
        grads = torch.autograd.grad(want, list(ref.parameters()), create_graph=True)
        total = want + lam * sum((x ** 2).sum() for x in grads)
    total.backward()
    got_total, got, got_lp = policy_objective(ours, tokens, old, adv, lam, weights=weights, ref_logprobs=refp,
                                              kl_coef=0.05, clip_high=0.25)
    got_total.backward()
    assert abs(got.item() - want.item()) <= 1e-4 * max(abs(want.item()), 0.1)
    assert (got_lp - l.detach() * (weights > 0)).abs().max() <= 1e-3
    _close([p.grad for p in ours.parameters()], [p.grad for p in ref.parameters()], 2e-3)


@pytest.mark.gpu
def test_policy_steps_under_autocast_run():
    """Everything together in bf16 autocast, two steps of an optimizer: finite, and the second
    step's ratios start where the first's log probabilities were."""
    cfg, _, model = _pair(dropout=0.1)
    tokens = _tokens(cfg, 2, 8)
    opt = torch.optim.SGD(model.parameters(), lr=1e-3)
    zeros = torch.zeros(2, cfg.seq_len, device="cuda")
    model.dropout_seed.fill_(3)
    _, lp = policy_step(model, tokens, zeros, zeros, autocast=True)
    adv = torch.randn(2, cfg.seq_len, device="cuda")
    for _ in range(2):
        loss, new = policy_step(model, tokens, lp, adv, lam=0.05, optimizer=opt, weights=torch.ones_like(adv),
                                ref_logprobs=lp, kl_coef=0.1)
        assert loss.isfinite() and new.isfinite().all()
    assert all(p.isfinite().all() for p in model.parameters())


@pytest.mark.parametrize("attention", ["naive", "flash"])
def test_more_tokens_than_positions_are_refused(attention):
    model = GPT(GPTConfig(n_layer=1, d_model=64, n_head=1, d_mlp=64, vocab=50, seq_len=16), attention=attention)
    with pytest.raises(IndexError):
        model(torch.zeros(1, 17, dtype=torch.long))
