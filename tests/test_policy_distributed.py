"""Data-parallel policy steps (two gloo ranks on CPU, the policy loss in torch): the averaged
gradient is that of the weighted mean over all ranks' rows, however the weights are spread."""

import datetime
import os
import socket
import sys

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
WORLD = 2


def _policy_loss(logits, actions, old, adv, *, ref_logprobs=None, weights=None, clip_low=0.2, clip_high=0.2,
                 kl_coef=0.0, normalizer=None):
    lp = torch.log_softmax(logits, -1).gather(1, actions[:, None])[:, 0]
    rho = torch.exp(lp - old)
    rows = -torch.minimum(rho * adv, rho.clamp(1 - clip_low, 1 + clip_high) * adv)
    w = torch.ones_like(adv) if weights is None else weights.to(adv.dtype)
    n = w.sum() if normalizer is None else torch.tensor(normalizer)
    return (w * rows).sum() / n if n != 0 else (0 * rows).sum(), lp.detach() * (w != 0)


def _rank_inputs(rank, weighting):
    g = torch.Generator().manual_seed(10 + rank)
    b, t = (2, 1)[rank] if weighting == "none" else 2, 12
    x = dict(tokens=torch.randint(0, 40, (b, t + 1), generator=g), old_logprobs=torch.full((b, t), -3.7),
             advantages=torch.randn(b, t, generator=g))
    if weighting == "ragged":
        x["weights"] = (torch.rand(b, t, generator=g) < (0.9, 0.15)[rank]).float()
        x["weights"][0, 0] = 0.5
    elif weighting == "mask":
        x["weights"] = torch.rand(b, t, generator=g) < (0.8, 0.2)[rank]
    elif weighting == "one empty":
        x["weights"] = torch.full((b, t), float(rank == 0))
    elif weighting == "all empty":
        x["weights"] = torch.zeros(b, t)
    elif weighting == "normalizer":
        x["normalizer"] = 7.0
    return x


CASES = [(w, 0.0) for w in ("ragged", "mask", "one empty", "all empty", "none", "normalizer")] + [("ragged", 0.3)]


def _step(rank, weighting, lam):
    from flash_hog_b200.gpt import GPT, GPTConfig, policy_objective, policy_step

    torch.manual_seed(0)
    model = GPT(GPTConfig(n_layer=1, d_model=32, n_head=2, d_mlp=32, vocab=40, seq_len=12), attention="naive")
    loss, _ = policy_step(model, **_rank_inputs(rank, weighting), lam=lam, distributed=True)
    mean_loss = loss.clone()
    dist.all_reduce(mean_loss)
    got = [p.grad.clone() for p in model.parameters()]
    all_in = [_rank_inputs(r, weighting) for r in range(WORLD)]
    model.zero_grad()
    if lam:  # each rank's objective on its share of the loss, averaged
        n = sum(x["weights"].sum().item() for x in all_in) / WORLD
        want_loss = 0.0
        for x in all_in:
            total, part, _ = policy_objective(model, **x, normalizer=n, lam=lam)
            (total / WORLD).backward()
            want_loss += part.item() / WORLD
    else:
        joint = {k: torch.cat([x[k] for x in all_in]) if k != "normalizer" else WORLD * all_in[0][k] for k in all_in[0]}
        total, part, _ = policy_objective(model, **joint)
        total.backward()
        want_loss = part.item()
    num = sum((a - p.grad).square().sum() for a, p in zip(got, model.parameters())).sqrt().item()
    den = sum(p.grad.square().sum() for p in model.parameters()).sqrt().item()
    # fp32: sums of up to 48 rows through some ten products, in another order: far below 1e-4.
    ok = num <= 1e-4 * den + 1e-12 and abs(mean_loss.item() / WORLD - want_loss) <= 1e-4 * max(1.0, abs(want_loss))
    return "ok" if ok else f"gradient {num:.2e} of {den:.2e} off, loss {mean_loss.item() / WORLD} for {want_loss}"


def _worker(rank, port, outdir):
    sys.path.insert(0, ROOT)
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=WORLD, timeout=datetime.timedelta(seconds=60))
    from flash_hog_b200 import fused

    fused.policy_loss = _policy_loss
    with open(os.path.join(outdir, f"rank{rank}"), "w") as f:
        f.write("\n".join(_step(rank, *case) for case in CASES))
    dist.destroy_process_group()


@pytest.fixture(scope="module")
def results(tmp_path_factory):
    out = tmp_path_factory.mktemp("ranks")
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    mp.spawn(_worker, args=(port, str(out)), nprocs=WORLD, join=True)
    return [(out / f"rank{r}").read_text().split("\n") for r in range(WORLD)]


@pytest.mark.parametrize("case", range(len(CASES)), ids=[f"{w}-{lam}" for w, lam in CASES])
def test_ranks_average_to_the_weighted_mean_over_all_rows(results, case):
    assert [r[case] for r in results] == ["ok"] * WORLD
