"""The operators around attention in a GPT training step, as they are measured.

Four operators: attention over a sliding window with a few first tokens that stay
visible (sinks), the embedding lookup and its gradient, dropout from a counter-based
generator, and the clipped policy loss. Each case is one pass a training step or a
server makes through one of them; ``own`` selects the framework's calls or the plain
form in elementary torch operations.
"""

import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------
# Cases
# ------------------------------------------------------------------------------------

def _attn(name, pass_, b, tq, tk, h, hk, d, window, sinks, align="top_left", dtype="bf16"):
    return dict(name=name, op="attention", pass_=pass_, b=b, tq=tq, tk=tk, h=h, hk=hk, d=d, window=window,
                sinks=sinks, align=align, dtype=dtype)


def _embed(name, pass_, n, vocab, d, dtype, scale, padding, zipf):
    return dict(name=name, op="embedding", pass_=pass_, n=n, vocab=vocab, d=d, dtype=dtype, scale=scale,
                padding=padding, zipf=zipf)


def _drop(name, rows, cols, p, dtype, residual):
    return dict(name=name, op="dropout", rows=rows, cols=cols, p=p, dtype=dtype, residual=residual)


def _policy(name, rows, vocab, dtype, kl, masked):
    return dict(name=name, op="policy", rows=rows, vocab=vocab, dtype=dtype, kl=kl, masked=masked)


def listed():
    return [
        # One new token of each of 16 sequences against its long key/value tensors.
        _attn("sinks_token_b16_k8192", "fwd", 16, 1, 8192, 16, 4, 64, 1024, 4, "bottom_right"),
        # A training step at the benchmark's headline shape, forward and backward.
        _attn("sinks_grad_b4h16s2048d64", "grad", 4, 2048, 2048, 16, 16, 64, 512, 4),
        # The grad-norm-penalty step of the 12-head GPT: forward, backward and its backward.
        _attn("sinks_hvp_b4h12s1024d64", "hvp", 4, 1024, 1024, 12, 12, 64, 256, 4),
        # Long-context training with grouped heads, the queries a ragged last part of the keys.
        _attn("sinks_grad_b1h8s8000d128", "grad", 1, 8000, 8192, 8, 2, 128, 2048, 64, "bottom_right"),
        # A server's step: one token of each of 64 sequences.
        _embed("embed_tokens_64", "fwd", 64, 32000, 768, "bf16", 1.0, -1, 1.1),
        # The GPT training step: 4 sequences of 1024 tokens, fp32 parameters.
        _embed("embed_grad_4096", "grad", 4096, 32000, 768, "fp32", 1.0, -1, 1.1),
        # A large ragged batch over a large vocabulary, scaled by sqrt(d), with padding.
        _embed("embed_grad_65001", "grad", 65001, 131072, 2048, "bf16", math.sqrt(2048.0), 0, 1.05),
        # Residual dropout of the GPT step under autocast: bf16 branch, fp32 residual stream.
        _drop("dropout_add_4096x768", 4096, 768, 0.1, "bf16", True),
        # Activation dropout of a large layer.
        _drop("dropout_16384x4096", 16384, 4096, 0.1, "bf16", False),
        # The GPT's head on a policy batch: 4096 tokens, a fifth of them prompt.
        _policy("policy_4096x32000", 4096, 32000, "bf16", 0.05, 0.2),
        # The end of a rollout: few rows over a large vocabulary, fp32 logits.
        _policy("policy_7x131072", 7, 131072, "fp32", 0.0, 0.0),
        # A long ragged batch over an odd vocabulary, half of it padding or prompt.
        _policy("policy_8191x50001", 8191, 50001, "bf16", 0.05, 0.5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_attention(rng):
    pass_ = rng.choice(["fwd", "grad", "hvp"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    d = rng.choice([64, 128])
    hk = rng.choice([1, 2, 3, 4, 8])
    h = hk * rng.choice([1, 1, 2, 4])
    b = rng.choice([1, 1, 2, 3, 4])
    most = {"fwd": 4.0e8, "grad": 2.5e8, "hvp": 1.0e8}[pass_] / (4 if dtype == "fp32" else 1)
    tk = _log(rng, 64, max(65, min(8192, int(math.sqrt(most / (b * h))))))
    if pass_ == "fwd" and rng.random() < 0.3:
        tq, align = 1, "bottom_right"
    elif rng.random() < 0.5:
        tq, align = tk, rng.choice(["top_left", "bottom_right"])
    else:
        tq, align = max(32, int(tk * rng.uniform(0.3, 1.0))), "bottom_right"
    tq = min(tq, tk)
    return _attn(None, pass_, b, tq, tk, h, hk, d, _log(rng, 16, 4096), _log(rng, 1, 256), align, dtype)


def _draw_embedding(rng):
    d = _log(rng, 16, 2048)
    vocab = _log(rng, 64, 131072)
    n = _log(rng, 1, 65001)
    pass_ = rng.choice(["fwd", "grad", "grad"])
    dtype = rng.choice(["bf16", "fp32"])
    if dtype == "fp32":
        n = max(1, n // 2)
        vocab = max(64, vocab // 2)
    return _embed(None, pass_, n, vocab, d, dtype, rng.choice([1.0, 0.5, math.sqrt(d)]),
                  rng.choice([-1, 0, vocab - 1]), rng.uniform(0.5, 1.5))


def _draw_dropout(rng):
    cols = _log(rng, 1, 8192)
    rows = max(1, min(_log(rng, 1, 65536), 60_000_000 // cols))
    dtype = rng.choice(["bf16", "fp32"])
    if dtype == "fp32":
        rows = max(1, rows // 2)
    return _drop(None, rows, cols, rng.choice([0.05, 0.1, 0.25, 0.5, 0.9]), dtype, rng.choice([True, False]))


def _draw_policy(rng):
    vocab = _log(rng, 1000, 131072)
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    most = 400_000_000 // (2 if dtype == "fp32" else 1)
    rows = max(2, min(_log(rng, 2, 8191), most // vocab))
    return _policy(None, rows, vocab, dtype, rng.choice([0.0, 0.01, 0.05]), rng.choice([0.0, 0.2, 0.5]))


def draw(rng):
    case = rng.choice([_draw_attention, _draw_embedding, _draw_dropout, _draw_policy])(rng)
    del case["name"]
    return case


# ------------------------------------------------------------------------------------
# Inputs
# ------------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def randn(*shape, dtype=dt, std=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)

    if case["op"] == "attention":
        q_shape = (case["b"], case["tq"], case["h"], case["d"])
        k_shape = (case["b"], case["tk"], case["hk"], case["d"])
        grad = case["pass_"] != "fwd"
        st = dict(case, q=randn(*q_shape), k=randn(*k_shape), v=randn(*k_shape))
        if grad:
            st["do"] = randn(*q_shape)
        if case["pass_"] == "hvp":
            st.update(ddq=randn(*q_shape), ddk=randn(*k_shape), ddv=randn(*k_shape))
        for name in ("q", "k", "v", "do"):
            if name in st:
                st[name].requires_grad_(grad)
        return st
    if case["op"] == "embedding":
        n, vocab = case["n"], case["vocab"]
        # Token frequencies fall like 1 / rank^zipf; ranks are spread over the vocabulary.
        weight = torch.arange(1, vocab + 1, device="cuda", dtype=torch.float64).pow(-case["zipf"])
        cdf = torch.cumsum(weight, 0)
        u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64) * cdf[-1]
        rank = torch.searchsorted(cdf, u).clamp_(max=vocab - 1)
        tokens = torch.randperm(vocab, generator=g, device="cuda")[rank]
        st = dict(case, tokens=tokens, weight=randn(vocab, case["d"], std=0.02))
        if case["pass_"] == "grad":
            st["weight"].requires_grad_(True)
            st["dy"] = randn(n, case["d"])
        return st
    if case["op"] == "dropout":
        shape = (case["rows"], case["cols"])
        st = dict(case, x=randn(*shape).requires_grad_(True), dy=randn(*shape, dtype=torch.float32),
                  seed=torch.tensor([(int(seed) * 0x9E3779B97F4A7C15 + 0x1234567) % (1 << 63)], device="cuda"))
        if case["residual"]:
            st["skip"] = randn(*shape, dtype=torch.float32).requires_grad_(True)
        else:
            st["dy"] = st["dy"].to(dt)
        return st
    rows, vocab = case["rows"], case["vocab"]
    actions = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    logits = randn(rows, vocab, std=2.0)
    # Sampled tokens are likely ones.
    logits[torch.arange(rows, device="cuda"), actions] += torch.rand(rows, generator=g, device="cuda").mul(8).to(dt)
    chosen = logits[torch.arange(rows, device="cuda"), actions].float()
    lp = torch.cat([chosen[i:i + 1024] - torch.logsumexp(logits[i:i + 1024].float(), 1)
                    for i in range(0, rows, 1024)])
    st = dict(case, logits=logits.requires_grad_(True), actions=actions,
              old=lp + randn(rows, dtype=torch.float32, std=0.2), adv=randn(rows, dtype=torch.float32))
    if case["kl"] > 0:
        st["ref"] = lp + randn(rows, dtype=torch.float32, std=0.3)
    if case["masked"] > 0:
        keep = torch.rand(rows, generator=g, device="cuda") >= case["masked"]
        keep[0] = True
        st["weights"] = keep.float()
    return st


# ------------------------------------------------------------------------------------
# One pass
# ------------------------------------------------------------------------------------

def run(state):
    if own:
        return {"attention": _own_attention, "embedding": _own_embedding, "dropout": _own_dropout,
                "policy": _own_policy}[state["op"]](state)
    with torch.no_grad():
        return {"attention": _plain_attention, "embedding": _plain_embedding, "dropout": _plain_dropout,
                "policy": _plain_policy}[state["op"]](state)


def _own_attention(st):
    from flash_hog_b200 import dot_product_attention

    q, k, v = st["q"], st["k"], st["v"]
    o = dot_product_attention(q, k, v, is_causal=True, causal_alignment=st["align"],
                              sliding_window_length=st["window"], sink_tokens=st["sinks"])
    if st["pass_"] == "fwd":
        return {"o": o}
    grads = torch.autograd.grad(o, (q, k, v), st["do"], create_graph=st["pass_"] == "hvp")
    out = {"o": o, **dict(zip(("dq", "dk", "dv"), grads))}
    if st["pass_"] == "hvp":
        second = torch.autograd.grad(grads, (q, k, v, st["do"]), (st["ddq"], st["ddk"], st["ddv"]))
        out.update(zip(("dq2", "dk2", "dv2", "ddo"), second))
    return {n: t.detach() for n, t in out.items()}


def _own_embedding(st):
    from flash_hog_b200 import fused

    pad = st["padding"] if st["padding"] >= 0 else None
    x = fused.embedding(st["tokens"], st["weight"], st["scale"], padding_idx=pad)
    if st["pass_"] == "fwd":
        return {"x": x}
    (dw,) = torch.autograd.grad(x, st["weight"], st["dy"])
    return {"x": x.detach(), "dw": dw}


def _own_dropout(st):
    from flash_hog_b200 import fused

    y = fused.dropout(st["x"], st["p"], st["seed"], subsequence=3, residual=st.get("skip"))
    leaves = [st["x"]] + ([st["skip"]] if "skip" in st else [])
    grads = torch.autograd.grad(y, leaves, st["dy"])
    return {"y": y.detach(), **dict(zip(("dx", "dresidual"), grads))}


def _own_policy(st):
    from flash_hog_b200 import fused

    loss, lp = fused.policy_loss(st["logits"], st["actions"], st["old"], st["adv"], ref_logprobs=st.get("ref"),
                                 weights=st.get("weights"), clip_low=0.2, clip_high=0.28, kl_coef=st["kl"])
    (dz,) = torch.autograd.grad(loss, st["logits"])
    return {"loss": loss.detach(), "logprobs": lp, "dz": dz}


# ------------------------------------------------------------------------------------
# Plain forms
# ------------------------------------------------------------------------------------

def _keep(st, device):
    i = torch.arange(st["tq"], device=device)[:, None] + (st["tk"] - st["tq"] if st["align"] == "bottom_right" else 0)
    j = torch.arange(st["tk"], device=device)[None, :]
    return (j <= i) & ((j > i - st["window"]) | (j < st["sinks"]))


def _plain_attention(st):
    dt, g, scale = DTYPES[st["dtype"]], st["h"] // st["hk"], st["d"] ** -0.5

    def heads(x):  # (B, T, N, D) -> (B, heads, T, D) in 32 bits, key heads repeated over their group
        x = x.float().transpose(1, 2)
        return x.repeat_interleave(g, 1) if x.shape[1] != st["h"] else x

    def out(x, key_side=False):
        if key_side:
            x = x.reshape(x.shape[0], st["hk"], g, *x.shape[2:]).sum(2)
        return x.transpose(1, 2).to(dt).contiguous()

    def mm(a, b):
        return a @ b

    def t(x):
        return x.transpose(-1, -2)

    q, k, v = heads(st["q"]), heads(st["k"]), heads(st["v"])
    keep = _keep(st, q.device)
    s = (mm(q, t(k)) * scale).masked_fill_(~keep, float("-inf"))
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
    p = torch.exp(s.sub_(m))
    p = p.div_(p.sum(-1, keepdim=True).clamp_min(1e-38))
    del s
    o = mm(p, v)
    res = {"o": out(o)}
    if st["pass_"] == "fwd":
        return res
    do = heads(st["do"])
    dp = mm(do, t(v))
    delta = (p * dp).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    res.update(dq=out(mm(ds, k) * scale), dk=out(mm(t(ds), q) * scale, True), dv=out(mm(t(p), do), True))
    if st["pass_"] == "grad":
        return res
    ddq, ddk, ddv = heads(st["ddq"]), heads(st["ddk"]), heads(st["ddv"])
    dds = (mm(ddq, t(k)) + mm(q, t(ddk))) * scale
    u = dds - (p * dds).sum(-1, keepdim=True)
    ddp = p * u
    e = mm(do, t(ddv)) + dp * u - dds * delta
    ds2 = p * (e - (p * e).sum(-1, keepdim=True))
    res.update(dq2=out((mm(ds, ddk) + mm(ds2, k)) * scale),
               dk2=out((mm(t(ds), ddq) + mm(t(ds2), q)) * scale, True),
               dv2=out(mm(t(ddp), do), True), ddo=out(mm(ddp, v) + mm(p, ddv)))
    return res


def _plain_embedding(st):
    dt, tokens, weight = DTYPES[st["dtype"]], st["tokens"], st["weight"]
    x = (weight[tokens].float() * st["scale"]).to(dt)
    if st["pass_"] == "fwd":
        return {"x": x}
    dw = torch.zeros(weight.shape, dtype=torch.float32, device=weight.device)
    dw.index_add_(0, tokens, st["dy"].float())
    dw.mul_(st["scale"])
    if st["padding"] >= 0:
        dw[st["padding"]] = 0.0
    return {"x": x, "dw": dw.to(dt)}


def _plain_draws(seed, n, subsequence):
    """n 16-bit draws: Philox4x32-10 (Salmon et al., 2011) on counters (block, subsequence), 8 draws a block."""
    blocks = (n + 7) // 8
    mask = 0xFFFFFFFF
    c0 = torch.arange(blocks, device=seed.device)
    c1 = c0 >> 32
    c0 = c0 & mask
    c2 = torch.full_like(c0, subsequence)
    c3 = torch.zeros_like(c0)
    k0, k1 = seed & mask, (seed >> 32) & mask

    def mul(a, b):  # (high, low) words of a 32 x 32 bit product
        p = a * b
        return (p >> 32) & mask, p & mask

    for _ in range(10):
        h0, l0 = mul(c0, 0xD2511F53)
        h1, l1 = mul(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & mask, (k1 + 0xBB67AE85) & mask
    words = torch.stack((c0, c1, c2, c3), 1)
    return torch.stack((words & 0xFFFF, words >> 16), 2).reshape(-1)[:n]


def _plain_dropout(st):
    x, dt = st["x"], DTYPES[st["dtype"]]
    limit = round(st["p"] * 65536)
    factor = 65536.0 / (65536 - limit)
    keep = (_plain_draws(st["seed"], x.numel(), 3) >= limit).view(x.shape)
    y = torch.where(keep, x.float() * factor, torch.zeros((), device=x.device))
    res = {}
    if "skip" in st:
        y = y + st["skip"]
        res["dresidual"] = st["dy"]
    else:
        y = y.to(dt)
    return {"y": y, "dx": torch.where(keep, st["dy"].float() * factor, torch.zeros((), device=x.device)).to(dt), **res}


def _plain_policy(st):
    z, a = st["logits"].float(), st["actions"][:, None]
    m = z.amax(1, keepdim=True)
    e = torch.exp(z - m)
    total = e.sum(1, keepdim=True, dtype=torch.float64)
    lp = ((z.gather(1, a) - m).double() - total.log()).squeeze(1)  # 64 bits: ratios next to the clip borders
    w = st["weights"] if "weights" in st else torch.ones_like(st["adv"])
    adv, log_ratio = st["adv"].double(), lp - st["old"].double()
    ratio = torch.exp(log_ratio)
    rows = -torch.minimum(ratio * adv, ratio.clamp(0.8, 1.28) * adv)
    clipped = ((adv > 0) & (ratio > 1.28)) | ((adv < 0) & (ratio < 0.8))
    coef = torch.where(clipped, torch.zeros_like(ratio), -adv * ratio)
    if st["kl"] > 0:
        d = st["ref"].double() - lp
        rows = rows + st["kl"] * (torch.exp(d) - d - 1)
        coef = coef + st["kl"] * (1 - torch.exp(d))
    count = w.double().sum()
    loss = (rows * w).sum() / count
    coef = (coef * w / count).float()[:, None]
    dz = e.mul_(-coef / total.float())
    dz.scatter_add_(1, a, coef)
    lp = torch.where(w > 0, lp, torch.zeros_like(lp))
    return {"loss": loss.float(), "logprobs": lp.float(), "dz": dz.to(st["logits"].dtype)}


# ------------------------------------------------------------------------------------
# What a pass cannot do without
# ------------------------------------------------------------------------------------

def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "attention":
        i = np.arange(case["tq"], dtype=np.int64)
        diag = i + (case["tk"] - case["tq"] if case["align"] == "bottom_right" else 0)
        hi = np.minimum(diag, case["tk"] - 1)
        lo = np.maximum(0, diag - case["window"] + 1)
        band = np.maximum(0, hi - lo + 1)
        front = np.maximum(0, np.minimum(np.minimum(lo, case["sinks"]), hi + 1))
        pairs = int((band + front).sum()) * case["b"] * case["h"]
        q = case["b"] * case["tq"] * case["h"] * case["d"] * size
        # Keys that some query sees: the sinks and the band of all queries.
        first = int(lo.min()) if case["tq"] else 0
        seen = case["tk"] - first + min(first, case["sinks"])
        k = case["b"] * seen * case["hk"] * case["d"] * size
        k_all = case["b"] * case["tk"] * case["hk"] * case["d"] * size
        products = {"fwd": 2, "grad": 7, "hvp": 19}[case["pass_"]]
        data = {"fwd": 2 * q + 2 * k, "grad": 4 * q + 2 * k + 2 * k_all,
                "hvp": 7 * q + 4 * k + 4 * k_all}[case["pass_"]]
        return {"bytes": data, "flops": 2 * products * pairs * case["d"]}
    if case["op"] == "embedding":
        row = case["d"] * size
        data = case["n"] * (8 + 2 * row)
        if case["pass_"] == "grad":
            data += case["n"] * row + case["vocab"] * row
        return {"bytes": data, "flops": case["n"] * case["d"] * (2 if case["pass_"] == "grad" else 1)}
    if case["op"] == "dropout":
        n = case["rows"] * case["cols"]
        per = (size + 4 + 4) + (4 + size) if case["residual"] else 4 * size
        return {"bytes": n * per, "flops": 4 * n}
    n = int(case["rows"] * (1 - case["masked"]) + 0.5) * case["vocab"]
    return {"bytes": n * size + case["rows"] * case["vocab"] * size + case["rows"] * 28, "flops": 6 * n}


# ------------------------------------------------------------------------------------
# The same from the definitions, in 64 bits
# ------------------------------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    return {"attention": _exact_attention, "embedding": _exact_embedding, "dropout": _exact_dropout,
            "policy": _exact_policy}[case["op"]](st)


def _exact_attention(st):
    """Head by head: the softmax of the visible scores, differentiated by autograd as often as the pass asks for."""
    group = st["h"] // st["hk"]
    names = [n for n in ("q", "k", "v", "do", "ddq", "ddk", "ddv") if n in st]
    keep = _keep(st, st["q"].device)
    blind = ~keep.any(1)
    sums = {}
    for b in range(st["b"]):
        for h in range(st["h"]):
            x = {n: st[n][b, :, h // group if n in ("k", "v", "ddk", "ddv") else h].detach().double() for n in names}
            with torch.enable_grad():
                for n in ("q", "k", "v", "do"):
                    if n in x:
                        x[n].requires_grad_(st["pass_"] != "fwd")
                s = (x["q"] @ x["k"].T) / math.sqrt(st["d"])
                # Rows without a visible key: softmax over zeros, then nothing of it.
                s = torch.where(keep, s, torch.where(blind[:, None], 0.0, -math.inf))
                p = torch.softmax(s, 1) * (~blind)[:, None]
                got = {"o": p @ x["v"]}
                if st["pass_"] != "fwd":
                    first = torch.autograd.grad(got["o"], (x["q"], x["k"], x["v"]), x["do"],
                                                create_graph=st["pass_"] == "hvp")
                    got.update(zip(("dq", "dk", "dv"), first))
                if st["pass_"] == "hvp":
                    got.update(zip(("dq2", "dk2", "dv2", "ddo"),
                                   torch.autograd.grad(first, (x["q"], x["k"], x["v"], x["do"]),
                                                       (x["ddq"], x["ddk"], x["ddv"]))))
            for n, v in got.items():
                key_side = n in ("dk", "dv", "dk2", "dv2")
                if n not in sums:
                    shape = st["k"].shape if key_side else st["q"].shape
                    sums[n] = torch.zeros(shape, dtype=torch.float64, device=v.device)
                sums[n][b, :, h // group if key_side else h] += v.detach()
    return sums


def _exact_embedding(st):
    tokens = st["tokens"]
    x = st["weight"].detach()[tokens].double() * st["scale"]
    if st["pass_"] == "fwd":
        return {"x": x}
    # Sums over runs of equal tokens, from running sums over the sorted rows.
    order = torch.argsort(tokens, stable=True)
    run = torch.cumsum(st["dy"][order].double(), 0)
    counts = torch.bincount(tokens, minlength=st["vocab"])
    end = torch.cumsum(counts, 0)
    run = torch.cat((torch.zeros_like(run[:1]), run))
    dw = (run[end] - run[end - counts]) * st["scale"]
    if st["padding"] >= 0:
        dw[st["padding"]] = 0.0
    return {"x": x, "dw": dw}


def _exact_dropout(st):
    n = st["x"].numel()
    key = int(st["seed"].item())
    lo, k = np.uint64(0xFFFFFFFF), [key & 0xFFFFFFFF, (key >> 32) & 0xFFFFFFFF]
    index = np.arange((n + 7) // 8, dtype=np.uint64)
    c = [index & lo, index >> np.uint64(32), np.full_like(index, 3), np.zeros_like(index)]
    for r in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        k0, k1 = np.uint64((k[0] + r * 0x9E3779B9) & 0xFFFFFFFF), np.uint64((k[1] + r * 0xBB67AE85) & 0xFFFFFFFF)
        c = [(b >> np.uint64(32)) ^ c[1] ^ k0, b & lo, (a >> np.uint64(32)) ^ c[3] ^ k1, a & lo]
    draws = np.empty((len(index), 8), np.uint16)
    for w in range(4):
        draws[:, 2 * w] = (c[w] & np.uint64(0xFFFF)).astype(np.uint16)
        draws[:, 2 * w + 1] = (c[w] >> np.uint64(16)).astype(np.uint16)
    limit = round(st["p"] * 65536)
    gate = torch.from_numpy((draws.reshape(-1)[:n] >= limit) / (1.0 - limit / 65536.0)).view(st["x"].shape)
    dy = st["dy"].double().cpu()
    res = {"y": st["x"].detach().double().cpu() * gate, "dx": dy * gate}
    if "skip" in st:
        res["y"] += st["skip"].detach().double().cpu()
        res["dresidual"] = dy
    return res


def _exact_policy(st):
    z = st["logits"].detach()
    w = st["weights"].double() if "weights" in st else torch.ones(st["rows"], dtype=torch.float64, device=z.device)
    count, losses, lps, grads = w.sum(), [], [], []
    for r0 in range(0, st["rows"], 512):
        part = slice(r0, min(st["rows"], r0 + 512))
        with torch.enable_grad():
            x = z[part].double().requires_grad_(True)
            lp = torch.log_softmax(x, 1).gather(1, st["actions"][part, None])[:, 0]
            ratio = torch.exp(lp - st["old"][part].double())
            adv = st["adv"][part].double()
            # min(rho A, clip(rho) A): the clipped side carries no gradient.
            upper = torch.where(adv >= 0, 1.28, math.inf)
            lower = torch.where(adv < 0, 0.8, 0.0)
            inside = (ratio <= upper) & (ratio >= lower)
            loss = -adv * torch.where(inside, ratio, torch.where(adv >= 0, 1.28, 0.8))
            if st["kl"] > 0:
                d = st["ref"][part].double() - lp
                loss = loss + st["kl"] * (torch.expm1(d) - d)
            loss = (loss * w[part]).sum() / count
            grads.append(torch.autograd.grad(loss, x)[0].to(torch.float32 if z.dtype == torch.bfloat16 else x.dtype))
        losses.append(loss.detach())
        lps.append(torch.where(w[part] > 0, lp.detach(), 0.0))
    return {"loss": torch.stack(losses).sum(), "logprobs": torch.cat(lps), "dz": torch.cat(grads)}
