"""The C++ entry points let other Python threads run while a call waits for the GPU's launch
queue."""

import threading
import time

import pytest
import torch

from flash_hog_b200 import dot_product_attention, fused


def _calls():
    q = torch.randn(1, 16, 1, 64, device="cuda", dtype=torch.bfloat16)
    x, seed = torch.randn(64, device="cuda"), torch.zeros(1, dtype=torch.long, device="cuda")
    w, tokens = torch.randn(10, 8, device="cuda"), torch.arange(4, device="cuda")
    z, vec = torch.randn(2, 16, device="cuda"), torch.zeros(2, device="cuda")
    act = torch.zeros(2, dtype=torch.long, device="cuda")
    return {
        "attention": lambda: dot_product_attention(q, q, q, is_causal=True),
        "dropout": lambda: fused.dropout(x, 0.5, seed),
        "embedding": lambda: fused.embedding(tokens, w),
        "policy_loss": lambda: fused.policy_loss(z, act, vec, vec),
    }


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["attention", "dropout", "embedding", "policy_loss"])
def test_other_threads_run_while_a_launch_waits(name):
    call = _calls()[name]
    call()
    torch.cuda.synchronize()
    ticks, done = [], threading.Event()

    def tick():
        while not done.is_set():
            ticks.append(time.perf_counter())
            time.sleep(0.002)

    thread = threading.Thread(target=tick)
    thread.start()
    try:
        begin = time.perf_counter()
        torch.cuda._sleep(2_000_000_000)  # a second or so, in which the queue of launches fills up
        for _ in range(3000):
            call()
        torch.cuda.synchronize()
        took = time.perf_counter() - begin
    finally:
        done.set()
        thread.join()
    gap = max(b - a for a, b in zip(ticks, ticks[1:]))
    # The first launch that finds the queue full (after a thousand or so, some 20 ms) waits for
    # the rest of the second; a thread that only shares the interpreter gets it every few
    # milliseconds.
    assert took > 0.5 and gap < 0.5 * took
