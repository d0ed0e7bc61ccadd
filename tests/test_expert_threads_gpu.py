"""GPU: calls from two threads whose kernels need different amounts of shared memory."""

from __future__ import annotations

import threading

import pytest
import torch

import test_int8_gpu as T
from piper_offload_b200 import int8, routing

pytestmark = pytest.mark.gpu


def both(calls, turns):
    """Each call so often on a thread and a stream of its own: what raised, and whether every result was the first one's."""
    failed, same = [], []
    gate = threading.Barrier(len(calls))

    def work(call):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                first = call()
                equal = torch.ones((), dtype=torch.bool, device="cuda")
                gate.wait()
                for _ in range(turns):
                    equal &= (call() == first).all()
                same.append(bool(equal))
        except Exception as exc:  # noqa: BLE001
            failed.append(exc)
            gate.abort()

    threads = [threading.Thread(target=work, args=(call,)) for call in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    return failed, same


def test_products_of_a_few_tokens(cuda_device):
    """One kernel, of which a weight of 128 x 256 needs two stages of shared memory and one of 9600 x 4096 twelve."""
    calls = []
    for rows, cols in ((128, 256), (9600, 4096)):
        w, _, _ = T.make_weight("rows", rows, cols, cuda_device)
        x = torch.randn(1, cols, device=cuda_device).bfloat16()
        calls.append(lambda w=w, x=x: int8.linear_int8(x, w))
    failed, same = both(calls, 4000)
    assert not failed and same == [True, True]


@pytest.mark.parametrize("tokens", [100, 400])
def test_routing_to_many_experts(tokens, cuda_device):
    """Above 682 experts placing takes more shared memory than any launch may have unasked, by their number."""
    calls = []
    for experts in (700, 1024):
        logits = torch.randn(tokens, experts, device=cuda_device)
        calls.append(lambda logits=logits: routing.route_tokens(logits, 4).source)
    failed, same = both(calls, 4000)
    assert not failed and same == [True, True]
