"""GPU: what the training operators' objects own while calls on other streams are
still queued."""

from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ks(cuda_ok):
    import torch

    from kernscope_b200 import ops

    torch.cuda.set_device(0)
    return ops, torch


def test_clipper_dropped_behind_a_queued_call(ks):
    """The clipper's table and scratch are not handed out again before the call on
    the other stream has run."""
    ops, torch = ks
    grads = [torch.full((5000,), 2.0, device="cuda"), torch.full((70,), 2.0, device="cuda")]
    outs = [torch.zeros_like(g) for g in grads]
    clipper = ops.GradClipper(grads, out=outs)
    held = {clipper._table.data_ptr(): clipper._table.numel(), clipper._scratch.data_ptr(): clipper._scratch.numel()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(400_000_000)  # about a fifth of a second
        busy = torch.cuda.Event()
        busy.record()
    norm = clipper.clip(1.0, stream=side)
    del clipper
    taken = [torch.empty(n, dtype=torch.uint8, device="cuda") for n in held.values() for _ in range(8)]
    if busy.query():
        pytest.skip("the other stream had finished too early to show anything")
    assert not held.keys() & {t.data_ptr() for t in taken}
    torch.cuda.synchronize()
    want = math.sqrt(4 * 5070)
    assert abs(float(norm) - want) <= 1e-5 * want
    for o in outs:
        assert (o - 2 / want).abs().max() <= 1e-6
