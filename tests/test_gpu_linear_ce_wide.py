"""GPU: a few to a few hundred tokens over a wide vocabulary, on both sides of the
rule that says which kernel takes the rows' statistics; bounds as in
test_gpu_linear_ce.py, from the same arithmetic."""

from __future__ import annotations

import pytest

from test_gpu_linear_ce import E, IGNORE, _dt, _exact, _make, _near

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("shape", [(2, 64, 140001), (64, 64, 140001), (60, 72, 30000), (300, 64, 140001), (500, 72, 30000)],
                         ids=str)
def test_wide_vocabulary(cuda_ok, shape, dtype):
    import torch

    from kernscope_b200 import ops

    torch.cuda.set_device(0)
    n, dim, vocab = shape
    h, w, t = _make(torch, n, dim, vocab, _dt(torch, dtype), seed=n + vocab)
    count = max(1, int((t != IGNORE).sum()))
    ref = _exact(torch, h, w, t, torch.full((n,), 1.0 / count, device="cuda"))
    mean, dh, dw = ops.linear_cross_entropy_grad(h, w, t)
    _near(torch, mean, ref["loss"].sum().reshape(1) / count,
          (ref["loss_tol"].sum() / count + E * ref["loss"].sum()).reshape(1), "mean")
    _near(torch, dh, ref["dh"], ref["dh_tol"], "dh")
    _near(torch, dw, ref["dw"], ref["dw_tol"], "dw")
    again = ops.linear_cross_entropy_grad(h, w, t)
    assert all(torch.equal(a, b) for a, b in zip((mean, dh, dw), again))
    assert ops.device_error_take() == 0
