"""GPU: the vocabulary-end operators together, as a training program runs them."""

from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def step(cuda_ok):
    import torch

    from kernscope_b200 import train_step

    torch.cuda.set_device(0)
    return torch, train_step


@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_gradients_of_the_whole_path(step, tied, dtype):
    """Every parameter's gradient against 64 bits.  Three roundings to 16 bits lie
    on the path (d, dh, the result; four for a tied table): in the 2-norm, where
    independent roundings add as squares, each is below its largest relative
    size u, so 3 u covers their sum."""
    torch, ts = step
    dt = {"bf16": torch.bfloat16, "fp16": torch.float16}[dtype]
    m = ts.VocabModel(700, 96, dt, tied, seed=3)
    tokens, targets = ts.synthetic_text(700, 1500, seed=5)
    targets[::7] = -100
    loss = m.gradients(tokens, targets)
    table, w = m.param[0].double(), m.param[-1].double()
    table.requires_grad_()
    w = table if tied else w.requires_grad_()
    h = (table[tokens] * m.scale)
    h = h + (m.param[0][tokens].double() * m.scale).to(dt).double().sub(h).detach()  # the lookup's rounding
    want = torch.nn.functional.cross_entropy(h @ w.t(), targets, ignore_index=-100)
    want.backward()
    assert abs(float(loss) - float(want)) <= 1e-5 * float(want)
    u = 2.0 ** -8 if dtype == "bf16" else 2.0 ** -11
    for got, ref in zip(m.grad, [table.grad] if tied else [table.grad, w.grad]):
        assert float((got.double() - ref).norm() / ref.norm()) <= 3 * u


@pytest.mark.parametrize("tied", [False, True])
def test_loss_falls(step, tied):
    torch, ts = step
    m = ts.VocabModel(512, 128, tied=tied)
    first = last = None
    for i in range(60):
        loss, norm = m.step(*ts.synthetic_text(512, 4096, seed=i), lr=4.0)
        assert math.isfinite(float(norm))
        first, last = (float(loss) if first is None else first), float(loss)
    assert last < first - 1.0


def test_command(step, capsys):
    torch, ts = step
    assert ts.main(["--tokens", "512", "--dim", "64", "--vocab", "300", "--steps", "3"]) == 0
    assert "gradient norm" in capsys.readouterr().out
