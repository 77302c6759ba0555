"""GPU: rows of hidden states without a gradient may hold anything.

d of such a row is 0, so the gradients are those of the same call with zeros in
its place: the same products in the same order, bit for bit.
"""

from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu

IGNORE = -100


@pytest.fixture(scope="module")
def ks(cuda_ok):
    import torch

    from kernscope_b200 import native, ops

    torch.cuda.set_device(0)
    return native, ops, torch


def _make(torch, n, dim, vocab, dtype, pad=0):
    """h, targets with every kind of row without gradient among others, and the rows
    of h that are foul: whole rows of NaN, one infinity, one NaN."""
    g = torch.Generator(device="cuda")
    g.manual_seed(n + dim)
    h = torch.randn(n, dim + pad, generator=g, device="cuda").to(dtype)[:, :dim]
    w = (torch.randn(vocab, dim + pad, generator=g, device="cuda") / math.sqrt(dim)).to(dtype)[:, :dim]
    t = torch.randint(0, vocab, (n,), generator=g, device="cuda")
    out = torch.rand(n, generator=g, device="cuda") < 0.3
    out[-1] = True
    t[out] = IGNORE
    rows = out.nonzero()[:, 0]
    h[rows[0::4]] = float("nan")
    h[rows[1::4], dim // 2] = float("inf")
    h[rows[2::4], dim - 1] = float("-inf")  # every fourth stays finite
    return h, w, t, out


def _zeroed(torch, h, rows):
    clean = h.clone()
    clean[rows] = 0
    return clean


TILES = [0, 128, (128, 256), 256]
SHAPES = [(1, 64, 40), (17, 72, 300), (64, 264, 1500), (65, 64, 700), (200, 136, 1111), (700, 72, 4099), (1300, 520, 900)]


@pytest.mark.parametrize("tile", TILES, ids=str)
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_loss_and_gradient(ks, shape, dtype, tile):
    N, ops, torch = ks
    n, dim, vocab = shape
    h, w, t, out = _make(torch, n, dim, vocab, getattr(torch, dtype), pad=(0, 8, 3)[n % 3])
    tm, tn = tile if isinstance(tile, tuple) else (tile, tile)
    for piece in (0, 256):  # with the exponentials kept, and from logits taken again
        cfg = N.LinearCeConfig(tm, tn, piece)
        want = ops.linear_cross_entropy_grad(_zeroed(torch, h, out), w, t, reduction="sum", cfg=cfg)
        got = ops.linear_cross_entropy_grad(h, w, t, reduction="sum", cfg=cfg)
        for name, a, b in zip(("loss", "dh", "dw"), got, want):
            assert torch.isfinite(b.float()).all() and torch.equal(a, b), (name, piece)
        assert (got[1][out] == 0).all()
    assert ops.device_error_take() == 0


@pytest.mark.parametrize("piece", [0, 256])
@pytest.mark.parametrize("reduction", ["none", "mean"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_backward(ks, shape, reduction, piece):
    """Rows whose own dloss is 0 too."""
    N, ops, torch = ks
    n, dim, vocab = shape
    h, w, t, out = _make(torch, n, dim, vocab, torch.bfloat16)
    cfg = N.LinearCeConfig(0, 0, piece)
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    dloss = torch.randn(n if reduction == "none" else 1, generator=g, device="cuda")
    if reduction == "none" and n > 1:
        t[out.nonzero()[0::2, 0]] = 3  # these have a target, and a dloss of 0
        dloss[out] = 0
    clean = _zeroed(torch, h, out)
    lse, clean_lse = ops.linear_cross_entropy(h, w, t)[1], ops.linear_cross_entropy(clean, w, t)[1]
    want = ops.linear_cross_entropy_backward(clean, w, t, clean_lse, dloss, reduction=reduction, cfg=cfg)
    got = ops.linear_cross_entropy_backward(h, w, t, lse, dloss, reduction=reduction, cfg=cfg)
    for name, a, b in zip(("dh", "dw"), got, want):
        assert torch.isfinite(b.float()).all() and torch.equal(a, b), name
    assert (got[0][out] == 0).all()


def test_targets_out_of_range_and_rows_without_any(ks):
    N, ops, torch = ks
    h, w, t, out = _make(torch, 150, 128, 500, torch.bfloat16)
    t[out.nonzero()[0::2, 0]] = 500
    loss, dh, dw = ops.linear_cross_entropy_grad(h, w, t)
    want = ops.linear_cross_entropy_grad(_zeroed(torch, h, out), w, t)
    assert torch.isnan(loss).all() and torch.equal(dh, want[1]) and torch.equal(dw, want[2])
    assert torch.isfinite(dw.float()).all() and torch.isfinite(dh.float()).all()
    t[:] = IGNORE
    h[:] = float("nan")
    loss, dh, dw = ops.linear_cross_entropy_grad(h, w, t)
    assert float(loss) == 0 and (dh == 0).all() and (dw == 0).all()


def test_rows_with_a_gradient_keep_theirs(ks):
    """A NaN in a token that counts still shows."""
    N, ops, torch = ks
    h, w, t, out = _make(torch, 90, 64, 200, torch.bfloat16)
    row = int((~out).nonzero()[0, 0])
    h[row, 1] = float("nan")
    loss, dh, dw = ops.linear_cross_entropy_grad(h, w, t)
    assert torch.isnan(loss).all() and torch.isnan(dh[row]).all() and torch.isnan(dw[:, 1]).all()
