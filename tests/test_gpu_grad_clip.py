"""GPU: global gradient norm and clipping against 64 bits.

The norm: squares summed in fp32 over at most 64 values a thread and chunk, the
rest in fp64, one rounding: relative error <= 64 x 2^-24.  An output is
g x c with c within 66 x 2^-24 of max_norm / (norm + eps), rounded once.
"""

from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
U = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "fp32": E}


@pytest.fixture(scope="module")
def ks(cuda_ok):
    import torch

    from kernscope_b200 import native, ops

    torch.cuda.set_device(0)
    return native, ops, torch


def _dt(torch, name):
    return {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}[name]


def _check(torch, ops, grads, names, max_norm, in_place, outs=None, eps=1e-6):
    before = [g.clone() for g in grads]
    clipper = ops.GradClipper(grads) if in_place else ops.GradClipper(grads, out=outs)
    norm = clipper.clip(max_norm, eps)
    want = math.sqrt(sum(float(g.double().square().sum()) for g in before))
    assert norm.shape == (1,) and norm.dtype == torch.float32
    assert abs(float(norm) - want) <= 64 * E * want
    c = min(1.0, max_norm / (want + eps))
    for g, b, o, name in zip(grads, before, grads if in_place else outs, names):
        exact = b.double() * c
        step = 2.0 ** -25 if name == "fp16" else 1e-38
        tol = (U[name] + 70 * E) * exact.abs() + step
        assert ((o.double() - exact).abs() <= tol).all()
        if c == 1.0:
            assert torch.equal(o, b)
        if not in_place:
            assert torch.equal(g, b)
    return norm


SETS = [  # sizes of the tensors
    [1], [7], [0, 3, 0], [31, 1000, 5, 8192, 8191, 8193], [16384 * 3 + 5, 16383], [1] * 300, [1_000_003, 17, 4096, 250_000],
    [20_000_000],
]


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32", "mixed"])
@pytest.mark.parametrize("sizes", SETS, ids=lambda s: f"{len(s)}x{max(s)}")
def test_norm_and_clipping(ks, sizes, dtype, in_place):
    N, ops, torch = ks
    g = torch.Generator(device="cuda")
    g.manual_seed(len(sizes))
    names = [["bf16", "fp32", "fp16"][i % 3] if dtype == "mixed" else dtype for i in range(len(sizes))]
    grads = [torch.randn(n, generator=g, device="cuda").to(_dt(torch, k)) for n, k in zip(sizes, names)]
    outs = None if in_place else [torch.full_like(x, 5) for x in grads]
    total = math.sqrt(sum(float(x.double().square().sum()) for x in grads))
    _check(torch, ops, grads, names, total * 0.3, in_place, outs)  # clipped
    _check(torch, ops, grads, names, total * 3 + 1, in_place, outs)  # kept as it is


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("g_off,o_off", [(0, 0), (1, 1), (3, 3), (1, 0), (0, 5), (2, 7)])
def test_unaligned_tensors_and_their_neighbours(ks, dtype, g_off, o_off):
    """Tensors that begin anywhere in a buffer; outputs whose alignment differs
    from the gradients'; nothing beside them is written."""
    N, ops, torch = ks
    for n in (1, 6, 9, 16380, 16400, 50_001):
        flat_g = torch.randn(n + 16, device="cuda").to(_dt(torch, dtype))
        flat_o = torch.full_like(flat_g, 7)
        _check(torch, ops, [flat_g[g_off:g_off + n]], [dtype], 0.5, False, [flat_o[o_off:o_off + n]])
        assert (flat_o[:o_off] == 7).all() and (flat_o[o_off + n:] == 7).all()


def test_same_bits_every_time_and_on_another_stream(ks):
    N, ops, torch = ks
    grads = [torch.randn(n, device="cuda") for n in (3_000_001, 77, 500_000)]
    outs = [torch.empty_like(x) for x in grads]
    clipper = ops.GradClipper(grads, out=outs)
    norm = clipper.clip(1.0)
    first = [o.clone() for o in outs]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for stream in (None, s, s):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        again = clipper.clip(1.0, stream=stream)
        torch.cuda.synchronize()
        assert torch.equal(norm, again) and all(torch.equal(a, b) for a, b in zip(first, outs))


def test_values_that_are_not_finite(ks):
    """The formula's own results: an infinite norm scales by zero, a NaN spreads."""
    N, ops, torch = ks
    x = torch.ones(5000, device="cuda")
    x[4321] = float("inf")
    norm = ops.GradClipper([x]).clip(1.0)
    assert math.isinf(float(norm)) and torch.isnan(x[4321]) and (x[:4321] == 0).all()
    x = torch.ones(5000, device="cuda").bfloat16()
    x[17] = float("nan")
    norm = ops.GradClipper([x]).clip(1.0)
    assert math.isnan(float(norm)) and torch.isnan(x).all()


def test_zero_gradients_and_zero_max_norm(ks):
    N, ops, torch = ks
    x = torch.zeros(1000, device="cuda")
    assert float(ops.GradClipper([x]).clip(1.0)) == 0 and (x == 0).all()
    x = torch.ones(1000, device="cuda")
    assert abs(float(ops.GradClipper([x]).clip(0.0)) - math.sqrt(1000)) < 1e-4 and (x == 0).all()


def test_refusals(ks):
    N, ops, torch = ks
    x = torch.ones(100, device="cuda")
    for bad in [
        lambda: ops.GradClipper([]),
        lambda: ops.GradClipper([x.cpu()]),
        lambda: ops.GradClipper([x.double()]),
        lambda: ops.GradClipper([x.view(10, 10).t()]),
        lambda: ops.GradClipper([x], out=[]),
        lambda: ops.GradClipper([x], out=[x.half()]),
        lambda: ops.GradClipper([x], out=[x[:50]]),
        lambda: ops.GradClipper([x, x]),  # a shared parameter's gradient would count and be scaled twice
        lambda: ops.GradClipper([x[:60], x[50:]]),
        lambda: ops.GradClipper([x[:50]], out=[x[10:60]]),
    ]:
        with pytest.raises(ValueError):
            bad()
    for max_norm, eps in ((-1.0, 1e-6), (float("nan"), 1e-6), (1.0, -1.0)):
        with pytest.raises(N.KsError) as e:
            ops.GradClipper([x]).clip(max_norm, eps)
        assert e.value.status == N.KS_ERR_INVALID_ARGS
