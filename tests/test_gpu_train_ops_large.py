"""GPU: the training operators where offsets pass 2^31 elements, inside CUDA
graphs, and on a side stream beside other work."""

from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu

FAR = (1 << 31) // 4096 + 3000  # rows of 4096 that pass 2^31 elements


@pytest.fixture(scope="module")
def ks(cuda_ok):
    import torch

    from kernscope_b200 import ops

    torch.cuda.set_device(0)
    return ops, torch


def test_lookup_and_gradient_far_into_the_table(ks):
    ops, torch = ks
    table = torch.zeros(FAR, 4096, dtype=torch.bfloat16, device="cuda")
    rows = torch.tensor([0, 5, (1 << 31) // 4096 - 1, (1 << 31) // 4096, FAR - 1], device="cuda")
    table[rows] = torch.arange(1, 6, device="cuda", dtype=torch.bfloat16)[:, None]
    out = ops.embedding(rows.flip(0), table, scale=2.0)
    assert torch.equal(out, table[rows.flip(0)] * 2)
    grad = ops.embedding_backward(rows, out, FAR, dtable=table)
    assert torch.equal(grad[rows], out)
    assert float(grad.float().abs().sum(dtype=torch.float64)) == float(out.float().abs().sum(dtype=torch.float64))


def test_gradient_of_far_positions(ks):
    ops, torch = ks
    n = FAR
    dout = torch.zeros(n, 4096, dtype=torch.bfloat16, device="cuda")
    tokens = torch.full((n,), -1, device="cuda")
    at = torch.tensor([1, (1 << 31) // 4096 + 1, n - 1], device="cuda")
    dout[at] = torch.tensor([1.0, 2.0, 4.0], dtype=torch.bfloat16, device="cuda")[:, None]
    tokens[at] = torch.tensor([7, 7, 3], device="cuda")
    grad = ops.embedding_backward(tokens, dout, 10)
    assert (grad[7] == 3).all() and (grad[3] == 4).all() and float(grad.float().sum()) == 4096 * 7.0


def test_cross_entropy_over_a_vocabulary_past_2_31_weights(ks):
    """Logits are 0 but for two far columns; the loss and the two gradients have
    closed forms: p = e^l / (V - 2 + sum e^l)."""
    ops, torch = ks
    dim, vocab = 4096, FAR
    w = torch.zeros(vocab, dim, dtype=torch.bfloat16, device="cuda")
    h = torch.zeros(3, dim, dtype=torch.bfloat16, device="cuda")
    h[:, 0] = 1
    far = [(1 << 31) // dim + 17, vocab - 1]
    w[far[0], 0], w[far[1], 0] = 12.0, 10.0
    t = torch.tensor([far[0], far[1], 2], device="cuda")
    total = vocab - 2 + math.exp(12) + math.exp(10)
    want = [math.log(total) - x for x in (12.0, 10.0, 0.0)]
    loss, lse = ops.linear_cross_entropy(h, w, t)
    for a, b in zip(loss.tolist(), want):
        assert abs(a - b) <= 1e-5 * b
    mean, dh, dw = ops.linear_cross_entropy_grad(h, w, t, reduction="sum", dw=torch.full_like(w, 3.0))
    assert abs(float(mean) - sum(want)) <= 1e-5 * sum(want)
    p = [math.exp(12) / total, math.exp(10) / total]
    # dw of a far column: three times its p, less one for the token it is the target of
    for v, q in zip(far, p):
        assert abs(float(dw[v, 0]) - (3 * q - 1)) <= 2.0 ** -7 * abs(3 * q - 1) and (dw[v, 1:] == 0).all()
    assert abs(float(dw[5, 0]) - 3 / total) <= 2.0 ** -6 * 3 / total
    # dh: p . w - w[target]
    s = 12 * p[0] + 10 * p[1]
    for got, b in zip(dh[:, 0].tolist(), (s - 12, s - 10, s)):
        assert abs(got - b) <= 2.0 ** -7 * (s + 12)


def test_clipping_of_one_tensor_past_2_31_elements(ks):
    ops, torch = ks
    n = (1 << 31) + 12345
    g = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    at = torch.tensor([0, 77, (1 << 31) - 1, 1 << 31, n - 1], device="cuda")
    g[at] = 2.0
    norm = ops.GradClipper([g]).clip(1.0)
    assert abs(float(norm) - math.sqrt(20)) <= 1e-5
    assert (g[at].float() - 2 / math.sqrt(20)).abs().max() <= 2.0 ** -8 and float(g.count_nonzero()) == 5


def _step(ops, tokens, targets, table, w, grad, outs, clipper):
    h = ops.embedding(tokens, table, scale=3.0)
    loss, dh, _ = ops.linear_cross_entropy_grad(h, w, targets, dw=grad[1])
    ops.embedding_backward(tokens, dh, table.shape[0], scale=3.0, dtable=grad[0])
    return loss, clipper.clip(0.5)


@pytest.mark.parametrize("n", [40, 700, 5000])
def test_a_captured_step_replays(ks, n):
    """The whole step in a CUDA graph gives the bits of the eager calls, on new
    inputs too."""
    ops, torch = ks
    gen = torch.Generator(device="cuda")
    gen.manual_seed(n)
    table, w = [torch.randn(900, 136, generator=gen, device="cuda").bfloat16() for _ in range(2)]
    tokens, targets = [torch.randint(0, 900, (n,), generator=gen, device="cuda") for _ in range(2)]
    grad = [torch.empty_like(table), torch.empty_like(w)]
    outs = [torch.empty_like(g) for g in grad]
    clipper = ops.GradClipper(grad, out=outs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(ops, tokens, targets, table, w, grad, outs, clipper)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = _step(ops, tokens, targets, table, w, grad, outs, clipper)
    for seed in (1, 2):
        gen.manual_seed(seed)
        tokens.copy_(torch.randint(0, 900, (n,), generator=gen, device="cuda"))
        targets.copy_(torch.randint(0, 900, (n,), generator=gen, device="cuda"))
        graph.replay()
        got = [x.clone() for x in (*captured, *grad, *outs)]
        want = [*_step(ops, tokens, targets, table, w, grad, outs, clipper), *grad, *outs]
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_streams_at_once(ks):
    """Calls on two streams with their own inputs do not disturb one another."""
    ops, torch = ks
    gen = torch.Generator(device="cuda")
    gen.manual_seed(3)
    work = []
    for k in range(2):
        table, w = [torch.randn(3000, 256, generator=gen, device="cuda").half() for _ in range(2)]
        tokens, targets = [torch.randint(0, 3000, (6000,), generator=gen, device="cuda") for _ in range(2)]
        work.append((tokens, targets, table, w))

    def run(k, stream):
        tokens, targets, table, w = work[k]
        h = ops.embedding(tokens, table, stream=stream)
        loss, dh, dw = ops.linear_cross_entropy_grad(h, w, targets, stream=stream)
        return loss, dw, ops.embedding_backward(tokens, dh, 3000, stream=stream)

    want = [run(0, None), run(1, None)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(10):
        for k in range(2):
            got[k].append(run(k, streams[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for r in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(r, want[k]))
