"""GPU: embedding lookup and its gradient against the definitions in 64 bits.

The lookup rounds one fp32 product: |error| <= u |value| + the type's smallest
step, u = 2^-8 bf16, 2^-11 fp16, 2^-24 fp32.  The gradient sums n_v rows in
fp32, in a chain whose length is at most n_v, and rounds once more to its type:
|error| <= n_v 2^-24 sum |dout| scale + u |value| + 2^-24 |value| + the step.
"""

from __future__ import annotations

import ctypes as C

import pytest

pytestmark = pytest.mark.gpu

U = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "fp32": 2.0 ** -24}
STEP = {"bf16": 1e-38, "fp16": 2.0 ** -25, "fp32": 1e-38}


@pytest.fixture(scope="module")
def ks(cuda_ok):
    import torch

    from kernscope_b200 import native, ops

    torch.cuda.set_device(0)
    return native, ops, torch


def _dt(torch, name):
    return {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}[name]


def _gen(torch, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _rows(torch, g, n, dim, pad, dtype, offset=0):
    flat = torch.randn(n * (dim + pad) + offset, generator=g, device="cuda").to(dtype)
    return flat[offset:].view(n, dim + pad)[:, :dim]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("shape", [(1, 1, 1), (1, 4096, 7), (3, 8, 100), (64, 2048, 500), (257, 1000, 300),
                                   (1000, 129, 2000), (5, 4100, 11)], ids=str)
@pytest.mark.parametrize("pad,offset", [(0, 0), (8, 0), (3, 1)])
def test_lookup(ks, shape, dtype, pad, offset):
    N, ops, torch = ks
    n, dim, vocab = shape
    g = _gen(torch, n + dim)
    table = _rows(torch, g, vocab, dim, pad, _dt(torch, dtype), offset)
    tokens = torch.randint(-2, vocab + 2, (n,), generator=g, device="cuda")
    scale = 1.7
    full = torch.full((n, dim + pad), 9.0, dtype=table.dtype, device="cuda")
    out = ops.embedding(tokens, table, scale, out=full[:, :dim])
    inside = (tokens >= 0) & (tokens < vocab)
    want = table.double()[tokens.clamp(0, vocab - 1)] * torch.tensor(scale, dtype=torch.float32).double().cuda()
    want[~inside] = 0
    assert ((out.double() - want).abs() <= U[dtype] * want.abs() + STEP[dtype]).all()
    assert (full[:, dim:] == 9).all()


def test_lookup_keeps_values_shape_and_zeros_outside(ks):
    N, ops, torch = ks
    table = torch.randn(10, 64, device="cuda").bfloat16()
    table[0] = float("inf")  # what an outside token must not touch
    tokens = torch.tensor([[1, 2, 3], [9, -1, 10]], device="cuda")
    out = ops.embedding(tokens, table)
    assert out.shape == (2, 3, 64)
    assert torch.equal(out[0], table[1:4]) and torch.equal(out[1, 0], table[9]) and (out[1, 1:] == 0).all()


def _check_grad(torch, got, tokens, dout, vocab, scale, out_name, base=None, padding=-1):
    keep = (tokens >= 0) & (tokens < vocab) & (tokens != padding)
    s = torch.tensor(scale, dtype=torch.float32).double().cuda()
    want = torch.zeros(vocab, dout.shape[1], dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(want)
    many = torch.zeros(vocab, 1, dtype=torch.float64, device="cuda")
    t = tokens[keep]
    want.index_add_(0, t, dout[keep].double())
    mag.index_add_(0, t, dout[keep].double().abs())
    many.index_add_(0, t, torch.ones(len(t), 1, dtype=torch.float64, device="cuda"))
    want *= s
    tol = many * 2.0 ** -24 * mag * s.abs()
    if base is not None:
        want += base.double()
        tol += 2.0 ** -24 * want.abs()
    tol += (U[out_name] + 2.0 ** -24) * (want.abs() + tol) + STEP[out_name]
    assert ((got.double() - want).abs() <= tol).all()
    absent = many[:, 0] == 0
    assert (got[absent] == (0 if base is None else base[absent])).all()


GRAD_SHAPES = [(1, 1, 1), (1, 512, 5), (31, 64, 3), (32, 65, 1), (33, 256, 40), (200, 1001, 50), (777, 264, 5003),
               (4096, 48, 1048575), (4096, 48, 1048576), (4097, 48, 300), (3500, 16, 3000000), (5000, 128, 1023),
               (5000, 40, 1024), (9000, 96, 70000), (12000, 24, 900), (70000, 8, 5), (20000, 72, 1100000)]


@pytest.mark.parametrize("names", [("bf16", "bf16"), ("bf16", "fp32"), ("fp16", "fp16"), ("fp16", "fp32"), ("fp32", "fp32")],
                         ids=lambda v: "-".join(v))
@pytest.mark.parametrize("shape", GRAD_SHAPES, ids=str)
def test_gradient(ks, shape, names):
    N, ops, torch = ks
    n, dim, vocab = shape
    g = _gen(torch, n + vocab)
    dout = _rows(torch, g, n, dim, 0, _dt(torch, names[0]))
    # frequent low tokens, some outside, as many as fit above
    tokens = (torch.rand(n, generator=g, device="cuda") ** 4 * (vocab + 2)).long() - 1
    got = ops.embedding_backward(tokens, dout, vocab, 0.75, dtype=_dt(torch, names[1]))
    assert got.dtype == _dt(torch, names[1])
    _check_grad(torch, got, tokens, dout, vocab, 0.75, names[1])


@pytest.mark.parametrize("chunk", [0, 1, 7, 8, 31, 32, 100, 1024])
@pytest.mark.parametrize("kind", ["one", "two", "few", "sorted", "all different", "edges", "outside"])
def test_runs_and_chunk_edges(ks, kind, chunk):
    """Tokens that fill many chunks, end at chunk edges or inside them."""
    N, ops, torch = ks
    n, dim, vocab = 9001, (136, 1000)[chunk % 4 == 0], 4000
    g = _gen(torch, 1)
    dout = _rows(torch, g, n, dim, 0, torch.bfloat16)
    i = torch.arange(n, device="cuda")
    tokens = {"one": torch.full_like(i, 3999), "two": i % 2, "few": (i * 7919) % 13, "sorted": i // 32,
              "all different": (i * 1009) % 4000, "edges": i // 128 * 2 + (i % 128 >= 8), "outside": torch.full_like(i, 4000)}[kind]
    cfg = N.EmbeddingGradConfig(chunk)
    args = dict(dtype=torch.float32, cfg=cfg)
    got = ops.embedding_backward(tokens, dout, vocab, 1.0, **args)
    _check_grad(torch, got, tokens, dout, vocab, 1.0, "fp32")
    assert torch.equal(got, ops.embedding_backward(tokens, dout, vocab, 1.0, **args))


def test_order_of_the_sum(ks):
    """Equal tokens are added in the order of their positions: with one chunk's
    worth of them the result is the left-to-right fp32 sum, bit for bit."""
    N, ops, torch = ks
    n, dim = 32, 64
    dout = (torch.randn(n, dim, generator=_gen(torch, 2), device="cuda") * 10.0 ** torch.arange(n, device="cuda").remainder(7)[:, None])
    want = torch.zeros(dim, device="cuda")
    for r in dout:
        want = want + r
    got = ops.embedding_backward(torch.full((n,), 5, device="cuda"), dout, 9, cfg=N.EmbeddingGradConfig(32))
    assert torch.equal(got[5], want)


@pytest.mark.parametrize("names", [("bf16", "bf16"), ("bf16", "fp32"), ("fp32", "fp32")], ids=lambda v: "-".join(v))
@pytest.mark.parametrize("pad,offset", [(0, 0), (8, 0), (3, 1)])
def test_accumulate_padding_and_strides(ks, names, pad, offset):
    N, ops, torch = ks
    n, dim, vocab = 900, 200, 333
    g = _gen(torch, 6)
    dout = _rows(torch, g, n, dim, pad, _dt(torch, names[0]), offset)
    tokens = torch.randint(0, vocab, (n,), generator=g, device="cuda")
    full = torch.randn(vocab, dim + pad, generator=g, device="cuda").to(_dt(torch, names[1]))
    base = full.clone()
    ops.embedding_backward(tokens, dout, vocab, 0.5, padding_idx=7, dtable=full[:, :dim], accumulate=True)
    _check_grad(torch, full[:, :dim], tokens, dout, vocab, 0.5, names[1], base=base[:, :dim], padding=7)
    assert torch.equal(full[:, dim:], base[:, dim:]) and torch.equal(full[7], base[7])
    full = base.clone()
    ops.embedding_backward(tokens, dout, vocab, 0.5, padding_idx=7, dtable=full[:, :dim])
    _check_grad(torch, full[:, :dim], tokens, dout, vocab, 0.5, names[1], padding=7)
    assert torch.equal(full[:, dim:], base[:, dim:])


@pytest.mark.parametrize("names", [("bf16", "bf16"), ("fp16", "fp32"), ("fp32", "fp32")], ids=lambda v: "-".join(v))
@pytest.mark.parametrize("dim", [1, 7, 250, 2047, 2056, 4099])
@pytest.mark.parametrize("pad,offset", [(1, 0), (2, 3), (5, 7), (8, 2)])
def test_gradient_of_unaligned_rows(ks, dim, pad, offset, names):
    """Rows at every offset within 16 bytes, one and several segments wide, with
    NaN in all that lies between them."""
    N, ops, torch = ks
    n, vocab = 300, 90
    g = _gen(torch, dim + pad)
    dtype = _dt(torch, names[0])
    flat = torch.full((n * (dim + pad) + offset + 16,), float("nan"), dtype=dtype, device="cuda")
    dout = flat[offset:offset + n * (dim + pad)].view(n, dim + pad)[:, :dim]
    dout.copy_(torch.randn(n, dim, generator=g, device="cuda"))
    tokens = torch.randint(0, vocab, (n,), generator=g, device="cuda")
    got = ops.embedding_backward(tokens, dout, vocab, 2.5, dtype=_dt(torch, names[1]))
    _check_grad(torch, got, tokens, dout, vocab, 2.5, names[1])
    full = torch.full((vocab, dim + 3), 9.0, dtype=_dt(torch, names[1]), device="cuda")
    ops.embedding_backward(tokens, dout, vocab, 2.5, dtable=full[:, :dim])
    assert torch.equal(full[:, :dim], got) and (full[:, dim:] == 9).all()


def test_excluded_rows_may_hold_anything(ks):
    N, ops, torch = ks
    dout = torch.randn(100, 64, device="cuda").bfloat16()
    tokens = torch.arange(100, device="cuda") % 10
    dout[tokens == 4] = float("nan")
    got = ops.embedding_backward(tokens, dout, 10, padding_idx=4)
    assert torch.isfinite(got.float()).all() and (got[4] == 0).all()


def test_large_batch_spans_the_cluster(ks):
    """More than one element per thread of the sorting cluster; a dirty workspace."""
    N, ops, torch = ks
    n, dim, vocab = 300_001, 16, 131072
    g = _gen(torch, 9)
    dout = _rows(torch, g, n, dim, 0, torch.float32)
    tokens = (torch.rand(n, generator=g, device="cuda") ** 6 * vocab).long()
    args = N.EmbeddingGradArgs(tokens_count=n, vocab=vocab, dim=dim, dout_stride=dim, dtable_stride=dim, dtype=N.KS_F32,
                               out_dtype=N.KS_F32)
    need = C.c_size_t(0)
    cfg = N.EmbeddingGradConfig()
    N.check("bytes", N.lib.ks_embedding_grad_workspace_bytes(C.byref(cfg), C.byref(args), C.byref(need)))
    ws = torch.full((need.value,), 0xFF, dtype=torch.uint8, device="cuda")
    got = ops.embedding_backward(tokens, dout, vocab, workspace=ws)
    _check_grad(torch, got, tokens, dout, vocab, 1.0, "fp32")
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    other = ops.embedding_backward(tokens, dout, vocab, stream=s)
    torch.cuda.synchronize()
    assert torch.equal(got, other)
    with pytest.raises(N.KsError) as e:
        ops.embedding_backward(tokens, dout, vocab, workspace=ws[:-256])
    assert e.value.status == N.KS_ERR_WORKSPACE


def test_gradient_against_differences(ks):
    """The lookup is linear in the table: the change of sum(dout * out) along a
    step is the gradient's product with the step, to the roundings of fp32."""
    N, ops, torch = ks
    g = _gen(torch, 12)
    vocab, dim, n = 50, 24, 400
    table = torch.randn(vocab, dim, generator=g, device="cuda")
    step = torch.randn(vocab, dim, generator=g, device="cuda") * 0.5
    dout = torch.randn(n, dim, generator=g, device="cuda")
    tokens = torch.randint(0, vocab, (n,), generator=g, device="cuda")
    grad = ops.embedding_backward(tokens, dout, vocab, scale=2.0)
    f = lambda t: (ops.embedding(tokens, t, scale=2.0).double() * dout.double()).sum()  # noqa: E731
    plus, minus = table + step, table - step
    change, slope = float(f(plus) - f(minus)), float((grad.double() * (plus.double() - minus.double())).sum())
    scale = float((grad.abs().double() * (2 * step).abs().double()).sum())
    assert abs(change - slope) <= n * 2.0 ** -22 * scale


def test_no_tokens_and_refusals(ks):
    N, ops, torch = ks
    table = torch.randn(10, 16, device="cuda")
    tokens = torch.zeros(4, dtype=torch.int64, device="cuda")
    dout = torch.randn(4, 16, device="cuda")
    assert ops.embedding(tokens[:0], table).shape == (0, 16)
    assert (ops.embedding_backward(tokens[:0], dout[:0], 10) == 0).all()
    for bad in [
        lambda: ops.embedding(tokens.int(), table),
        lambda: ops.embedding(tokens.cpu(), table),
        lambda: ops.embedding(tokens, table.cpu()),
        lambda: ops.embedding(tokens, table.double()),
        lambda: ops.embedding(tokens, table.t()),
        lambda: ops.embedding(tokens, table, out=torch.empty(3, 16, device="cuda")),
        lambda: ops.embedding_backward(tokens, dout[:3], 10),
        lambda: ops.embedding_backward(tokens, dout, 10, accumulate=True),
        lambda: ops.embedding_backward(tokens, dout, 10, dtable=torch.empty(9, 16, device="cuda")),
        lambda: ops.embedding_backward(tokens, dout, 10, dtable=torch.empty(10, 16, device="cuda").half()),
        lambda: ops.embedding_backward(tokens, dout.t(), 10),
    ]:
        with pytest.raises(ValueError):
            bad()
    for chunk in (-1, 1025):
        with pytest.raises(N.KsError) as e:
            ops.embedding_backward(tokens, dout, 10, cfg=N.EmbeddingGradConfig(chunk))
        assert e.value.status == N.KS_ERR_INVALID_CONFIG
