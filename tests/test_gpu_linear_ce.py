"""GPU: linear cross entropy (loss, log-sum-exp and gradients) against the
formulas in 64 bits.

Bounds, per element, from the arithmetic the kernels do (u = half a unit in
the last place of the inputs' type, 2^-8 bf16 / 2^-11 fp16; e = 2^-24 fp32):

* a logit is an fp32 sum of dim exact products: |error| <= 2 dim e |h|.|w|
  (the factor 2 for accumulators that truncate);
* lse adds the exponentials' and the logarithm's own error, a few e of the
  magnitudes involved: 32 e (1 + |lse| + max |l|);
* d = f (exp(l - lse) - 1) is rounded to 16 bits, p once before that where the
  call keeps exponentials (2 u in all), and multiplied in fp32:
  |error of dh| <= (2 u + 2 x error of a logit + 2 n e) |d|.|w| + u |dh|, n the
  length of the sum; dw the same with |d|^T.|h|.  |d| is taken as
  f (p + [v == t]): the subtraction's operands.  fp16 adds its smallest
  steps: 2^-25 / 1024 per d, 2^-25 per output (with the scale of the loss).
"""

from __future__ import annotations

import ctypes as C
import math

import pytest

pytestmark = pytest.mark.gpu

IGNORE = -100
E = 2.0 ** -24


@pytest.fixture(scope="module")
def ks(cuda_ok):
    import torch

    from kernscope_b200 import native, ops

    torch.cuda.set_device(0)
    return native, ops, torch


def _dt(torch, name):
    return {"bf16": torch.bfloat16, "fp16": torch.float16}[name]


def _cfg(N, tile, piece=0):
    tile_m, tile_n = tile if isinstance(tile, tuple) else (tile, tile)
    return N.LinearCeConfig(tile_m, tile_n, piece)


def _make(torch, n, dim, vocab, dtype, seed=0, h_pad=0, w_pad=0, lean=6.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    w = (torch.randn(vocab, dim + w_pad, generator=g, device="cuda") / math.sqrt(dim)).to(dtype)
    t = torch.randint(0, vocab, (n,), generator=g, device="cuda")
    h = torch.randn(n, dim + h_pad, generator=g, device="cuda")
    h[:, :dim] += lean * torch.rand(n, 1, generator=g, device="cuda") * w[t][:, :dim].float()
    t[torch.rand(n, generator=g, device="cuda") < 0.1] = IGNORE
    return h.to(dtype)[:, :dim], w[:, :dim], t


def _exact(torch, h, w, t, f=None):
    """lse, loss, valid and (with the rows' factors f) dh, dw with their bounds' terms."""
    hd, wd = h.double(), w.double()
    l = hd @ wd.t()
    lse = torch.logsumexp(l, 1)
    valid = t != IGNORE
    at = t.clamp(min=0)
    rows = torch.arange(len(t), device="cuda")
    loss = torch.where(valid, lse - l[rows, at], torch.zeros_like(lse))
    lerr = 2 * h.shape[1] * E * (hd.abs() @ wd.abs().t()).max(1).values
    lse_tol = lerr + 32 * E * (1 + lse.abs() + l.abs().max(1).values)
    out = dict(lse=lse, loss=loss, valid=valid, lse_tol=lse_tol, loss_tol=2 * lse_tol)
    if f is not None:
        f = f.double() * valid
        p = (l - lse[:, None]).exp()
        hot = torch.zeros_like(p)
        hot[rows, at] = 1
        d = (p - hot) * f[:, None]
        mag = (p + hot) * f.abs()[:, None]
        fp16 = h.dtype == torch.float16
        u = 2.0 ** -11 if fp16 else 2.0 ** -8
        step = (2.0 ** -25 / 1024 if fp16 else 0.0) * f.abs().max()
        rel = 2 * u + 2 * lse_tol[:, None]
        out["dh"], out["dw"] = d @ wd, d.t() @ hd
        tiny = 2.0 ** -25 if fp16 else 0.0
        out["dh_tol"] = (rel + 2 * w.shape[0] * E) * (mag @ wd.abs()) + step * wd.abs().sum(0) + u * out["dh"].abs() + tiny
        out["dw_tol"] = (((rel + 2 * h.shape[0] * E) * mag).t() @ hd.abs() + step * hd.abs().sum(0) + u * out["dw"].abs()
                         + tiny)
    return out


def _near(torch, got, want, tol, name):
    got = got.double()
    assert got.shape == want.shape
    off = (got - want).abs() - tol
    assert torch.isfinite(got).all(), f"{name}: not finite"
    worst = int(off.argmax())
    assert off.max() <= 0, f"{name}: {got.flatten()[worst]} for {want.flatten()[worst]}, tolerance {tol.flatten()[worst]}"


def _dirty(torch, n):
    """Scratch whose every 16- and 32-bit value is NaN."""
    return torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda")


SHAPES = [  # tokens, dim, vocab: one of each, tile edges, odd, long rows, more tiles than SMs at 128
    (1, 1, 1), (1, 64, 2), (2, 8, 33), (127, 63, 127), (128, 64, 128), (129, 65, 129), (255, 200, 257), (256, 512, 256),
    (257, 264, 1000), (300, 130, 2500), (3, 1024, 5003), (700, 72, 4099), (1100, 1001, 515), (16, 4096, 300),
    (2100, 1300, 9000),  # more items of dh than the SMs take in one round, an uneven rest
]


@pytest.mark.parametrize("tile", [0, 128, (128, 256), 256])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_loss_and_gradients(ks, shape, dtype, tile):
    N, ops, torch = ks
    n, dim, vocab = shape
    h, w, t = _make(torch, n, dim, vocab, _dt(torch, dtype), seed=n + dim + vocab)
    cfg = _cfg(N, tile)
    count = max(1, int((t != IGNORE).sum()))
    ref = _exact(torch, h, w, t, torch.full((n,), 1.0 / count, device="cuda"))
    loss, lse = ops.linear_cross_entropy(h, w, t, cfg=cfg)
    _near(torch, lse, ref["lse"], ref["lse_tol"], "lse")
    _near(torch, loss, ref["loss"], ref["loss_tol"], "loss")
    assert (loss[~ref["valid"]] == 0).all()
    nan = lambda x: torch.full(x.shape, float("nan"), dtype=x.dtype, device="cuda")  # noqa: E731
    mean, dh, dw = ops.linear_cross_entropy_grad(h, w, t, dh=nan(h), dw=nan(w), cfg=cfg)
    _near(torch, mean, ref["loss"].sum().reshape(1) / count, (ref["loss_tol"].sum() / count + E * ref["loss"].sum()).reshape(1),
          "mean")
    _near(torch, dh, ref["dh"], ref["dh_tol"], "dh")
    _near(torch, dw, ref["dw"], ref["dw_tol"], "dw")
    assert ops.device_error_take() == 0


@pytest.mark.parametrize("tile", [128, (128, 256), 256])
@pytest.mark.parametrize("h_pad,w_pad", [(0, 0), (8, 16), (3, 0), (0, 5), (1, 1)])
def test_strides_and_output_rows(ks, h_pad, w_pad, tile):
    """Row strides of inputs and outputs, those TMA cannot address among them;
    nothing is written between the outputs' rows."""
    N, ops, torch = ks
    n, dim, vocab = 150, 120, 700
    h, w, t = _make(torch, n, dim, vocab, torch.bfloat16, seed=5, h_pad=h_pad, w_pad=w_pad)
    dh_all = torch.full((n, dim + h_pad), 7.0, dtype=torch.bfloat16, device="cuda")
    dw_all = torch.full((vocab, dim + w_pad), 7.0, dtype=torch.bfloat16, device="cuda")
    ref = _exact(torch, h, w, t, torch.ones(n, device="cuda"))
    cfg = _cfg(N, tile, 256)  # three pieces
    loss, dh, dw = ops.linear_cross_entropy_grad(h, w, t, reduction="sum", dh=dh_all[:, :dim], dw=dw_all[:, :dim], cfg=cfg)
    _near(torch, dh, ref["dh"], ref["dh_tol"], "dh")
    _near(torch, dw, ref["dw"], ref["dw_tol"], "dw")
    assert (dh_all[:, dim:] == 7).all() and (dw_all[:, dim:] == 7).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("offset", [1, 4])
def test_unaligned_bases(ks, dtype, offset):
    """Tensors that begin at any multiple of their element size."""
    N, ops, torch = ks
    n, dim, vocab, dt = 40, 64, 300, _dt(torch, dtype)
    h0, w0, t = _make(torch, n, dim, vocab, dt, seed=9)

    def shifted(x):
        flat = torch.empty(x.numel() + offset, dtype=dt, device="cuda")
        y = flat[offset:].view(x.shape)
        return y.copy_(x)

    h, w = shifted(h0.contiguous()), shifted(w0.contiguous())
    dh, dw = shifted(torch.zeros_like(h)), shifted(torch.zeros_like(w))
    ref = _exact(torch, h, w, t, torch.ones(n, device="cuda"))
    ops.linear_cross_entropy_grad(h, w, t, reduction="sum", dh=dh, dw=dw)
    _near(torch, dh, ref["dh"], ref["dh_tol"], "dh")
    _near(torch, dw, ref["dw"], ref["dw_tol"], "dw")


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
@pytest.mark.parametrize("piece", [0, 256, 512])
def test_backward_with_incoming_gradient(ks, reduction, dtype, piece):
    N, ops, torch = ks
    n, dim, vocab = 200, 96, 1111
    h, w, t = _make(torch, n, dim, vocab, _dt(torch, dtype), seed=11)
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    _, lse = ops.linear_cross_entropy(h, w, t)
    if reduction == "none":
        dloss = torch.randn(n, generator=g, device="cuda")
        f = dloss * 0.5
    else:
        dloss = torch.full((1,), 3.0, device="cuda")
        f = torch.full((n,), 1.5, device="cuda") / (int((t != IGNORE).sum()) if reduction == "mean" else 1)
    ref = _exact(torch, h, w, t, f)
    cfg = _cfg(N, 0, piece)
    dh, dw = ops.linear_cross_entropy_backward(h, w, t, lse, dloss, reduction=reduction, grad_scale=0.5, cfg=cfg)
    _near(torch, dh, ref["dh"], ref["dh_tol"], "dh")
    _near(torch, dw, ref["dw"], ref["dw_tol"], "dw")
    ones = torch.ones(n if reduction == "none" else 1, device="cuda")
    a = ops.linear_cross_entropy_backward(h, w, t, lse, ones, reduction=reduction)
    b = ops.linear_cross_entropy_backward(h, w, t, lse, None, reduction=reduction)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_large_and_small_incoming_gradients_keep_fp16_range(ks):
    """dloss of 1e4 and 1e-4 (a loss scale and its inverse): the rows' factors
    are taken out of the 16-bit d by a power of two."""
    N, ops, torch = ks
    n, dim, vocab = 64, 64, 500
    h, w, t = _make(torch, n, dim, vocab, torch.float16, seed=2)
    _, lse = ops.linear_cross_entropy(h, w, t)
    base = ops.linear_cross_entropy_backward(h, w, t, lse, torch.ones(n, device="cuda"))[1].double()
    for k in (10, -10):
        dloss = torch.full((n,), 2.0 ** k, device="cuda")
        dw = ops.linear_cross_entropy_backward(h, w, t, lse, dloss, grad_scale=2.0 ** -k)[1]
        assert torch.equal(dw.double(), base)  # powers of two change no rounding


@pytest.mark.parametrize("tile", [128, (128, 256), 256])
def test_workspace_least_and_dirty(ks, tile):
    """The least workspace, full of NaN: the same loss, and gradients within the
    bounds (more pieces, another order of the sum)."""
    N, ops, torch = ks
    n, dim, vocab = 333, 160, 3000
    h, w, t = _make(torch, n, dim, vocab, torch.bfloat16, seed=21)
    cfg = _cfg(N, tile)
    a = ops._linear_ce_args(h, w, t, N.KS_CE_GRAD, "sum", IGNORE)
    least, want = ops.linear_cross_entropy_workspace_bytes(a, cfg)
    assert least < want
    ref = _exact(torch, h, w, t, torch.ones(n, device="cuda"))
    got = []
    for size in (least, (least + want) // 2, want, want + 4096):
        loss, dh, dw = ops.linear_cross_entropy_grad(h, w, t, reduction="sum", cfg=cfg, workspace=_dirty(torch, size))
        _near(torch, dh, ref["dh"], ref["dh_tol"], "dh")
        _near(torch, dw, ref["dw"], ref["dw_tol"], "dw")
        got.append(float(loss))
    assert len(set(got)) == 1
    with pytest.raises(N.KsError) as e:
        ops.linear_cross_entropy_grad(h, w, t, reduction="sum", cfg=cfg, workspace=_dirty(torch, least - 1))
    assert e.value.status == N.KS_ERR_WORKSPACE


@pytest.mark.parametrize("tile", [128, (128, 256), 256])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_loss_of_one_large_logit(ks, dtype, tile):
    """Logits of a few hundred, targets with probability near one: the loss is a
    difference of nearly equal numbers and stays within the bound of an fp32 dot
    product, the target's logit being the same number in both."""
    N, ops, torch = ks
    n, dim, vocab = 64, 2048, 1000
    h, w, t = _make(torch, n, dim, vocab, _dt(torch, dtype), seed=31, lean=300.0)
    loss, lse = ops.linear_cross_entropy(h, w, t, cfg=_cfg(N, tile))
    ref = _exact(torch, h, w, t)
    _near(torch, lse, ref["lse"], ref["lse_tol"], "lse")
    valid = ref["valid"]
    # dot product: at most dim / 256 + 13 additions deep
    tol = 32 * E * (1 + ref["lse"].abs()) + 24 * E * (h.double().abs() * w.double().abs()[t.clamp(min=0)]).sum(1)
    _near(torch, loss[valid], ref["loss"][valid], 2 * tol[valid], "loss")


def test_no_token_counts(ks):
    N, ops, torch = ks
    h, w, _ = _make(torch, 70, 64, 300, torch.bfloat16)
    t = torch.full((70,), IGNORE, device="cuda")
    h[3] = float("nan")  # an ignored row's values reach nothing but its own lse
    h[4, 5] = float("inf")
    for reduction in ("mean", "sum"):
        loss, dh, dw = ops.linear_cross_entropy_grad(h, w, t, reduction=reduction)
        assert float(loss) == 0 and (dh == 0).all()
    clean = torch.ones(70, dtype=torch.bool, device="cuda")
    clean[3:5] = False
    _, dh, dw = ops.linear_cross_entropy_grad(h[clean].contiguous(), w, t[clean].contiguous())
    assert (dh == 0).all() and (dw == 0).all()
    loss, lse = ops.linear_cross_entropy(h, w, t)
    assert (loss == 0).all() and torch.isfinite(lse[clean]).all() and torch.isnan(lse[3])


def test_target_out_of_range_and_other_ignore_index(ks):
    N, ops, torch = ks
    h, w, _ = _make(torch, 6, 64, 300, torch.bfloat16)
    t = torch.tensor([0, 299, 300, -1, 7, 7], device="cuda")
    loss, lse = ops.linear_cross_entropy(h, w, t, ignore_index=7)
    assert torch.isfinite(loss[:2]).all() and torch.isnan(loss[2:4]).all() and (loss[4:] == 0).all()
    total, dh, dw = ops.linear_cross_entropy_grad(h, w, t, ignore_index=7, reduction="sum")
    assert torch.isnan(total).all()
    assert torch.isfinite(dh.float()).all() and (dh[2:] == 0).all() and torch.isfinite(dw.float()).all()


def test_infinities_and_extreme_logits(ks):
    """Logits of -inf drop out; a row of -inf alone, +inf and NaN end in NaN or
    -inf as the formula does; logits near 1e4 neither overflow nor lose the sum."""
    N, ops, torch = ks
    dim, vocab = 64, 300
    h = torch.zeros(5, dim, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(vocab, dim, dtype=torch.bfloat16, device="cuda")
    h[:, 0] = 1
    w[:, 0] = torch.arange(vocab, device="cuda").remainder(5).to(torch.bfloat16)
    w[100:, 1] = float("-inf")
    h[0, 1] = 1  # columns from 100 on are -inf in row 0; in the others 0 * -inf = NaN
    t = torch.zeros(5, dtype=torch.int64, device="cuda")
    loss, lse = ops.linear_cross_entropy(h, w, t)
    want = torch.logsumexp(w[:100, 0].double(), 0)
    assert abs(float(lse[0]) - float(want)) < 1e-5 and torch.isnan(lse[1:]).all()
    w[:, 1] = float("-inf")
    assert float(ops.linear_cross_entropy(h[:1], w, t[:1])[1]) == float("-inf")
    w[:, 1] = 0
    w[:, 0] *= 2500
    loss, lse = ops.linear_cross_entropy(h, w, t)
    want = torch.logsumexp(w[:, 0].double(), 0)
    assert (lse.double() - want).abs().max() <= 32 * E * 3 * 1e4 and torch.isfinite(loss).all()
    w[7, 0] = float("inf")
    assert torch.isnan(ops.linear_cross_entropy(h, w, t)[0]).all()


def test_same_bits_every_time_and_on_another_stream(ks):
    N, ops, torch = ks
    h, w, t = _make(torch, 400, 256, 2000, torch.bfloat16, seed=4)
    first = ops.linear_cross_entropy_grad(h, w, t)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for stream in (None, s, s):
        got = ops.linear_cross_entropy_grad(h, w, t, stream=stream)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(first, got))


@pytest.mark.parametrize("piece", [0, 256])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("n", [1, 2, 5, 33, 64])
def test_few_tokens_keep_the_targets_residual(ks, n, dtype, piece):
    """With few tokens dw's rows are single terms, and the rounding of the target's
    d would be that of the whole row; its residual is carried, so dh and dw are
    within their own rounding, at most u / sqrt(3) in the 2-norm where errors are
    spread evenly within half a unit (0.62 u leaves 7 % for the sample), plus what the other probabilities' two
    roundings (2 u each, of sum p^2 against the target's (1 - p)^2) and 8 e of fp32
    add.  Several tokens share a target."""
    N, ops, torch = ks
    h, w, t = _make(torch, n, 264, 1500, _dt(torch, dtype), seed=40 + n, lean=3.0)
    t = torch.where(t == IGNORE, t, t % 7 * 211)
    t[0] = 211
    ref = _exact(torch, h, w, t, torch.ones(n, device="cuda"))
    _, dh, dw = ops.linear_cross_entropy_grad(h, w, t, reduction="sum", cfg=_cfg(N, 0, piece))
    u = 2.0 ** -8 if dtype == "bf16" else 2.0 ** -11
    p = ((h.double() @ w.double().t()) - ref["lse"][:, None]).exp()[t != IGNORE]
    others = p.clone()
    others[torch.arange(len(p)), t[t != IGNORE]] = 0
    spread = float(others.norm() / (1 - p[torch.arange(len(p)), t[t != IGNORE]]).norm())
    for got, want in ((dh, ref["dh"]), (dw, ref["dw"])):
        assert float((got.double() - want).norm() / want.norm()) <= (0.62 + 3 * spread) * u


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_gradients_against_differences(ks, dtype):
    """Central differences of the kernel's own loss along random +-1 steps of a
    size the type holds exactly.  With |step| = 2^-6 on values below 4 the
    third-order term is below (2^-6)^2 relative to the slope times the spread
    of the logits' change; 3 % covers it and the 16-bit rounding of the
    gradient (random, over thousands of elements)."""
    N, ops, torch = ks
    dt = _dt(torch, dtype)
    n, dim, vocab = 24, 64, 150
    g = torch.Generator(device="cuda")
    g.manual_seed(8)
    grid = 2.0 ** -5  # values and steps on a grid that bf16 holds below 4
    rnd = lambda *s: (torch.randn(*s, generator=g, device="cuda").clamp(-3, 3) / grid).round().mul(grid)  # noqa: E731
    h, w = rnd(n, dim), rnd(vocab, dim) * 0.25
    t = torch.randint(0, vocab, (n,), generator=g, device="cuda")
    loss, dh, dw = ops.linear_cross_entropy_grad(h.to(dt), w.to(dt), t, reduction="sum")
    for which in ("h", "w"):
        x, dx, step = (h, dh, 2 * grid) if which == "h" else (w, dw, grid / 2)
        # along the gradient's signs, so that the slope is far from zero
        delta = torch.sign(dx.float()) * step
        keep = (x.to(dt).float() + delta).to(dt).float() - delta == x.to(dt).float()
        keep &= (x.to(dt).float() - delta).to(dt).float() + delta == x.to(dt).float()
        small = dx.float().abs() > dx.float().abs().median()
        pick = torch.rand(x.shape, generator=g, device="cuda") < 0.02
        delta = torch.where(keep & small & pick, delta, torch.zeros_like(delta))
        assert (delta != 0).sum() > 5
        plus, minus = (x + delta).to(dt), (x - delta).to(dt)
        args = lambda y: (y, w.to(dt)) if which == "h" else (h.to(dt), y)  # noqa: E731
        lp = ops.linear_cross_entropy(*args(plus), t, reduction="none")[0].double().sum()
        lm = ops.linear_cross_entropy(*args(minus), t, reduction="none")[0].double().sum()
        slope = (dx.double() * (plus.double() - minus.double())).sum()
        assert abs(float(lp - lm) - float(slope)) <= 0.03 * abs(float(slope))


def test_no_tokens(ks):
    N, ops, torch = ks
    h, w, t = _make(torch, 4, 64, 100, torch.bfloat16)
    loss, lse = ops.linear_cross_entropy(h[:0], w, t[:0])
    assert loss.numel() == 0 and lse.numel() == 0
    loss, dh, dw = ops.linear_cross_entropy_grad(h[:0], w, t[:0])
    assert float(loss) == 0 and dh.shape == (0, 64) and (dw == 0).all()


def test_refusals(ks):
    N, ops, torch = ks
    h, w, t = _make(torch, 8, 64, 100, torch.bfloat16)
    for bad in [
        lambda: ops.linear_cross_entropy(h.cpu(), w, t),
        lambda: ops.linear_cross_entropy(h.float(), w, t),
        lambda: ops.linear_cross_entropy(h, w.half(), t),
        lambda: ops.linear_cross_entropy(h[:, :32], w, t),
        lambda: ops.linear_cross_entropy(h.t(), w, t),
        lambda: ops.linear_cross_entropy(h[:, ::2], w[:, ::2], t),
        lambda: ops.linear_cross_entropy(h[:1].expand(8, 64), w, t),
        lambda: ops.linear_cross_entropy(h, w, t.int()),
        lambda: ops.linear_cross_entropy(h, w, t[:7]),
        lambda: ops.linear_cross_entropy(h, w, t, reduction="max"),
        lambda: ops.linear_cross_entropy_grad(h, w, t, reduction="none"),
        lambda: ops.linear_cross_entropy_grad(h, w, t, dh=h.half()),
        lambda: ops.linear_cross_entropy_grad(h, w, t, dw=w[:50]),
        lambda: ops.linear_cross_entropy_backward(h, w, t, torch.zeros(7, device="cuda")),
        lambda: ops.linear_cross_entropy_backward(h, w, t, torch.zeros(8, device="cuda"), torch.ones(1, device="cuda")),
    ]:
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(N.KsError) as e:
        ops.linear_cross_entropy(h, w, t, cfg=N.LinearCeConfig(256, 128, 0))
    assert e.value.status == N.KS_ERR_INVALID_CONFIG
    with pytest.raises(N.KsError) as e:
        ops.linear_cross_entropy_grad(h, w, t, cfg=_cfg(N, 0, 100))
    assert e.value.status == N.KS_ERR_INVALID_CONFIG
    a = ops._linear_ce_args(h, w, t, N.KS_CE_FORWARD, "none", IGNORE)
    cfg = N.LinearCeConfig()
    assert N.lib.ks_linear_ce_launch(C.byref(cfg), C.byref(a), None) == N.KS_ERR_INVALID_ARGS  # no loss
