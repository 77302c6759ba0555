"""CPU: the training operators' C ABI without a GPU -- refusals before any CUDA
call, workspace sizes, the clipping plan -- and the Python checks."""

from __future__ import annotations

import ctypes as C

import pytest
import torch


@pytest.fixture(scope="module")
def N():
    from kernscope_b200 import native

    return native


def _ce(N, **kw):
    a = N.LinearCeArgs(0x1000, 0x2000, 0x3000, 100, 64, 1000, 64, 64, N.KS_BF16, N.KS_CE_GRAD, N.KS_CE_MEAN, 1.0, -100,
                       None, 0x4000, None, 0x5000, 0x6000, 64, 64, None, 0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_linear_ce_validate(N):
    ok = N.LinearCeConfig(0, 0, 0)
    assert N.validate("linear_ce", ok, _ce(N)) == (0, "")
    for cfg in (N.LinearCeConfig(256, 256, 256), N.LinearCeConfig(128, 256, 512), N.LinearCeConfig(128, 128, 0)):
        assert N.validate("linear_ce", cfg, _ce(N))[0] == 0
    for cfg in (N.LinearCeConfig(128, 0, 0), N.LinearCeConfig(256, 128, 0), N.LinearCeConfig(64, 64, 0),
                N.LinearCeConfig(0, 0, 100), N.LinearCeConfig(0, 0, -256)):
        st, reason = N.validate("linear_ce", cfg, _ce(N))
        assert st == N.KS_ERR_INVALID_CONFIG and reason
    for kw, want in [(dict(tokens=0), N.KS_ERR_INVALID_ARGS), (dict(dim=-1), N.KS_ERR_INVALID_ARGS),
                     (dict(vocab=1 << 31), N.KS_ERR_INVALID_ARGS), (dict(h_stride=63), N.KS_ERR_INVALID_ARGS),
                     (dict(dw_stride=63), N.KS_ERR_INVALID_ARGS), (dict(dtype=N.KS_F32), N.KS_ERR_INVALID_CONFIG),
                     (dict(ce_pass=3), N.KS_ERR_INVALID_CONFIG), (dict(reduction=5), N.KS_ERR_INVALID_CONFIG),
                     (dict(reduction=N.KS_CE_NONE), N.KS_ERR_INVALID_CONFIG)]:
        st, reason = N.validate("linear_ce", ok, _ce(N, **kw))
        assert st == want and reason, kw


def test_linear_ce_launch_refuses_before_any_cuda_call(N):
    cfg = N.LinearCeConfig(0, 0, 0)
    f = N.lib.ks_linear_ce_launch
    assert f(None, C.byref(_ce(N)), None) == N.KS_ERR_INVALID_ARGS
    assert f(C.byref(cfg), None, None) == N.KS_ERR_INVALID_ARGS
    for kw in (dict(h=None), dict(w=None), dict(targets=None), dict(loss=None), dict(dh=None), dict(dw=None),
               dict(h=0x1001), dict(targets=0x3004), dict(loss=0x4002), dict(ce_pass=N.KS_CE_BACKWARD)):
        assert f(C.byref(cfg), C.byref(_ce(N, **kw)), None) == N.KS_ERR_INVALID_ARGS, kw
    assert f(C.byref(cfg), C.byref(_ce(N)), None) == N.KS_ERR_WORKSPACE
    assert f(C.byref(cfg), C.byref(_ce(N, workspace=0x10010, workspace_bytes=1 << 30)), None) == N.KS_ERR_WORKSPACE


@pytest.mark.parametrize("tokens,dim,vocab", [(1, 1, 1), (16, 1024, 32000), (333, 1001, 10007), (8192, 4096, 131072),
                                              (100000, 64, 257)])
def test_linear_ce_workspace(N, tokens, dim, vocab):
    """least <= what a limit gives <= max(limit, least); a workspace of that size is accepted as planned."""
    cfg = N.LinearCeConfig(0, 0, 0)
    least, want = C.c_size_t(0), C.c_size_t(0)
    for ce_pass in (N.KS_CE_FORWARD, N.KS_CE_BACKWARD, N.KS_CE_GRAD):
        a = _ce(N, tokens=tokens, dim=dim, vocab=vocab, h_stride=dim, w_stride=dim, dh_stride=dim, dw_stride=dim,
                ce_pass=ce_pass)
        for limit in (0, 1 << 20, 1 << 26, 1 << 32):
            assert N.lib.ks_linear_ce_workspace_bytes(C.byref(cfg), C.byref(a), limit, C.byref(least), C.byref(want)) == 0
            assert 0 < least.value <= want.value <= max(limit, least.value)
    # forward keeps a few bytes per token and tile, never the logits
    a.ce_pass = N.KS_CE_FORWARD
    N.lib.ks_linear_ce_workspace_bytes(C.byref(cfg), C.byref(a), 1 << 40, C.byref(least), C.byref(want))
    packed = 2 * (dim + 8) * (tokens + vocab) if dim % 8 else 0
    assert want.value - packed <= 8192 + (tokens + 256) * (16 + 8 * (vocab // 64 + 4))


def test_embedding_refuses_before_any_cuda_call(N):
    def lookup(**kw):
        a = N.EmbeddingArgs(0x1000, 10, 0x2000, 0x3000, 100, 64, 64, 64, N.KS_BF16, 1.0)
        for k, v in kw.items():
            setattr(a, k, v)
        return N.lib.ks_embedding_launch(C.byref(a), None)

    assert N.lib.ks_embedding_launch(None, None) == N.KS_ERR_INVALID_ARGS
    for kw in (dict(tokens=None), dict(table=None), dict(out=None), dict(tokens_count=0), dict(dim=0), dict(vocab=-1),
               dict(table_stride=63), dict(out_stride=1), dict(tokens=0x1004), dict(table=0x2001)):
        assert lookup(**kw) == N.KS_ERR_INVALID_ARGS, kw
    assert lookup(dtype=N.KS_F64) == N.KS_ERR_INVALID_CONFIG

    def grad(cfg=N.EmbeddingGradConfig(0), **kw):
        a = N.EmbeddingGradArgs(0x1000, 10, 0x2000, 0x3000, 100, 64, 64, 64, N.KS_BF16, N.KS_F32, 0, 1.0, -1, None, 0)
        for k, v in kw.items():
            setattr(a, k, v)
        return N.lib.ks_embedding_grad_launch(C.byref(cfg), C.byref(a), None)

    for kw in (dict(tokens=None), dict(dout=None), dict(dtable=None), dict(tokens_count=-1), dict(dout_stride=8),
               dict(dtable=0x3002)):
        assert grad(**kw) == N.KS_ERR_INVALID_ARGS, kw
    assert grad(dtype=N.KS_F32, out_dtype=N.KS_BF16) == N.KS_ERR_INVALID_CONFIG
    assert grad(N.EmbeddingGradConfig(2000)) == N.KS_ERR_INVALID_CONFIG
    assert grad() == N.KS_ERR_WORKSPACE


def _plan(N, sizes, dtype, base=0x10000, out=None):
    t = (N.GradTensor * max(1, len(sizes)))()
    for i, n in enumerate(sizes):
        t[i] = N.GradTensor(base + i * (1 << 24), out, n, dtype)
    size, chunks = C.c_size_t(0), C.c_int64(0)
    assert N.lib.ks_grad_clip_plan(t, len(sizes), None, 0, C.byref(size), C.byref(chunks)) == 0
    blob = (C.c_ubyte * max(1, size.value))()
    assert N.lib.ks_grad_clip_plan(t, len(sizes), blob, size.value, C.byref(size), C.byref(chunks)) == 0
    rows = [(int.from_bytes(bytes(blob[i:i + 8]), "little"), int.from_bytes(bytes(blob[i + 16:i + 20]), "little"))
            for i in range(0, size.value, 32)]
    return t, rows, chunks.value, size.value


@pytest.mark.parametrize("offset", [0, 2, 6, 14])
def test_grad_clip_plan_covers_every_element_once(N, offset):
    sizes = [1, 0, 7, 16384, 16385, 16383, 50_000]
    t, rows, chunks, size = _plan(N, sizes, N.KS_BF16, 0x10000 + offset)
    assert chunks == len(rows) and size == 32 * chunks
    at = iter(rows)
    for tensor, n in zip(t, sizes):
        p, left = tensor.grad, n
        while left:
            q, count = next(at)
            assert q == p and 0 < count <= 16384 and (p == tensor.grad or p % 16 == 0)
            p, left = p + 2 * count, left - count
    assert next(at, None) is None


def test_grad_clip_refuses(N):
    size, chunks = C.c_size_t(0), C.c_int64(0)
    bad = lambda t: N.lib.ks_grad_clip_plan(C.byref(t), 1, None, 0, C.byref(size), C.byref(chunks))  # noqa: E731
    assert bad(N.GradTensor(0x1001, None, 4, N.KS_BF16)) == N.KS_ERR_INVALID_ARGS
    assert bad(N.GradTensor(None, None, 4, N.KS_BF16)) == N.KS_ERR_INVALID_ARGS
    assert bad(N.GradTensor(0x1000, None, -1, N.KS_BF16)) == N.KS_ERR_INVALID_ARGS
    assert bad(N.GradTensor(0x1000, None, 4, N.KS_F64)) == N.KS_ERR_INVALID_CONFIG
    t = N.GradTensor(0x1000, None, 40000, N.KS_F32)
    blob = (C.c_ubyte * 32)()
    assert N.lib.ks_grad_clip_plan(C.byref(t), 1, blob, 32, C.byref(size), C.byref(chunks)) == N.KS_ERR_WORKSPACE
    a = N.GradClipArgs(0x1000, 1, 1.0, 1e-6, 0x2000, 0x3000, 64)
    assert N.lib.ks_grad_clip_launch(None, None) == N.KS_ERR_INVALID_ARGS
    for kw, want in [(dict(norm=None), N.KS_ERR_INVALID_ARGS), (dict(table=None), N.KS_ERR_INVALID_ARGS),
                     (dict(table=0x1010), N.KS_ERR_INVALID_ARGS), (dict(max_norm=-1.0), N.KS_ERR_INVALID_ARGS),
                     (dict(max_norm=float("nan")), N.KS_ERR_INVALID_ARGS), (dict(workspace=None), N.KS_ERR_WORKSPACE),
                     (dict(workspace_bytes=8), N.KS_ERR_WORKSPACE)]:
        b = N.GradClipArgs.from_buffer_copy(a)
        for k, v in kw.items():
            setattr(b, k, v)
        assert N.lib.ks_grad_clip_launch(C.byref(b), None) == want, kw


def test_python_front_end_refuses_cpu_tensors(N, monkeypatch):
    from kernscope_b200 import ops

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    h, w, t = torch.zeros(4, 8).bfloat16(), torch.zeros(10, 8).bfloat16(), torch.zeros(4, dtype=torch.int64)
    for call in (lambda: ops.linear_cross_entropy(h, w, t), lambda: ops.linear_cross_entropy_grad(h, w, t),
                 lambda: ops.linear_cross_entropy_backward(h, w, t, torch.zeros(4)), lambda: ops.embedding(t, w),
                 lambda: ops.embedding_backward(t, h, 10), lambda: ops.GradClipper([h])):
        with pytest.raises(ValueError):
            call()
