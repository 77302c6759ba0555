"""GPU: a second driver context on the same device, as a plugin in a host program
of its own may make: what the library asks the runtime for once belongs to the
context it was asked in."""

from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def N(cuda_ok):
    from kernscope_b200 import native

    return native


def _embedding_gradient(N, n=5000, dim=1024, vocab=37):
    """The gradient of rows of ones (how often each token occurs), with memory of the
    current context; kernels with more shared memory than the default among them."""
    lib, held = N.lib, []

    def device(host_or_bytes):
        p = C.c_void_p()
        size = host_or_bytes if isinstance(host_or_bytes, int) else host_or_bytes.nbytes
        N.check("malloc", lib.ks_gpu_malloc(C.byref(p), size))
        held.append(p)
        if not isinstance(host_or_bytes, int):
            N.check("h2d", lib.ks_gpu_memcpy_htod(p, host_or_bytes.ctypes.data, size, None))
        return p

    tokens = np.arange(n, dtype=np.int64) % vocab
    a = N.EmbeddingGradArgs(device(tokens), n, device(np.ones((n, dim), np.float32)), device(vocab * dim * 4), vocab, dim, dim,
                            dim, N.KS_F32, N.KS_F32, 0, 1.0, -1, None, 0)
    cfg, need = N.EmbeddingGradConfig(0), C.c_size_t(0)
    N.check("bytes", lib.ks_embedding_grad_workspace_bytes(C.byref(cfg), C.byref(a), C.byref(need)))
    a.workspace, a.workspace_bytes = device(need.value).value, need.value
    status = lib.ks_embedding_grad_launch(C.byref(cfg), C.byref(a), None)
    got = np.zeros((vocab, dim), np.float32)
    N.check("sync", lib.ks_gpu_synchronize())
    N.check("d2h", lib.ks_gpu_memcpy_dtoh(got.ctypes.data, a.dtable, got.nbytes, None))
    N.check("sync", lib.ks_gpu_synchronize())
    for p in held:
        N.check("free", lib.ks_gpu_free(p))
    return status, got, np.bincount(tokens, minlength=vocab).astype(np.float32)[:, None]


def test_kernels_in_a_second_context(N):
    N.check("device", N.lib.ks_gpu_set_device(0))
    status, got, want = _embedding_gradient(N)
    assert status == 0 and (got == want).all()
    cu = C.CDLL("libcuda.so.1")
    ctx, old = C.c_void_p(), C.c_void_p()
    assert cu.cuCtxCreate_v2(C.byref(ctx), 0, 0) == 0
    try:
        status, got, want = _embedding_gradient(N)
        assert status == 0 and (got == want).all()
    finally:
        assert cu.cuCtxPopCurrent_v2(C.byref(old)) == 0 and cu.cuCtxDestroy_v2(ctx) == 0
    status, got, want = _embedding_gradient(N)
    assert status == 0 and (got == want).all()
