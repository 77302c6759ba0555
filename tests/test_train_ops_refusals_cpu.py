"""CPU: arguments that the training operators' front end has to refuse, and what
it hands to the C entries.  Tensors here lie in host memory and say that they are
on the GPU; the launches are replaced by a recorder, so nothing runs."""

from __future__ import annotations

import contextlib
import ctypes as C

import pytest
import torch


class FakeCuda(torch.Tensor):
    """A host tensor that passes for one on cuda:0."""

    is_cuda = True
    device = torch.device("cuda", 0)

    def get_device(self):
        return 0

    def record_stream(self, stream):
        FakeCuda.recorded.append((self.data_ptr(), stream.cuda_stream))


def fake(t):
    return t.as_subclass(FakeCuda)


class Recorder:
    """The library with its launches replaced: each notes its argument struct (the
    object itself) and returns `status`."""

    def __init__(self, lib):
        self._lib, self.calls = lib, []

    def __getattr__(self, name):
        if not name.endswith("_launch"):
            return getattr(self._lib, name)

        def launch(*args):
            structs = [a._obj for a in args if hasattr(a, "_obj")]
            self.calls.append((name, structs[-1]))
            return 0

        return launch


@pytest.fixture
def front(monkeypatch):
    from kernscope_b200 import native, ops

    FakeCuda.recorded = []
    recorder = Recorder(native.lib)
    monkeypatch.setattr(native, "lib", recorder)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "stream", lambda s: contextlib.nullcontext())
    monkeypatch.setattr(ops, "_raw_stream", lambda stream, dev: 0 if stream is None else stream.cuda_stream)
    return native, ops, recorder


@pytest.mark.parametrize("shape", [(32, 64), (16, 128), (1, 2048), (64, 33), (2048, 1)], ids=str)
def test_embedding_out_of_another_shape(front, shape):
    """A 2-D out is [tokens, dim]: of one with as many values but other rows, only
    the row stride would be used, and rows written past its end."""
    N, ops, rec = front
    table, tokens = fake(torch.zeros(100, 32).bfloat16()), fake(torch.zeros(64, dtype=torch.int64))
    with pytest.raises(ValueError):
        ops.embedding(tokens, table, out=fake(torch.zeros(shape).bfloat16()))
    assert not rec.calls


@pytest.mark.parametrize("shape", [(64, 32), (8, 8, 32), (2048,), (1, 64, 32)], ids=str)
def test_embedding_out_that_holds_the_rows(front, shape):
    N, ops, rec = front
    table, tokens = fake(torch.zeros(100, 32).bfloat16()), fake(torch.zeros(64, dtype=torch.int64))
    out = fake(torch.zeros(shape).bfloat16())
    assert ops.embedding(tokens, table, out=out) is out
    (name, a), = rec.calls
    assert name == "ks_embedding_launch" and (a.out, a.out_stride, a.tokens_count, a.dim) == (out.data_ptr(), 32, 64, 32)


def test_embedding_out_whose_rows_cannot_be_viewed(front):
    N, ops, rec = front
    table, tokens = fake(torch.zeros(100, 32).bfloat16()), fake(torch.zeros(64, dtype=torch.int64))
    with pytest.raises(ValueError):
        ops.embedding(tokens, table, out=fake(torch.zeros(8, 16, 32).bfloat16()[:, :8]))
    assert not rec.calls


def test_rows_overlap_against_every_byte(front):
    """The overlap test against sets of bytes: equal and different strides, rows
    between one another's, one row, none."""
    import random

    N, ops, rec = front
    r = random.Random(3)
    seen = {0: 0, 1: 0}
    for i in range(4000):
        def rows():
            width = r.randint(1, 9)
            return r.randint(1, 120), r.choice([0, 1, 1, 2, 3, 7]), width, r.choice([width, 10, 10, 10, r.randint(width, 24)])

        a, b = rows(), rows()
        held = lambda t: {t[0] + k * t[3] + c for k in range(t[1]) for c in range(t[2])}  # noqa: E731
        want = int(bool(held(a) & held(b)))
        assert N.lib.ks_rows_overlap(*a, *b) == want, (a, b)
        seen[want] += 1
    assert min(seen.values()) > 500
    assert N.lib.ks_rows_overlap(None, 4, 8, 8, 1, 4, 8, 8) == 0
    far = (1 << 62, 1 << 40, 1 << 20, 1 << 60)  # no overflow
    assert N.lib.ks_rows_overlap(*far, 1 << 61, 4, 8, 8) == 0


def _scratch(n):
    flat = torch.zeros(n + 256, dtype=torch.uint8)
    at = -flat.data_ptr() % 256
    return fake(flat[at:at + n])


def _ce_case(n=70, dim=64, vocab=300):
    wide = fake(torch.zeros(max(n, vocab) * 3, 4 * dim).bfloat16())
    return (wide, wide[:n, :dim], wide[:vocab, dim:2 * dim], fake(torch.zeros(n, dtype=torch.int64)), fake(torch.zeros(n)),
            _scratch(64 << 20))


@pytest.fixture
def refusing(front, monkeypatch):
    """The real launches, which refuse before any CUDA call; one that would go on
    stops at the check for a device instead (this test is for machines without)."""
    if torch.cuda.is_available():
        pytest.skip("an accepted launch would run on host addresses")
    N, ops, rec = front
    monkeypatch.setattr(N, "lib", rec._lib)
    return N, ops


CE_ALIASES = {  # dh and dw as views of the buffer that also holds h (columns 0..63) and w (64..127)
    "dh is h": lambda b, n, v, d: (b[:n, :d], None),
    "dh begins inside h": lambda b, n, v, d: (b[n - 1:2 * n - 1, :d], None),
    "dh shares one column with w": lambda b, n, v, d: (b[:n, 2 * d - 1:3 * d - 1], None),
    "dw is w": lambda b, n, v, d: (None, b[:v, d:2 * d]),
    "dw shares one row with h": lambda b, n, v, d: (None, b[n - 1:n - 1 + v, :d]),
    "dw shares one row with dh": lambda b, n, v, d: (b[v:v + n, 2 * d:3 * d], b[v + n - 1:2 * v + n - 1, 2 * d:3 * d]),
}


@pytest.mark.parametrize("alias", CE_ALIASES, ids=str)
def test_cross_entropy_gradients_that_overlap(refusing, alias):
    """dw's tiles are written while others still read h and w, and dh's beside them."""
    N, ops = refusing
    wide, h, w, t, lse, ws = _ce_case()
    dh, dw = CE_ALIASES[alias](wide, 70, 300, 64)
    for call in (lambda: ops.linear_cross_entropy_grad(h, w, t, dh=dh, dw=dw, workspace=ws),
                 lambda: ops.linear_cross_entropy_backward(h, w, t, lse, dh=dh, dw=dw, workspace=ws)):
        with pytest.raises(ValueError, match="overlaps"):
            call()


def test_cross_entropy_workspace_that_overlaps(refusing):
    N, ops = refusing
    wide, h, w, t, lse, ws = _ce_case()
    inside = ws[4096:4096 + 300 * 64 * 2].view(torch.bfloat16).view(300, 64)
    for call in (lambda: ops.linear_cross_entropy(h, inside, t, workspace=ws),
                 lambda: ops.linear_cross_entropy_grad(h, w, t, dw=inside, workspace=ws)):
        with pytest.raises(ValueError, match="overlaps"):
            call()


def test_cross_entropy_gradients_between_the_inputs_rows(refusing):
    """Column ranges of one buffer share nothing: the launch goes on to look for a device."""
    N, ops = refusing
    wide, h, w, t, lse, ws = _ce_case()
    with pytest.raises(N.KsError) as e:
        ops.linear_cross_entropy_grad(h, w, t, dh=wide[:70, 128:192], dw=wide[:300, 192:], workspace=ws)
    assert e.value.status not in (N.KS_ERR_INVALID_ARGS, N.KS_ERR_WORKSPACE)


def test_cross_entropy_c_entry_refuses_overlaps(refusing):
    N, ops = refusing
    ws = _scratch(1 << 20)
    cfg = N.LinearCeConfig(0, 0, 0)

    def launch(**kw):
        a = N.LinearCeArgs(0x100000, 0x200000, 0x300000, 10, 64, 100, 64, 64, N.KS_BF16, N.KS_CE_GRAD, N.KS_CE_MEAN, 1.0,
                           -100, None, 0x400000, 0x500000, 0x600000, 0x700000, 64, 64, ws.data_ptr(), 1 << 20)
        for k, v in kw.items():
            setattr(a, k, v)
        return N.lib.ks_linear_ce_launch(C.byref(cfg), C.byref(a), None)

    assert launch() not in (N.KS_ERR_INVALID_ARGS, N.KS_ERR_WORKSPACE)  # no device
    for kw in (dict(dh=0x100000), dict(dh=0x200000), dict(dw=0x200000), dict(dw=0x100000), dict(dw=0x600000),
               dict(dh=0x300000), dict(loss=0x300000), dict(loss=0x500000), dict(lse=0x300040), dict(lse=0x700000),
               dict(dloss=0x400000), dict(h=ws.data_ptr()), dict(dw=ws.data_ptr())):
        assert launch(**kw) == N.KS_ERR_INVALID_ARGS, kw
    # the backward pass reads lse and writes no loss
    assert launch(ce_pass=N.KS_CE_BACKWARD, loss=0x300000) != N.KS_ERR_INVALID_ARGS
    assert launch(ce_pass=N.KS_CE_BACKWARD, dh=0x500000) == N.KS_ERR_INVALID_ARGS
    # the forward pass writes neither dh nor dw
    assert launch(ce_pass=N.KS_CE_FORWARD, dh=0x100000, dw=0x200000) != N.KS_ERR_INVALID_ARGS


@pytest.mark.parametrize("dtype", [None, torch.float32], ids=str)
@pytest.mark.parametrize("accumulate", [False, True])
def test_embedding_gradient_that_overlaps(refusing, accumulate, dtype):
    """The table's rows are zeroed (or written) while dout is still to be read."""
    N, ops = refusing
    n, dim, vocab = 40, 32, 100
    buf = fake(torch.zeros(400, 4 * dim).bfloat16())
    tokens = fake(torch.zeros(n, dtype=torch.int64))
    ws = _scratch(1 << 20)
    as_table = lambda t: t if dtype is None else t.view(torch.float32)  # noqa: E731
    width = dim if dtype is None else 2 * dim  # columns of bf16 that a row of the table takes
    call = lambda dout, dtable, ws=ws: ops.embedding_backward(tokens, dout, vocab, dtable=dtable, accumulate=accumulate,  # noqa: E731
                                                              workspace=ws)
    for dout, dtable in ((buf[:n, :dim], as_table(buf[:vocab, :width])),
                         (buf[vocab - 1:vocab - 1 + n, :dim], as_table(buf[:vocab, :width])),
                         (buf[:n, width - 1:width - 1 + dim], as_table(buf[:vocab, :width]))):
        with pytest.raises(ValueError, match="dtable overlaps dout"):
            call(dout, dtable)
    with pytest.raises(ValueError, match="workspace"):
        call(buf[:n, :dim], fake(ws[:vocab * width * 2]).view(torch.bfloat16 if dtype is None else dtype).view(vocab, dim))
    with pytest.raises(N.KsError) as e:  # the table's rows lie between dout's: on to the check for a device
        call(buf[:n, width:width + dim], as_table(buf[:vocab, :width]))
    assert e.value.status not in (N.KS_ERR_INVALID_ARGS, N.KS_ERR_WORKSPACE)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
def test_embedding_out_that_overlaps(refusing, dtype):
    """Rows of the table that another warp has yet to read."""
    N, ops = refusing
    n, dim, vocab = 40, 32, 100
    buf = fake(torch.zeros(400, 4 * dim, dtype=dtype))
    tokens = fake(torch.zeros(n, dtype=torch.int64))
    table = buf[:vocab, dim:2 * dim]
    for out in (table[:n], buf[vocab - 1:vocab - 1 + n, dim:2 * dim], buf[:n, 1:dim + 1], buf[:n, 2 * dim - 1:3 * dim - 1]):
        with pytest.raises(ValueError, match="out overlaps table"):
            ops.embedding(tokens, table, out=out)
    for out in (buf[:n, :dim], buf[:n, 2 * dim:3 * dim], buf[vocab:vocab + n, dim:2 * dim]):  # on to the check for a device
        with pytest.raises(N.KsError) as e:
            ops.embedding(tokens, table, out=out)
        assert e.value.status != N.KS_ERR_INVALID_ARGS


BAD_WORKSPACES = {"in host memory": lambda: torch.zeros(1 << 20, dtype=torch.uint8),
                  "every other byte": lambda: fake(torch.zeros(1 << 21, dtype=torch.uint8))[::2],
                  "columns of a matrix": lambda: fake(torch.zeros(1024, 2048, dtype=torch.uint8))[:, :1024]}


@pytest.mark.parametrize("kind", BAD_WORKSPACES, ids=str)
def test_workspace_that_kernels_cannot_use(front, kind):
    """A host address, or bytes between which lie another tensor's."""
    N, ops, rec = front
    ws = BAD_WORKSPACES[kind]()
    h, w, t = fake(torch.zeros(8, 64).bfloat16()), fake(torch.zeros(100, 64).bfloat16()), fake(torch.zeros(8, dtype=torch.int64))
    for call in (lambda: ops.linear_cross_entropy(h, w, t, workspace=ws),
                 lambda: ops.linear_cross_entropy_grad(h, w, t, workspace=ws),
                 lambda: ops.linear_cross_entropy_backward(h, w, t, fake(torch.zeros(8)), workspace=ws),
                 lambda: ops.embedding_backward(t, h, 100, workspace=ws)):
        with pytest.raises(ValueError, match="workspace"):
            call()
    assert not rec.calls


def test_workspace_of_any_type(front):
    N, ops, rec = front
    h, t = fake(torch.zeros(8, 64).bfloat16()), fake(torch.zeros(8, dtype=torch.int64))
    ws = fake(torch.zeros(1 << 10, 1 << 8))
    ops.embedding_backward(t, h, 100, workspace=ws)
    (_, a), = rec.calls
    assert (a.workspace, a.workspace_bytes) == (ws.data_ptr(), 1 << 20)


class Stream:
    def __init__(self, raw):
        self.cuda_stream = raw


@pytest.fixture
def clipping(front, monkeypatch):
    """Host memory for what a clipper allocates on the GPU."""
    N, ops, rec = front
    empty = torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, device=None, **k: fake(empty(*a, **k)))
    monkeypatch.setattr(torch.Tensor, "to", lambda self, *a, **k: fake(self))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: Stream(0))
    return ops, rec


def test_clipper_keeps_its_memory_for_the_stream_it_ran_on(clipping):
    """The table and the scratch come from the pool of the stream that was current when
    the clipper was made; after a call on another stream, dropping the clipper (and
    with it the last reference to a gradient) must not free them for reuse there."""
    ops, rec = clipping
    grads, outs = [fake(torch.ones(n)) for n in (100, 7)], [fake(torch.ones(n)) for n in (100, 7)]
    clipper = ops.GradClipper(grads, out=outs)
    clipper.clip(1.0)
    assert not FakeCuda.recorded  # its own stream
    clipper.clip(1.0, stream=Stream(7))
    mine = {a.table for _, a in rec.calls} | {a.workspace for _, a in rec.calls}
    assert len(mine) == 2
    assert {(p, 7) for p in mine | {t.data_ptr() for t in grads + outs}} == set(FakeCuda.recorded)
    clipper.clip(1.0, stream=Stream(9))
    assert {p for p, s in FakeCuda.recorded if s == 9} == {p for p, s in FakeCuda.recorded if s == 7}


def test_clipper_calls_have_arguments_of_their_own(clipping, monkeypatch):
    """Two host threads in clip() at once: each launch has its own limit and leaves
    its norm where its own caller looks."""
    import threading

    ops, rec = clipping
    clipper = ops.GradClipper([fake(torch.ones(100))])
    both = threading.Barrier(2, timeout=20)
    raw, returned, failed = ops._raw_stream, {}, []

    def meet(stream, dev):  # each thread fetches its stream while the other is in clip() too
        both.wait()
        return raw(stream, dev)

    def launch(args, stream):
        both.wait()  # both have filled their arguments
        a = args._obj
        rec.calls.append((a.max_norm, a.norm))
        return 0

    def call(limit):
        try:
            returned[limit] = clipper.clip(limit).data_ptr()
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    monkeypatch.setattr(ops, "_raw_stream", meet)
    monkeypatch.setattr(rec, "ks_grad_clip_launch", launch, raising=False)
    threads = [threading.Thread(target=call, args=(limit,)) for limit in (1.0, 2.0)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed and sorted(rec.calls) == sorted((k, p) for k, p in returned.items())


@pytest.mark.parametrize("ce_pass", ["KS_CE_FORWARD", "KS_CE_BACKWARD", "KS_CE_GRAD"])
@pytest.mark.parametrize("tokens,dim,vocab", [(8192, 4096, 512), (2048, 4096, 1024), (4096, 2048, 4000), (1000, 64, 512),
                                              (64, 4096, 512), (65, 1001, 257), (333, 1000, 10007), (1, 1, 1)])
def test_least_workspace_of_the_cross_entropy(refusing, tokens, dim, vocab, ce_pass):
    """The least size is no more than what a call makes use of under any limit, is
    accepted, and one byte less is not."""
    N, ops = refusing
    cfg = N.LinearCeConfig(0, 0, 0)
    a = N.LinearCeArgs(1 << 40, 2 << 40, 3 << 40, tokens, dim, vocab, dim, dim, N.KS_BF16, getattr(N, ce_pass), N.KS_CE_SUM, 1.0,
                       -100, None, 4 << 40, 5 << 40, 6 << 40, 7 << 40, dim, dim, 8 << 40, 0)
    least, want = C.c_size_t(0), C.c_size_t(0)
    sizes = set()
    for limit in (0, 1, 1 << 20, 8 << 20, 64 << 20, 1 << 30, 1 << 40):
        assert N.lib.ks_linear_ce_workspace_bytes(C.byref(cfg), C.byref(a), limit, C.byref(least), C.byref(want)) == 0
        assert 0 < least.value <= want.value <= max(limit, least.value)
        sizes |= {least.value, want.value}
    for size in sizes:
        a.workspace_bytes = size
        assert N.lib.ks_linear_ce_launch(C.byref(cfg), C.byref(a), None) not in (N.KS_ERR_WORKSPACE, N.KS_ERR_INVALID_ARGS)
    a.workspace_bytes = least.value - 1
    assert N.lib.ks_linear_ce_launch(C.byref(cfg), C.byref(a), None) == N.KS_ERR_WORKSPACE
