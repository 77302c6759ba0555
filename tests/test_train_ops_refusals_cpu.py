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
