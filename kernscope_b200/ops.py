"""Torch-tensor front end of the C ABI (device memory and streams from torch).

Each function validates dtype/layout, builds the family's config and args
structs, and calls ``ks_<family>_launch`` on the current torch stream.  Any
non-zero status raises ``KsError``; there is no CPU or library fallback.

Default configurations are the sm_100a picks for the benchmark shapes; the
tuner (``kernscope-tune``) searches the full config spaces.
"""

from __future__ import annotations

import ctypes as C

import torch

from . import native as N


def _stream_ptr(stream=None) -> C.c_void_p:
    s = stream if stream is not None else torch.cuda.current_stream()
    return C.c_void_p(s.cuda_stream)


def _check_bf16_2d(name, t):
    if not (t.is_cuda and t.dtype == torch.bfloat16 and t.is_contiguous()):
        raise ValueError(f"{name} must be a contiguous bf16 CUDA tensor")


def _pow2_block(cols: int, vec: int, per_thread: int) -> int:
    want = max(1, cols // (vec * per_thread))
    b = 128
    while b < want and b < 1024:
        b *= 2
    return b


def _cluster_default(family: str, make, rows, cols: int):
    """A few very long rows (at most 64 rows of 65536+ columns) leave most SMs
    idle one CTA per row; spreading each row over a cluster measured
    1590 -> 1987 GB/s (softmax) and 1310 -> 1778 GB/s (layernorm) at
    64 x 131072 on B200.  With more rows the per-row CTAs win."""
    if rows is None or rows > 64 or cols < 65536:
        return None
    for block in (512, 1024):
        cfg = make(block, 8, N.KS_MODE_CLUSTER)
        if N.validate(family, cfg, rows, cols)[0] == 0:
            return cfg
    return None


def default_softmax_config(cols: int, rows: int | None = None) -> N.SoftmaxConfig:
    c = _cluster_default("softmax", N.SoftmaxConfig, rows, cols)
    if c is not None:
        return c
    if rows is not None and rows >= 1024 and 16384 < cols <= 32768 and cols % 8 == 0:
        # 1024-thread STAGED CTAs keep three 64 KB rows in flight: 2048 x 32768
        # measured 3786 -> 4123 GB/s against ONEPASS on B200 (equal at 1024 rows)
        return N.SoftmaxConfig(1024, 8, N.KS_MODE_STAGED)
    vec = 8 if cols % 8 == 0 else 4 if cols % 4 == 0 else 2 if cols % 2 == 0 else 1
    block = _pow2_block(cols, vec, 4)
    mode = N.KS_MODE_ONEPASS if cols <= block * 32 else N.KS_MODE_TWOPASS
    return N.SoftmaxConfig(block, vec, mode)


def default_layernorm_config(cols: int, rows: int | None = None) -> N.LayerNormConfig:
    c = _cluster_default("layernorm", N.LayerNormConfig, rows, cols)
    if c is not None:
        return c
    if 8192 < cols <= 16384 and cols % 8 == 0:
        # a two-row bulk-copy ring per 512-thread CTA: 4096 x 16384 measured
        # 3787 -> 4295 GB/s against ONEPASS on B200 (2048 rows: 3627 -> 3771)
        return N.LayerNormConfig(512, 8, N.KS_MODE_STAGED)
    vec = 8 if cols % 8 == 0 else 4 if cols % 4 == 0 else 2 if cols % 2 == 0 else 1
    block = _pow2_block(cols, vec, 4)
    mode = N.KS_MODE_ONEPASS if cols <= block * 32 else N.KS_MODE_TWOPASS
    return N.LayerNormConfig(block, vec, mode)


def default_bias_gelu_config(cols: int, gelu: str = "tanh") -> N.BiasGeluConfig:
    vec = 8 if cols % 8 == 0 else 4 if cols % 4 == 0 else 2 if cols % 2 == 0 else 1
    if gelu != "tanh":
        # 8-wide erf: 1024 threads run the kernel that looks every bf16 code up
        # in a shared-memory table (one CTA per SM)
        return N.BiasGeluConfig(1024 if vec == 8 else 128, vec, N.KS_GELU_ERF)
    return N.BiasGeluConfig(128, vec, N.KS_GELU_TANH)


def default_reduction_config(cols: int, axis: int) -> N.ReductionConfig:
    if axis == -1:
        return N.ReductionConfig(512, 4, N.KS_MODE_STRIDED)
    vec = 8 if cols % 8 == 0 else 4 if cols % 4 == 0 else 2 if cols % 2 == 0 else 1
    return N.ReductionConfig(256, vec, N.KS_MODE_TREE)


def default_matmul_config(m: int, n: int, k: int) -> N.MatmulConfig:
    if n >= 256 and m * n >= 2048 * 2048:
        # 256x256 tiles on one CTA (two M=128 MMAs per B tile, cta_group 1),
        # bands of 8 N-tiles whose B panels stay in L2 (group_m -8)
        return N.MatmulConfig(256, 256, 64, 3, 1, -8, 1)
    return N.MatmulConfig(128, 128, 64, 6, 2, 8)


def default_flash_attention_config(causal: bool) -> N.FlashAttentionConfig:
    return N.FlashAttentionConfig(256, 128, 2, 1 if causal else 0)


def softmax(x: torch.Tensor, out=None, cfg=None, stream=None) -> torch.Tensor:
    _check_bf16_2d("x", x)
    rows, cols = x.shape
    out = torch.empty_like(x) if out is None else out
    cfg = cfg or default_softmax_config(cols, rows)
    args = N.SoftmaxArgs(x.data_ptr(), out.data_ptr(), rows, cols)
    N.check("ks_softmax_launch", N.lib.ks_softmax_launch(C.byref(cfg), C.byref(args), _stream_ptr(stream)))
    return out


def layernorm(x, gamma, beta, eps: float = 1e-5, out=None, cfg=None, stream=None) -> torch.Tensor:
    for nm, t in (("x", x), ("gamma", gamma), ("beta", beta)):
        _check_bf16_2d(nm, t)
    rows, cols = x.shape
    out = torch.empty_like(x) if out is None else out
    cfg = cfg or default_layernorm_config(cols, rows)
    args = N.LayerNormArgs(x.data_ptr(), gamma.data_ptr(), beta.data_ptr(), out.data_ptr(), rows, cols, eps)
    N.check("ks_layernorm_launch", N.lib.ks_layernorm_launch(C.byref(cfg), C.byref(args), _stream_ptr(stream)))
    return out


def bias_gelu(x, bias, gelu: str = "tanh", out=None, cfg=None, stream=None) -> torch.Tensor:
    _check_bf16_2d("x", x)
    _check_bf16_2d("bias", bias)
    cols = bias.numel()
    out = torch.empty_like(x) if out is None else out
    cfg = cfg or default_bias_gelu_config(cols, gelu)
    args = N.BiasGeluArgs(x.data_ptr(), bias.data_ptr(), out.data_ptr(), x.numel(), cols)
    N.check("ks_bias_gelu_launch", N.lib.ks_bias_gelu_launch(C.byref(cfg), C.byref(args), _stream_ptr(stream)))
    return out


_DT = {torch.bfloat16: N.KS_BF16, torch.float32: N.KS_F32}


def reduction_args(x, out, axis: int, out_dtype, workspace=None, partial_f64=None) -> N.ReductionArgs:
    rows, cols = (x.shape[0], x.numel() // x.shape[0]) if x.dim() >= 1 else (1, 1)
    if x.dim() == 1:
        rows, cols = 1, x.numel()
    return N.ReductionArgs(x.data_ptr(), out.data_ptr(), rows, cols, _DT[x.dtype], _DT[out_dtype], axis,
                           workspace.data_ptr() if workspace is not None else None,
                           workspace.numel() if workspace is not None else 0,
                           partial_f64.data_ptr() if partial_f64 is not None else None)


def reduction_workspace(x, axis: int = 0, out_dtype=None, cfg=None) -> torch.Tensor:
    out_dtype = out_dtype or x.dtype
    cols = x.numel() // x.shape[0] if x.dim() > 1 else x.numel()
    cfg = cfg or default_reduction_config(cols, axis)
    dummy = torch.empty(1, dtype=out_dtype, device=x.device)
    args = reduction_args(x, dummy, axis, out_dtype)
    n = C.c_size_t(0)
    N.check("ks_reduction_workspace_bytes",
            N.lib.ks_reduction_workspace_bytes(C.byref(cfg), C.byref(args), C.byref(n)))
    return torch.empty(max(int(n.value), 256), dtype=torch.uint8, device=x.device)


def reduction(x, axis: int = 0, out_dtype=None, out=None, cfg=None, workspace=None, partial_f64=None,
              stream=None) -> torch.Tensor:
    """axis 0: y[j] = sum_i x[i, j]; axis -1: full sum of x (fp32 in/out)."""
    if not (x.is_cuda and x.is_contiguous() and x.dtype in _DT):
        raise ValueError("x must be a contiguous bf16/fp32 CUDA tensor")
    out_dtype = out_dtype or x.dtype
    cols = x.numel() // x.shape[0] if x.dim() > 1 else x.numel()
    if out is None:
        out = torch.empty(1 if axis == -1 else cols, dtype=out_dtype, device=x.device)
    cfg = cfg or default_reduction_config(cols, axis)
    if workspace is None:
        workspace = reduction_workspace(x, axis, out_dtype, cfg)
    args = reduction_args(x, out, axis, out_dtype, workspace, partial_f64)
    N.check("ks_reduction_launch", N.lib.ks_reduction_launch(C.byref(cfg), C.byref(args), _stream_ptr(stream)))
    return out


def matmul(a, b, out=None, cfg=None, stream=None) -> torch.Tensor:
    _check_bf16_2d("a", a)
    _check_bf16_2d("b", b)
    m, k = a.shape
    k2, n = b.shape
    if k != k2:
        raise ValueError("inner dimensions differ")
    out = torch.empty((m, n), dtype=torch.bfloat16, device=a.device) if out is None else out
    cfg = cfg or default_matmul_config(m, n, k)
    args = N.MatmulArgs(a.data_ptr(), b.data_ptr(), out.data_ptr(), m, n, k)
    N.check("ks_matmul_launch", N.lib.ks_matmul_launch(C.byref(cfg), C.byref(args), _stream_ptr(stream)))
    return out


def flash_attention(q, k, v, causal: bool = True, scale: float = 0.0, out=None, cfg=None,
                    stream=None) -> torch.Tensor:
    """q [B,H,Nq,d], k/v [B,H,Nk,d] (or [Nq,d]/[Nk,d] single head)."""
    for nm, t in (("q", q), ("k", k), ("v", v)):
        _check_bf16_2d(nm, t)
    if q.dim() == 2:
        b, h, nq, d = 1, 1, q.shape[0], q.shape[1]
        nk = k.shape[0]
    else:
        b, h, nq, d = q.shape
        nk = k.shape[2]
    out = torch.empty_like(q) if out is None else out
    cfg = cfg or default_flash_attention_config(causal)
    cfg.causal = 1 if causal else 0
    args = N.FlashAttentionArgs(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), b, h, nq, nk, d, scale)
    N.check("ks_flash_attention_launch",
            N.lib.ks_flash_attention_launch(C.byref(cfg), C.byref(args), _stream_ptr(stream)))
    return out


# ---------------------------------------------------------------------------
# Training operators at the vocabulary end of a language model.
#
# The smallest of these calls take a few microseconds on the GPU, so the host
# side is kept short: one pass of checks, raw stream handles, sizes of scratch
# remembered per problem size (never per tensor).
# ---------------------------------------------------------------------------
_DT_TRAIN = {torch.bfloat16: N.KS_BF16, torch.float16: N.KS_F16, torch.float32: N.KS_F32}
_DT_HALF = {torch.bfloat16: N.KS_BF16, torch.float16: N.KS_F16}
_REDUCTIONS = {"none": N.KS_CE_NONE, "mean": N.KS_CE_MEAN, "sum": N.KS_CE_SUM}


def _raw_stream(stream, dev: int) -> int:
    return torch._C._cuda_getCurrentRawStream(dev) if stream is None else stream.cuda_stream


def _empty(like, shape, dtype, stream) -> torch.Tensor:
    """An uninitialised tensor on `like`'s device, from the pool of the stream
    that the launch goes to: scratch freed after the call is then reused only
    behind the launch."""
    if stream is None:
        return like.new_empty(shape, dtype=dtype)
    with torch.cuda.stream(stream):
        return like.new_empty(shape, dtype=dtype)


def _zero(t, stream) -> torch.Tensor:
    if stream is None:
        return t.zero_()
    with torch.cuda.stream(stream):
        return t.zero_()


def _rows(name, t, dtypes, dev: int) -> tuple[int, int, int]:
    """(rows, columns, row stride) of a 2-D tensor on device `dev` whose rows are
    dense and do not overlap."""
    if t.dtype in dtypes and t.get_device() == dev and t.dim() == 2:
        (r, c), (s0, s1) = t.shape, t.stride()
        if (s1 == 1 or c <= 1) and (s0 >= c or r <= 1):
            return r, c, (s0 if s0 > c else c)
    raise ValueError(f"{name} must be a 2-D tensor of {' or '.join(str(d) for d in dtypes)} on the current CUDA device, "
                     f"with dense rows that do not overlap (got {t.dtype} {tuple(t.shape)}, strides {t.stride()}, "
                     f"{t.device})")


def _as_rows(name, t, n: int, dim: int) -> torch.Tensor:
    """t, or its view as [n, dim] where it has another rank than 2."""
    if t.dim() == 2:
        return t
    try:
        return t.view(n, dim)
    except RuntimeError:
        raise ValueError(f"{name} must be [{n}, {dim}] or view as it (got {tuple(t.shape)}, strides {t.stride()})") from None


def _values(name, t, dtype, n: int, dev: int) -> int:
    """Address of a contiguous tensor of n values on device `dev`."""
    if t.dtype is dtype and t.get_device() == dev and t.numel() == n and t.is_contiguous():
        return t.data_ptr()
    raise ValueError(f"{name} must be a contiguous {dtype} tensor of {n} values on the current CUDA device (got "
                     f"{t.dtype} {tuple(t.shape)}, {t.device})")


def _scratch(workspace, dev: int) -> tuple[int, int]:
    """(address, bytes) of a caller's workspace: any type, contiguous, on device `dev`."""
    if workspace.get_device() == dev and workspace.is_contiguous():
        return workspace.data_ptr(), workspace.numel() * workspace.element_size()
    raise ValueError(f"workspace must be a contiguous tensor on the current CUDA device (got {tuple(workspace.shape)}, "
                     f"strides {workspace.stride()}, {workspace.device})")


def _name_overlap(outputs: int, **memory) -> None:
    """After a launch that was refused for its arguments: a ValueError where one of
    the first `outputs` tensors shares memory with another.  memory: (address, rows,
    bytes per row, bytes between rows) of each."""
    names = list(memory)
    for i, a in enumerate(names[:outputs]):
        for b in names[i + 1:]:
            if N.lib.ks_rows_overlap(*memory[a], *memory[b]):
                raise ValueError(f"{a} overlaps {b}")


def _linear_ce_args(h, w, targets, ce_pass, reduction, ignore_index, grad_scale=1.0) -> N.LinearCeArgs:
    dev = torch.cuda.current_device()
    n, dim, h_stride = _rows("h", h, _DT_HALF, dev)
    vocab, w_dim, w_stride = _rows("w", w, (h.dtype,), dev)
    if dim != w_dim:
        raise ValueError("h and w differ in their last dimension")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {sorted(_REDUCTIONS)}")
    return N.LinearCeArgs(h.data_ptr(), w.data_ptr(), _values("targets", targets, torch.int64, n, dev), n, dim, vocab,
                          h_stride, w_stride, _DT_HALF[h.dtype], ce_pass, _REDUCTIONS[reduction], grad_scale,
                          ignore_index, None, None, None, None, None, dim, dim)


# Default bound on the scratch of one call.  Where 2 bytes for every (token,
# vocabulary entry) fit, loss and gradient take the logits once; with less, twice.
LINEAR_CE_WORKSPACE_LIMIT = 4 << 30


def linear_cross_entropy_workspace_bytes(args: N.LinearCeArgs, cfg=None, limit=None) -> tuple[int, int]:
    """(least, preferred) workspace bytes of one ks_linear_ce_launch."""
    cfg = cfg or N.LinearCeConfig()
    least, want = C.c_size_t(0), C.c_size_t(0)
    N.check("ks_linear_ce_workspace_bytes",
            N.lib.ks_linear_ce_workspace_bytes(C.byref(cfg), C.byref(args),
                                               LINEAR_CE_WORKSPACE_LIMIT if limit is None else limit,
                                               C.byref(least), C.byref(want)))
    return least.value, want.value


_CE_DEFAULT = N.LinearCeConfig()
_ce_scratch: dict = {}  # problem size and alignment -> preferred workspace bytes


def _linear_ce_run(a, cfg, workspace, like, stream):
    if workspace is None:
        if cfg is None:
            # all that the size depends on: sizes, and what keeps a row from a 16-byte boundary
            key = (a.tokens, a.dim, a.vocab, a.ce_pass, LINEAR_CE_WORKSPACE_LIMIT, (a.h | a.h_stride << 1) & 15,
                   (a.w | a.w_stride << 1) & 15, ((a.dh or 0) | a.dh_stride << 1) & 15,
                   ((a.dw or 0) | a.dw_stride << 1) & 15)
            size = _ce_scratch.get(key)
            if size is None:
                if len(_ce_scratch) >= 4096:
                    _ce_scratch.clear()
                size = _ce_scratch[key] = linear_cross_entropy_workspace_bytes(a)[1]
        else:
            size = linear_cross_entropy_workspace_bytes(a, cfg)[1]
        workspace = _empty(like, size, torch.uint8, stream)
        a.workspace, a.workspace_bytes = workspace.data_ptr(), size
    else:
        a.workspace, a.workspace_bytes = _scratch(workspace, like.get_device())
    status = N.lib.ks_linear_ce_launch(C.byref(cfg or _CE_DEFAULT), C.byref(a), _raw_stream(stream, like.get_device()))
    if status == N.KS_ERR_INVALID_ARGS:
        n, row = a.tokens, a.dim * 2
        _name_overlap(3, dh=(a.dh, n, row, a.dh_stride * 2), dw=(a.dw, a.vocab, row, a.dw_stride * 2),
                      workspace=(a.workspace, 1, a.workspace_bytes, 0), h=(a.h, n, row, a.h_stride * 2),
                      w=(a.w, a.vocab, row, a.w_stride * 2), targets=(a.targets, 1, n * 8, 0),
                      lse=(a.lse, 1, n * 4, 0), dloss=(a.dloss, 1, n * 4 if a.reduction == N.KS_CE_NONE else 4, 0))
    N.check("ks_linear_ce_launch", status)


def linear_cross_entropy(h, w, targets, ignore_index: int = -100, reduction: str = "none", cfg=None, workspace=None,
                         stream=None):
    """Loss of each token (or their mean or sum) and log-sum-exp of each token's
    logits h @ w.T, without the logits in memory: h [tokens, dim], w [vocab,
    dim] (bf16 or fp16), targets int64.  Returns (loss, lse) in fp32."""
    a = _linear_ce_args(h, w, targets, N.KS_CE_FORWARD, reduction, ignore_index)
    n = a.tokens
    loss = _empty(h, n if reduction == "none" else 1, torch.float32, stream)
    lse = _empty(h, n, torch.float32, stream)
    if n == 0:
        return _zero(loss, stream), lse
    a.loss, a.lse = loss.data_ptr(), lse.data_ptr()
    _linear_ce_run(a, cfg, workspace, h, stream)
    return loss, lse


def _linear_ce_grads(a, h, w, dh, dw, stream):
    for name, t, like in (("dh", dh, h), ("dw", dw, w)):
        if t is None:
            t = _empty(like, like.shape, like.dtype, stream)
        else:
            rows, cols, stride = _rows(name, t, (like.dtype,), like.get_device())
            if (rows, cols) != tuple(like.shape):
                raise ValueError(f"{name} must have the shape {tuple(like.shape)}")
            setattr(a, name + "_stride", stride)
        setattr(a, name, t.data_ptr())
        if name == "dh":
            dh = t
        else:
            dw = t
    return dh, dw


def linear_cross_entropy_backward(h, w, targets, lse, dloss=None, ignore_index: int = -100, reduction: str = "none",
                                  grad_scale: float = 1.0, dh=None, dw=None, cfg=None, workspace=None, stream=None):
    """Gradients (dh, dw) of linear_cross_entropy from its lse.  dloss: the
    incoming fp32 gradient, one value per token for reduction "none", one value
    otherwise; None stands for ones.  Tokens with targets == ignore_index take no
    part, and the mean divides by the number of the others.  dh and dw, where
    given, overlap neither one another nor h or w."""
    a = _linear_ce_args(h, w, targets, N.KS_CE_BACKWARD, reduction, ignore_index, grad_scale)
    dev = h.get_device()
    a.lse = _values("lse", lse, torch.float32, a.tokens, dev)
    if dloss is not None:
        a.dloss = _values("dloss", dloss, torch.float32, a.tokens if reduction == "none" else 1, dev)
    dh, dw = _linear_ce_grads(a, h, w, dh, dw, stream)
    if a.tokens == 0:
        return dh, _zero(dw, stream)
    _linear_ce_run(a, cfg, workspace, h, stream)
    return dh, dw


def linear_cross_entropy_grad(h, w, targets, ignore_index: int = -100, reduction: str = "mean", grad_scale: float = 1.0,
                              dh=None, dw=None, cfg=None, workspace=None, stream=None):
    """Loss (fp32, one value) and the gradients of grad_scale * loss with respect
    to h and w in one call: what a training step needs of its last layer.  dh and
    dw, where given, overlap neither one another nor h or w."""
    a = _linear_ce_args(h, w, targets, N.KS_CE_GRAD, reduction, ignore_index, grad_scale)
    if reduction == "none":
        raise ValueError("loss and gradient in one call need reduction 'mean' or 'sum'")
    loss = _empty(h, 1, torch.float32, stream)
    dh, dw = _linear_ce_grads(a, h, w, dh, dw, stream)
    if a.tokens == 0:
        return _zero(loss, stream), dh, _zero(dw, stream)
    a.loss = loss.data_ptr()
    _linear_ce_run(a, cfg, workspace, h, stream)
    return loss, dh, dw


def embedding(tokens, table, scale: float = 1.0, out=None, stream=None) -> torch.Tensor:
    """scale * table[tokens] (tokens int64 of any shape, table [vocab, dim] in
    bf16, fp16 or fp32); tokens outside [0, vocab) give rows of zeros.  `out`:
    [number of tokens, dim] with any row stride, or what views as that; it does not
    overlap table."""
    dev = torch.cuda.current_device()
    vocab, dim, table_stride = _rows("table", table, _DT_TRAIN, dev)
    n = tokens.numel()
    ids = _values("tokens", tokens, torch.int64, n, dev)
    if out is None:
        out = _empty(table, (*tokens.shape, dim), table.dtype, stream)
        out_stride = dim
    else:
        rows, cols, out_stride = _rows("out", _as_rows("out", out, n, dim), (table.dtype,), dev)
        if (rows, cols) != (n, dim):
            raise ValueError(f"out must be [{n}, {dim}], or of another rank and {n} rows of {dim} as a view")
    if n == 0:
        return out
    args = N.EmbeddingArgs(ids, n, table.data_ptr(), out.data_ptr(), vocab, dim, table_stride, out_stride,
                           _DT_TRAIN[table.dtype], scale)
    status = N.lib.ks_embedding_launch(C.byref(args), _raw_stream(stream, dev))
    if status == N.KS_ERR_INVALID_ARGS:
        size = table.element_size()
        _name_overlap(1, out=(args.out, n, dim * size, out_stride * size),
                      table=(args.table, vocab, dim * size, table_stride * size), tokens=(ids, 1, n * 8, 0))
    N.check("ks_embedding_launch", status)
    return out


_EMB_DEFAULT = N.EmbeddingGradConfig()
_emb_scratch: dict = {}  # problem size -> workspace bytes


def embedding_backward(tokens, dout, vocab: int, scale: float = 1.0, padding_idx: int = -1, dtable=None, dtype=None,
                       accumulate: bool = False, cfg=None, workspace=None, stream=None) -> torch.Tensor:
    """Gradient of `embedding` with respect to its table: [vocab, dim] in dout's
    type or fp32 (`dtype`, or that of `dtable`).  accumulate adds to `dtable`'s
    values and touches the rows of `tokens` alone; otherwise every row is
    written.  Tokens equal to padding_idx or outside [0, vocab) have no part.
    dtable, where given, does not overlap dout."""
    dev = torch.cuda.current_device()
    rows = dout if dout.dim() == 2 else dout.view(tokens.numel(), dout.shape[-1])
    n, dim, dout_stride = _rows("dout", rows, _DT_TRAIN, dev)
    ids = _values("tokens", tokens, torch.int64, n, dev)
    if dtable is None:
        if accumulate:
            raise ValueError("accumulate needs the dtable to add to")
        if dtype not in (None, dout.dtype, torch.float32):
            raise ValueError("the gradient has the type of dout or float32")
        dtable = _empty(dout, (vocab, dim), dtype or dout.dtype, stream)
        dtable_stride = dim
    else:
        r, c, dtable_stride = _rows("dtable", dtable, (dout.dtype, torch.float32), dev)
        if (r, c) != (vocab, dim) or (dtype is not None and dtable.dtype != dtype):
            raise ValueError(f"dtable must be [{vocab}, {dim}]" + (f" of {dtype}" if dtype is not None else ""))
    if n == 0:
        return dtable if accumulate else _zero(dtable, stream)
    args = N.EmbeddingGradArgs(ids, n, rows.data_ptr(), dtable.data_ptr(), vocab, dim, dout_stride, dtable_stride,
                               _DT_TRAIN[dout.dtype], _DT_TRAIN[dtable.dtype], accumulate, scale, padding_idx)
    cfg = cfg or _EMB_DEFAULT
    if workspace is None:
        key = (n, vocab, dim, args.dtype, cfg.chunk)
        size = _emb_scratch.get(key)
        if size is None:
            if len(_emb_scratch) >= 4096:
                _emb_scratch.clear()
            need = C.c_size_t(0)
            N.check("ks_embedding_grad_workspace_bytes",
                    N.lib.ks_embedding_grad_workspace_bytes(C.byref(cfg), C.byref(args), C.byref(need)))
            size = _emb_scratch[key] = need.value
        workspace = _empty(dout, size, torch.uint8, stream)
        args.workspace, args.workspace_bytes = workspace.data_ptr(), size
    else:
        args.workspace, args.workspace_bytes = _scratch(workspace, dev)
    status = N.lib.ks_embedding_grad_launch(C.byref(cfg), C.byref(args), _raw_stream(stream, dev))
    if status == N.KS_ERR_INVALID_ARGS:
        size, out_size = dout.element_size(), dtable.element_size()
        _name_overlap(2, dtable=(args.dtable, vocab, dim * out_size, dtable_stride * out_size),
                      workspace=(args.workspace, 1, args.workspace_bytes, 0),
                      dout=(args.dout, n, dim * size, dout_stride * size), tokens=(ids, 1, n * 8, 0))
    N.check("ks_embedding_grad_launch", status)
    return dtable


class GradClipper:
    """Global norm and clipping of a fixed set of gradients.

    `grads`: dense CUDA tensors in bf16, fp16 or fp32; `out`: where the scaled
    gradients go, one tensor of the same type and size each (default: in place).
    The table of work is made once, here, and holds the tensors' addresses: make
    a new clipper when gradients move.  ``clip(max_norm)`` enqueues both passes
    and returns the norm before clipping (fp32, one value, on the device).  The
    partial sums live in the clipper: calls of one clipper must not overlap on
    the GPU (as calls that scale the same gradients must not).  A clipper may be
    dropped while its calls still run, on whatever stream; one whose calls were
    captured in a CUDA graph has to live as long as the graph.
    """

    def __init__(self, grads, out=None):
        self.grads = list(grads)
        self.out = self.grads if out is None else list(out)
        if len(self.out) != len(self.grads):
            raise ValueError("grads and out differ in length")
        if not self.grads:
            raise ValueError("no gradients")
        self.device = self.grads[0].device
        for g, o in zip(self.grads, self.out):
            for t in (g, o):
                if not (t.is_cuda and t.device == self.device and t.dtype in _DT_TRAIN and t.is_contiguous()):
                    raise ValueError("gradients must be contiguous bf16, fp16 or fp32 tensors on one CUDA device")
            if o.dtype != g.dtype or o.numel() != g.numel():
                raise ValueError("an output differs in type or size from its gradient")
        # a tensor twice, or two that overlap, would be counted and scaled twice
        spans = sorted({(t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), i)
                        for i, pair in enumerate(zip(self.grads, self.out)) for t in pair if t.numel()})
        if any(b[0] < a[1] for a, b in zip(spans, spans[1:])):
            raise ValueError("gradients (or outputs) overlap")
        n = len(self.grads)
        tensors = (N.GradTensor * n)(*[N.GradTensor(g.data_ptr(), o.data_ptr(), g.numel(), _DT_TRAIN[g.dtype])
                                       for g, o in zip(self.grads, self.out)])
        size, chunks = C.c_size_t(0), C.c_int64(0)
        N.check("ks_grad_clip_plan", N.lib.ks_grad_clip_plan(tensors, n, None, 0, C.byref(size), C.byref(chunks)))
        host = torch.empty(max(32, size.value), dtype=torch.uint8)
        N.check("ks_grad_clip_plan", N.lib.ks_grad_clip_plan(tensors, n, host.data_ptr(), host.numel(), C.byref(size),
                                                             C.byref(chunks)))
        need = C.c_size_t(0)
        N.check("ks_grad_clip_workspace_bytes", N.lib.ks_grad_clip_workspace_bytes(chunks.value, C.byref(need)))
        self._table = host.to(self.device)
        self._scratch = torch.empty(need.value, dtype=torch.uint8, device=self.device)
        self._index = self.device.index
        self._streams = {_raw_stream(None, self._index)}  # whose pool the table and the scratch come from
        self._args = N.GradClipArgs(self._table.data_ptr(), chunks.value, 0.0, 0.0, None, self._scratch.data_ptr(),
                                    need.value)

    def clip(self, max_norm: float, eps: float = 1e-6, stream=None) -> torch.Tensor:
        if self._index != torch.cuda.current_device():
            raise ValueError(f"the gradients are on {self.device}, not on the current device")
        norm = _empty(self._scratch, 1, torch.float32, stream)
        raw = _raw_stream(stream, self._index)
        if raw not in self._streams:
            # the clipper may be dropped with this call still queued there, and what it alone
            # keeps alive must not be given to another tensor before
            user = torch.cuda.current_stream(self.device) if stream is None else stream
            for t in (self._table, self._scratch, *self.grads, *self.out):
                t.record_stream(user)
            self._streams.add(raw)
        args = N.GradClipArgs.from_buffer_copy(self._args)  # another host thread may be in here too
        args.max_norm, args.eps, args.norm = max_norm, eps, norm.data_ptr()
        N.check("ks_grad_clip_launch", N.lib.ks_grad_clip_launch(C.byref(args), raw))
        return norm


def device_error_take() -> int:
    w = C.c_int(0)
    N.check("ks_device_error_take", N.lib.ks_device_error_take(C.byref(w)))
    return w.value


def _copy(dst: torch.Tensor, src: torch.Tensor, stream) -> None:
    """One async copy through the C ABI (pinned host <-> device, either way)."""
    n = src.numel() * src.element_size()
    sp = _stream_ptr(stream)
    if dst.is_cuda:
        N.check("ks_gpu_memcpy_htod", N.lib.ks_gpu_memcpy_htod(C.c_void_p(dst.data_ptr()),
                                                               C.c_void_p(src.data_ptr()), n, sp))
    else:
        N.check("ks_gpu_memcpy_dtoh", N.lib.ks_gpu_memcpy_dtoh(C.c_void_p(dst.data_ptr()),
                                                               C.c_void_p(src.data_ptr()), n, sp))


class HostRowPipeline:
    """Row-wise families on host-resident data: rows move in chunks through
    three streams -- host-to-device copy, kernel, device-to-host copy -- so the
    copy of one chunk's input, the kernel on the previous chunk and the copy
    of an earlier chunk's output overlap (PCIe moves both directions at once).

    ``step(host_in, dev_in, host_out, dev_out, launch)`` runs one pass over all
    rows: ``host_in`` / ``dev_in`` are matching [rows, ...] tensors (pinned
    host, device), ``launch(r0, r1, stream)`` enqueues the family on rows
    [r0, r1) of the device tensors, and the result lands in ``host_out``.
    Consecutive steps pipeline as well; a chunk's device buffers are reused
    only after the previous step's kernel and output copy are done with them.
    Returns an event that completes when this step's output is on the host.

    The default is two chunks per step: because consecutive steps pipeline,
    larger chunks lose nothing to filling the pipeline and pay the per-copy
    cost less often (measured on B200 for softmax 4096x8192 over 20 steps:
    95.1 GB/s with 2 chunks, 92.7 with 4, 87.4 with 8, 79.6 with 16, against
    98 GB/s of bidirectional PCIe copy).
    """

    def __init__(self, rows: int, chunk_rows: int | None = None):
        if chunk_rows is None:
            chunk_rows = (rows + 1) // 2
        self.chunks = [(r, min(rows, r + chunk_rows)) for r in range(0, rows, max(1, chunk_rows))]
        self.s_in, self.s_k, self.s_out = (torch.cuda.Stream() for _ in range(3))
        self.ev_k = [None] * len(self.chunks)
        self.ev_out = [None] * len(self.chunks)

    def step(self, host_in, dev_in, host_out, dev_out, launch):
        for i, (r0, r1) in enumerate(self.chunks):
            if self.ev_k[i] is not None:
                self.s_in.wait_event(self.ev_k[i])  # the last step's kernel has read this chunk
            for h, d in zip(host_in, dev_in):
                _copy(d[r0:r1], h[r0:r1], self.s_in)
            e_in = torch.cuda.Event()
            e_in.record(self.s_in)
            self.s_k.wait_event(e_in)
            if self.ev_out[i] is not None:
                self.s_k.wait_event(self.ev_out[i])  # the last step's output copy has read this chunk
            launch(r0, r1, self.s_k)
            self.ev_k[i] = torch.cuda.Event()
            self.ev_k[i].record(self.s_k)
            self.s_out.wait_event(self.ev_k[i])
            _copy(host_out[r0:r1], dev_out[r0:r1], self.s_out)
            self.ev_out[i] = torch.cuda.Event()
            self.ev_out[i].record(self.s_out)
        return self.ev_out[-1]

    def join(self, stream=None) -> None:
        """Make `stream` (default: current) wait for everything enqueued."""
        s = stream if stream is not None else torch.cuda.current_stream()
        for st in (self.s_in, self.s_k, self.s_out):
            s.wait_stream(st)
