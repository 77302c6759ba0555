"""Measured cases of the training operators at the vocabulary end of a language model.

Five entry points of ``kernscope_b200.ops`` are covered, each in a plain torch
form (32-bit arithmetic, one rounding at the end) and as the library's call:

* ``score``      -- per-token loss and log-sum-exp of a linear layer over the
  vocabulary, ``ops.linear_cross_entropy``;
* ``loss_grad``  -- the mean loss over the tokens that count, with the
  gradients of the hidden states and of the vocabulary weights,
  ``ops.linear_cross_entropy_grad``;
* ``embed``      -- scaled rows of the token table, ``ops.embedding``;
* ``embed_grad`` -- the table's dense gradient, ``ops.embedding_backward``;
* ``clip``       -- the global norm over many gradients and the gradients
  scaled to at most ``max_norm``, ``ops.GradClipper``.

A case is a dict: ``op``, ``dtype`` and the op's sizes (``tokens``, ``dim``,
``vocab``; for ``clip`` ``tensors``, ``total`` elements and ``align``, the
multiple of elements at which each tensor of the flat buffer begins; ``layout``
draws the tensors' sizes).  ``pad`` is the distance in elements between the end
of one row of hidden states (or of the incoming gradient) and the next.
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

IGNORE = -100  # the target of a token that has no loss
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # a handful of candidate tokens scored against the whole vocabulary: bound by reading the weights
        dict(name="score_few", op="score", dtype="bf16", tokens=16, dim=1024, vocab=32000, pad=0),
        # perplexity of a batch of held-out text in half precision
        dict(name="score_eval", op="score", dtype="fp16", tokens=4096, dim=2048, vocab=65536, pad=0),
        # a fine-tuning step on one short, ragged sequence with a small odd vocabulary
        dict(name="loss_grad_ragged", op="loss_grad", dtype="fp16", tokens=333, dim=1000, vocab=10007, pad=24),
        # an ordinary training micro-batch
        dict(name="loss_grad_step", op="loss_grad", dtype="bf16", tokens=4096, dim=2048, vocab=32768, pad=0),
        # the largest: a long micro-batch of a wide model with a multilingual vocabulary
        dict(name="loss_grad_large", op="loss_grad", dtype="bf16", tokens=8192, dim=4096, vocab=131072, pad=0),
        # one token for each of a batch of requests that are being generated
        dict(name="embed_decode", op="embed", dtype="bf16", tokens=64, dim=2048, vocab=32000, pad=0),
        # a packed batch of training text
        dict(name="embed_train", op="embed", dtype="bf16", tokens=65536, dim=4096, vocab=131072, pad=0),
        # the gradient of a short sequence into a small table, odd sizes
        dict(name="embed_grad_ragged", op="embed_grad", dtype="fp16", tokens=777, dim=1001, vocab=5003, pad=7),
        # the gradient of an ordinary micro-batch
        dict(name="embed_grad_step", op="embed_grad", dtype="bf16", tokens=8192, dim=2048, vocab=32768, pad=0),
        # a packed batch with a table kept in 32 bits
        dict(name="embed_grad_large", op="embed_grad", dtype="fp32", tokens=131072, dim=1024, vocab=131072, pad=0),
        # the adapters of a fine-tuned model: many small gradients, packed without gaps
        dict(name="clip_adapters", op="clip", dtype="fp32", tensors=48, total=600_011, align=1, layout=3),
        # the gradients of a billion-parameter model, 16-bit matrices beside 32-bit vectors
        dict(name="clip_model", op="clip", dtype="mixed", tensors=61, total=1 << 30, align=16, layout=5),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["score", "loss_grad", "loss_grad", "embed", "embed_grad", "embed_grad", "clip"])
    if op == "clip":
        return dict(op=op, dtype=rng.choice(["bf16", "fp16", "fp32", "mixed"]), tensors=rng.randint(1, 61),
                    total=_log_uniform(rng, 1000, 1 << 29), align=rng.choice([1, 8, 16]), layout=rng.randint(0, 1 << 20))
    dtypes = ["bf16", "fp16"] if op in ("score", "loss_grad") else ["bf16", "fp16", "fp32"]
    dim = _log_uniform(rng, 64, 4096)
    if rng.random() < 0.75:
        dim = max(64, dim // 8 * 8)
    tokens = _log_uniform(rng, 1, 8192 if op in ("score", "loss_grad") else 131072)
    return dict(op=op, dtype=rng.choice(dtypes), tokens=tokens, dim=dim, vocab=_log_uniform(rng, 100, 131072),
                pad=rng.choice([0, 0, 8, 5]))


def _sizes(case):
    """Elements of each tensor, and where it begins in its type's flat buffer."""
    r = random.Random(case["layout"])
    weight = [10 ** r.uniform(0, 3) for _ in range(case["tensors"])]
    unit = case["total"] / sum(weight)
    sizes = [max(1, int(v * unit)) for v in weight]
    names = [("fp32" if i % 3 == 2 else "bf16") if case["dtype"] == "mixed" else case["dtype"] for i in range(len(sizes))]
    at, places = {}, []
    for n, name in zip(sizes, names):
        first = -(-at.get(name, 0) // case["align"]) * case["align"]
        places.append((name, first, n))
        at[name] = first + n
    return places, at


def _zipf(vocab):
    """Probability of each token id: frequent tokens have low ids, as in a trained tokenizer."""
    p = 1.0 / (np.arange(vocab, dtype=np.float64) + 2.7)
    return p / p.sum()


def _tokens(gen, n, vocab):
    cdf = torch.from_numpy(np.cumsum(_zipf(vocab))).cuda()
    u = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)
    return torch.searchsorted(cdf, u).clamp_(max=vocab - 1)


def _rows(gen, n, dim, pad, dtype):
    """[n, dim] of normal values whose rows lie dim + pad elements apart."""
    return torch.randn(n, dim + pad, generator=gen, device="cuda").to(dtype)[:, :dim]


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    op = case["op"]
    if op == "clip":
        places, at = _sizes(case)
        target = 10 ** random.Random(seed).uniform(-0.3, 1.3)  # the norm that comes out: clipped, mostly
        unit = target / math.sqrt(sum(n for _, _, n in places))
        flat = {name: torch.randn(n, generator=gen, device="cuda").mul_(unit).to(DTYPES[name]) for name, n in sorted(at.items())}
        out = {name: torch.empty_like(t) for name, t in flat.items()}
        for name in out:
            out[name].zero_()  # the gaps between tensors stay zero
        return {"op": op, "max_norm": 1.0, "flat_out": out, "grads": [flat[name][a:a + n] for name, a, n in places],
                "outs": [out[name][a:a + n] for name, a, n in places]}
    n, dim, vocab, dtype = case["tokens"], case["dim"], case["vocab"], DTYPES[case["dtype"]]
    tokens = _tokens(gen, n, vocab)
    if op == "embed":
        return {"op": op, "tokens": tokens, "table": torch.randn(vocab, dim, generator=gen, device="cuda").to(dtype), "scale": math.sqrt(dim)}
    if op == "embed_grad":
        return {"op": op, "tokens": tokens, "dout": _rows(gen, n, dim, case["pad"], dtype), "vocab": vocab, "scale": math.sqrt(dim)}
    # Rows of hidden states that lean towards their target's weights: probabilities of the target from 1/vocab to near one.
    w = (torch.randn(vocab, dim, generator=gen, device="cuda") / math.sqrt(dim)).to(dtype)
    lean = 12 * torch.rand(n, 1, generator=gen, device="cuda")
    h = torch.randn(n, dim + case["pad"], generator=gen, device="cuda")
    h[:, :dim] += lean * w[tokens].float()
    # one token in twenty, of a prompt or of padding, has no loss
    targets = torch.where(torch.rand(n, generator=gen, device="cuda") < 0.05, torch.full_like(tokens, IGNORE), tokens)
    return {"op": op, "h": h.to(dtype)[:, :dim], "w": w, "targets": targets}


def _plain_loss(h, w, targets):
    logits = h.float() @ w.float().t()
    top = logits.max(dim=1, keepdim=True).values
    e = torch.exp(logits - top)
    s = e.sum(dim=1, keepdim=True)
    lse = (torch.log(s) + top)[:, 0]
    counts = targets != IGNORE
    at = torch.where(counts, targets, torch.zeros_like(targets))
    loss = torch.where(counts, lse - logits.gather(1, at[:, None])[:, 0], torch.zeros_like(lse))
    return loss, lse, counts, at, e, s


def _plain(s):
    op = s["op"]
    if op == "score":
        loss, lse = _plain_loss(s["h"], s["w"], s["targets"])[:2]
        return loss, lse
    if op == "loss_grad":
        loss, _, counts, at, e, total = _plain_loss(s["h"], s["w"], s["targets"])
        n = counts.sum().clamp(min=1).float()
        d = e.div_(total)
        d[torch.arange(d.shape[0], device=d.device), at] -= 1.0
        d *= (counts.float() / n)[:, None]
        return (loss.sum() / n).reshape(1), (d @ s["w"].float()).to(s["w"].dtype), (d.t() @ s["h"].float()).to(s["w"].dtype)
    if op == "embed":
        return (s["table"][s["tokens"]].float() * s["scale"]).to(s["table"].dtype)
    if op == "embed_grad":
        total = torch.zeros(s["vocab"], s["dout"].shape[1], device="cuda")
        total.index_add_(0, s["tokens"], s["dout"].float())
        return (total * s["scale"]).to(s["dout"].dtype)
    norm = torch.stack([g.float().square().sum() for g in s["grads"]]).sum().sqrt()
    coef = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    [o.copy_(g.float() * coef) for g, o in zip(s["grads"], s["outs"])]
    return norm.reshape(1), s["flat_out"]


def run(state):
    if not own:
        return _plain(state)
    from kernscope_b200 import ops

    s, op = state, state["op"]
    if op == "score":
        return ops.linear_cross_entropy(s["h"], s["w"], s["targets"], ignore_index=IGNORE, reduction="none")
    if op == "loss_grad":
        return ops.linear_cross_entropy_grad(s["h"], s["w"], s["targets"], ignore_index=IGNORE, reduction="mean")
    if op == "embed":
        return ops.embedding(s["tokens"], s["table"], scale=s["scale"])
    if op == "embed_grad":
        return ops.embedding_backward(s["tokens"], s["dout"], s["vocab"], scale=s["scale"])
    if "clipper" not in s:  # a training program makes this once, for the buffers that its gradients live in
        s["clipper"] = ops.GradClipper(s["grads"], out=s["outs"])
    return s["clipper"].clip(s["max_norm"]), s["flat_out"]


def work(case):
    op = case["op"]
    if op == "clip":
        places, _ = _sizes(case)
        return {"bytes": sum(2 * n * SIZE[name] for name, _, n in places), "flops": sum(3 * n for _, _, n in places)}
    n, dim, vocab, size = case["tokens"], case["dim"], case["vocab"], SIZE[case["dtype"]]
    if op == "score":
        return {"bytes": (n + vocab) * dim * size + 16 * n, "flops": 2 * n * vocab * dim}
    if op == "loss_grad":  # the logits and the two products of their gradient
        return {"bytes": 2 * (n + vocab) * dim * size + 8 * n, "flops": 6 * n * vocab * dim}
    if op == "embed":  # each distinct row of the table once
        distinct = float((1 - (1 - _zipf(vocab)) ** n).sum())
        return {"bytes": (n + distinct) * dim * size + 8 * n, "flops": n * dim}
    return {"bytes": (n + vocab) * dim * size + 8 * n, "flops": n * dim}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "clip":
        norm = math.sqrt(sum(float(torch.dot(g.double(), g.double())) for g in s["grads"]))
        coef = min(1.0, s["max_norm"] / (norm + 1e-6))
        for g, o in zip(s["grads"], s["outs"]):
            o.copy_(g)
        return torch.tensor([norm], dtype=torch.float64), {k: v.double() * coef for k, v in s["flat_out"].items()}
    if op == "embed":
        return s["table"].double().index_select(0, s["tokens"]) * s["scale"]
    if op == "embed_grad":
        order = torch.argsort(s["tokens"], stable=True)
        total = torch.zeros(s["vocab"], case["dim"], dtype=torch.float64, device="cuda")
        for part in order.split(16384):
            total.index_add_(0, s["tokens"][part], s["dout"][part].double() * s["scale"])
        return total
    w, targets = s["w"].double(), s["targets"]
    n = max(1, int((targets != IGNORE).sum()))
    losses, lses, dh = [], [], []
    dw = torch.zeros_like(w) if op == "loss_grad" else None
    for a in range(0, case["tokens"], 2048):  # rows at a time: their logits take vocab * 16 KiB each
        h, t = s["h"][a:a + 2048].double(), targets[a:a + 2048]
        valid = (t != IGNORE).double()
        hot = torch.arange(len(t), device="cuda")
        logits = h @ w.t()
        lse = torch.logsumexp(logits, dim=1)
        losses.append((lse - logits[hot, t.clamp(min=0)]) * valid)
        lses.append(lse)
        if op == "loss_grad":
            p = logits.sub_(lse[:, None]).exp_()
            p[hot, t.clamp(min=0)] -= 1
            p *= valid[:, None] / n
            dh.append(p @ w)
            dw.addmm_(p.t(), h)
    if op == "score":
        return torch.cat(losses), torch.cat(lses)
    return (torch.cat(losses).sum() / n).reshape(1), torch.cat(dh), dw
