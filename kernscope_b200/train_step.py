"""A training step at the vocabulary end, with the library's operators in order:

    h = scale * table[tokens]                      ops.embedding
    loss, dh, dw = cross entropy of h w^T          ops.linear_cross_entropy_grad
    dtable = scale * sum of dh by token            ops.embedding_backward
    norm, gradients scaled to max_norm             ops.GradClipper
    table, w -= lr * gradient

The model is the smallest that uses them all: next-token prediction from the
current token alone, through embeddings of `dim` values (with ``--tied`` one
table serves both ends, and the lookup's gradient is added to the loss's).  The
text is synthetic: every token has a few likely successors.

    python -m kernscope_b200.train_step --tokens 8192 --dim 256 --vocab 4096 --steps 50
"""

from __future__ import annotations

import argparse
import math
import sys

import torch

from . import ops


class VocabModel:
    """Parameters, gradient buffers and the step."""

    def __init__(self, vocab: int, dim: int, dtype=torch.bfloat16, tied: bool = False, seed: int = 0):
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed)
        self.tied, self.scale = tied, math.sqrt(dim)
        draw = lambda: (torch.randn(vocab, dim, generator=gen, device="cuda") / math.sqrt(dim))  # noqa: E731
        # fp32 masters, 16-bit copies for the operators
        self.master = [draw()] if tied else [draw(), draw()]
        self.param = [m.to(dtype) for m in self.master]
        self.grad = [torch.empty_like(p) for p in self.param]
        self.clipper = ops.GradClipper(self.grad)

    def gradients(self, tokens: torch.Tensor, targets: torch.Tensor, ignore_index: int = -100) -> torch.Tensor:
        """Loss (one value, on the device); the gradients land in ``self.grad``."""
        table, w = self.param[0], self.param[-1]
        h = ops.embedding(tokens, table, scale=self.scale)
        loss, dh, _ = ops.linear_cross_entropy_grad(h, w, targets, ignore_index=ignore_index, dw=self.grad[-1])
        ops.embedding_backward(tokens, dh, table.shape[0], scale=self.scale, dtable=self.grad[0], accumulate=self.tied)
        return loss

    def step(self, tokens, targets, lr: float, max_norm: float = 1.0, ignore_index: int = -100):
        """One step; (loss, gradient norm before clipping), on the device."""
        loss = self.gradients(tokens, targets, ignore_index)
        norm = self.clipper.clip(max_norm)
        for m, p, g in zip(self.master, self.param, self.grad):
            m.sub_(g, alpha=lr)
            p.copy_(m)
        return loss, norm


def synthetic_text(vocab: int, tokens: int, seed: int, branches: int = 4):
    """(tokens, targets): independent pairs of a token and one of its few successors."""
    gen = torch.Generator()
    gen.manual_seed(1)
    after = torch.randint(0, vocab, (vocab, branches), generator=gen)
    gen.manual_seed(seed)
    first = torch.randint(0, vocab, (tokens,), generator=gen)
    second = after[first, torch.randint(0, branches, (tokens,), generator=gen)]
    return first.cuda(), second.cuda()


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--tokens", type=int, default=8192)
    ap.add_argument("--dim", type=int, default=256)
    ap.add_argument("--vocab", type=int, default=4096)
    ap.add_argument("--steps", type=int, default=50)
    ap.add_argument("--lr", type=float, default=10.0)
    ap.add_argument("--max-norm", type=float, default=1.0)
    ap.add_argument("--dtype", default="bf16", choices=("bf16", "fp16"))
    ap.add_argument("--tied", action="store_true")
    a = ap.parse_args(argv)
    torch.cuda.set_device(0)
    model = VocabModel(a.vocab, a.dim, {"bf16": torch.bfloat16, "fp16": torch.float16}[a.dtype], a.tied)
    for i in range(a.steps):
        tokens, targets = synthetic_text(a.vocab, a.tokens, seed=100 + i)
        loss, norm = model.step(tokens, targets, a.lr, a.max_norm)
        if i % 10 == 0 or i + 1 == a.steps:
            print(f"step {i:4d}  loss {float(loss):.4f}  gradient norm {float(norm):.3f}")
    return 0


if __name__ == "__main__":
    sys.exit(main())
