"""An attention block with a learned relative-position bias, forward and backward.

The matrix products are torch's; the row work between them runs as ask_b200 plans:

    x = dropout(embedding)
    u = norm(x)                                              block_norm, pre norm alone
    s = (u Wq) (u Wk)^T;  p = D(softmax(scale s + bias))     bias_softmax
    y = (p (u Wv)) Wo
    h = x + D(gate * norm(y));  z = norm(h)                  block_norm, post norm, gate, dropout and pre norm

``python examples/encoder_block.py`` runs one step on the GPU and prints the loss and the gradients' norms.  Each
dropout has a stream of its own; all share the seed tensor {seed, offset}, which a training loop advances by
:attr:`EncoderBlock.offset_step` a step, so that every step draws new masks.
"""
from __future__ import annotations

import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import ask_b200  # noqa: E402
from ask_b200 import recipes as R  # noqa: E402


class EncoderBlock:
    """One block for [batch, tokens, width] activations of type `dtype` (f32, f16 or bf16)."""

    EMBEDDING, PROBABILITIES, BRANCH = range(3)  # dropout streams

    def __init__(self, batch: int, tokens: int, width: int, heads: int, dtype: str = "bf16", dropout: float = 0.1,
                 buckets: int = 32, max_distance: int = 128, device: int = 0):
        self.shape = (batch, tokens, width, heads)
        self.type = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype]
        self.device = device
        rows = batch * tokens
        #: blocks of random words that a step may draw: those of its largest dropout
        self.offset_step = (max(rows * width, batch * heads * tokens * tokens) + 3) // 4
        bias = dict(thresholds=R.bucket_thresholds(buckets, max_distance), bidirectional=True,
                    scale=1 / math.sqrt(width // heads), lengths=True, dropout=dropout, stream_id=self.PROBABILITIES)
        join = dict(gate_groups=1, dropout=dropout, stream_id=self.BRANCH)
        plan = lambda recipe: ask_b200.Plan(recipe, device)  # noqa: E731
        self.embed = plan(R.dropout(dtype, rows * width, dropout, stream_id=self.EMBEDDING))
        self.first = plan(R.block_norm(dtype, rows, width, branch=False))
        self.softmax = plan(R.bias_softmax(dtype, batch, heads, tokens, tokens, **bias))
        self.join = plan(R.block_norm(dtype, rows, width, **join))
        self.first_grad = plan(R.block_norm_grad(dtype, rows, width, branch=False))
        self.softmax_grad = plan(R.bias_softmax_grad(dtype, batch, heads, tokens, tokens, **bias))
        self.join_grad = plan(R.block_norm_grad(dtype, rows, width, **join))
        plans = (self.first_grad, self.softmax_grad, self.join_grad)
        self.scratch = self._empty(max(p.scratch_bytes for p in plans), dtype=torch.uint8)
        g = torch.Generator(device=f"cuda:{device}").manual_seed(1)
        normal = lambda *s, std: torch.randn(*s, generator=g, device=f"cuda:{device}") * std  # noqa: E731
        self.weights = {k: normal(width, width, std=width**-0.5).to(self.type) for k in ("q", "k", "v", "o")}
        self.table = normal(buckets, heads, std=0.5)
        self.w_first, self.w_post, self.w_pre, self.gate = (torch.ones(width, device=f"cuda:{device}") for _ in range(4))

    def _empty(self, *shape, dtype=None):
        return torch.empty(*shape, dtype=dtype or self.type, device=f"cuda:{self.device}")

    def _run(self, plan, inputs, outputs):
        plan.launch(inputs, outputs, self.scratch if plan.scratch_bytes else None, torch.cuda.current_stream())

    def _heads(self, t):  # [rows, width] -> [batch, heads, tokens, width / heads]
        b, n, d, h = self.shape
        return t.view(b, n, h, d // h).transpose(1, 2)

    def _rows(self, t):
        b, n, d, h = self.shape
        return t.transpose(1, 2).reshape(b * n, d)

    def forward(self, embedding, lengths, seed):
        """z [rows, width]; what backward() needs is kept in `self.saved`."""
        b, n, d, h = self.shape
        f32 = torch.float32
        x, u, r1 = self._empty(b * n, d), self._empty(b * n, d), self._empty(b * n, dtype=f32)
        self._run(self.embed, [embedding, seed], [x])
        self._run(self.first, [x, self.w_first], [u, r1])
        q, k, v = (self._heads(u @ self.weights[name]) for name in "qkv")
        s = (q @ k.transpose(2, 3)).contiguous()
        p, lse = self._empty(b, h, n, n), self._empty(b, h, n, dtype=f32)
        self._run(self.softmax, [s, self.table, lengths, seed], [p, lse])
        mixed = self._rows(p @ v)
        y = mixed @ self.weights["o"]
        out, z, r2, r3 = self._empty(b * n, d), self._empty(b * n, d), self._empty(b * n, dtype=f32), self._empty(b * n, dtype=f32)
        self._run(self.join, [x, y, self.w_post, self.gate, self.w_pre, seed], [out, z, r2, r3])
        self.saved = (x, u, r1, q, k, v, s, p, lse, mixed, y, out, r2, r3, lengths, seed)
        return z

    def backward(self, dz):
        """Gradients of sum(dz * z): of the embedding, the weights, the bias table, the norms' weights and the gate."""
        b, n, d, h = self.shape
        f32 = torch.float32
        x, u, r1, q, k, v, s, p, lse, mixed, y, out, r2, r3, lengths, seed = self.saved
        g = {name: self._empty(d, dtype=f32) for name in ("w_first", "w_post", "gate", "w_pre")}
        g["table"] = self._empty(*self.table.shape, dtype=f32)
        dx, dy = self._empty(b * n, d), self._empty(b * n, d)
        self._run(self.join_grad, [torch.zeros_like(dz), dz, out, y, self.w_post, self.gate, self.w_pre, r2, r3, seed],
                  [dx, dy, g["w_post"], g["gate"], g["w_pre"]])
        g["o"] = mixed.t() @ dy
        dmixed = self._heads(dy @ self.weights["o"].t())
        dp, dv = (dmixed @ v.transpose(2, 3)).contiguous(), p.transpose(2, 3) @ dmixed
        ds = self._empty(b, h, n, n)
        self._run(self.softmax_grad, [s, dp, lse, self.table, lengths, seed], [ds, g["table"]])
        parts = {"q": self._rows(ds @ k), "k": self._rows(ds.transpose(2, 3) @ q), "v": self._rows(dv)}
        for name, part in parts.items():
            g[name] = u.t() @ part
        du = sum(part @ self.weights[name].t() for name, part in parts.items())
        through = self._empty(b * n, d)
        self._run(self.first_grad, [du, x, self.w_first, r1], [through, g["w_first"]])
        dx = dx + through
        g["embedding"] = self._empty(b * n, d)
        self._run(self.embed, [dx, seed], [g["embedding"]])  # the gradient of dropout is dropout with its own mask
        return g


def main() -> None:
    batch, tokens, width, heads = 4, 512, 1024, 16
    block = EncoderBlock(batch, tokens, width, heads)
    embedding = torch.randn(batch * tokens, width, device="cuda").to(block.type)
    lengths = torch.tensor([tokens, tokens, tokens // 2, tokens // 3], dtype=torch.int32, device="cuda")
    seed = torch.tensor([2024, 0], dtype=torch.int64, device="cuda")
    for step in range(2):
        z = block.forward(embedding, lengths, seed)
        loss = z.float().square().mean()
        grads = block.backward((z.float() * (2 / z.numel())).to(z.dtype))
        seed[1] += block.offset_step
        print(f"step {step}: loss {float(loss):.4f}  " + "  ".join(f"|d{k}| {float(v.float().norm()):.3e}" for k, v in grads.items()))


if __name__ == "__main__":
    main()
