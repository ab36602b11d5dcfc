"""Trains a small language model on the training-step operators and the quantised
AdamW step: tokens are embedded by ``scaled_embedding``, blocks are joined by
``residual_norm`` (a norm behind each block, a learned gate, the norm before the
next), the head is tied to the table, and the loss is ``topk_distill`` against a
teacher's top logits, whose gradient overwrites the logits.

The teacher is a fixed table of next-token logits, so that a run needs no data:

    python stream-mm2026_b200/examples/distill_lm.py --steps 200
"""
from __future__ import annotations

import argparse
import math
import sys
from pathlib import Path

import torch
import torch.nn.functional as F
from torch import nn

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
from mdq_b200 import MDQAdamWSimpleFusedIO, ops  # noqa: E402


class Block(nn.Module):
    """Causal attention beside a gated MLP, both from the normed input."""

    def __init__(self, dim: int, heads: int):
        super().__init__()
        self.heads = heads
        self.qkv = nn.Linear(dim, 3 * dim, bias=False)
        self.up = nn.Linear(dim, 4 * dim, bias=False)
        self.out = nn.Linear(3 * dim, dim, bias=False)

    def forward(self, n):
        batch, length, dim = n.shape
        q, k, v = (t.view(batch, length, self.heads, -1).transpose(1, 2)
                   for t in self.qkv(n).chunk(3, -1))
        a = F.scaled_dot_product_attention(q, k, v, is_causal=True)
        gate, up = self.up(n).chunk(2, -1)
        return self.out(torch.cat((a.transpose(1, 2).reshape(n.shape), F.silu(gate) * up), -1))


class SmallLM(nn.Module):
    def __init__(self, vocab: int, dim: int, layers: int, heads: int):
        super().__init__()
        self.table = nn.Parameter(torch.randn(vocab, dim) / math.sqrt(dim))
        self.blocks = nn.ModuleList(Block(dim, heads) for _ in range(layers))
        # norm 0 stands before the first block, norm k behind block k - 1
        self.pre = nn.ParameterList(torch.ones(dim) for _ in range(layers + 1))
        self.post = nn.ParameterList(torch.ones(dim) for _ in range(layers))
        self.gate = nn.ParameterList(torch.full((dim,), 0.5) for _ in range(layers))

    def forward(self, ids):
        """bf16 logits; the residual stream stays in fp32."""
        scale = math.sqrt(self.table.shape[1])
        x = ops.scaled_embedding(ids, self.table, scale, out_dtype=torch.float32)
        x, n = ops.residual_norm(x, None, None, self.pre[0])
        with torch.autocast("cuda", torch.bfloat16):
            for k, block in enumerate(self.blocks):
                x, n = ops.residual_norm(x, block(n), self.post[k], self.pre[k + 1],
                                         gate=self.gate[k])
            return n @ self.table.t()


class Teacher:
    """The top entries of fixed next-token logits for every token."""

    def __init__(self, vocab: int, top: int, device, seed: int = 1):
        g = torch.Generator(device=device).manual_seed(seed)
        self.index = torch.rand(vocab, vocab, generator=g, device=device).argsort(-1)[:, :top].contiguous()
        self.logits = 2 * torch.randn(vocab, top, generator=g, device=device)

    def __call__(self, ids):
        return self.logits[ids], self.index[ids]


def train(steps: int = 200, vocab: int = 512, dim: int = 128, layers: int = 2, heads: int = 4,
          batch: int = 16, length: int = 64, top: int = 16, temperature: float = 1.5,
          lr: float = 3e-3, seed: int = 0, every: int = 20, say=print):
    """Runs ``steps`` steps and returns the mean loss of each."""
    torch.manual_seed(seed)
    device = torch.device("cuda")
    model = SmallLM(vocab, dim, layers, heads).to(device)
    teacher = Teacher(vocab, top, device)
    # (the optimizer's time constant grows with the logarithm of the layers, which is 0 for one)
    optimizer = MDQAdamWSimpleFusedIO(model.parameters(), lr=lr, weight_decay=0.0, block_size=256,
                                      layer_count=max(2, layers), batch_size=batch)
    losses, padded = [], length // 8
    for step in range(steps):
        ids = torch.randint(0, vocab, (batch, length), device=device)
        weight = torch.ones(batch, length, device=device)
        weight[:, length - padded:] = 0       # as a batch's padding would be
        logits = model(ids)
        at = logits.detach()
        result = ops.topk_distill(at, *teacher(ids), temperature=temperature, weight=weight,
                                  scale=1.0 / (batch * (length - padded)), out=at)
        logits.backward(result.grad)
        optimizer.step()
        optimizer.zero_grad()
        losses.append(result.loss)
        if every and (step % every == 0 or step == steps - 1):
            say(f"step {step:5d}  loss {float(result.loss):.4f}")
    return [float(v) for v in torch.stack(losses).cpu()] if losses else []


def main(argv=None):
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawTextHelpFormatter)
    for name, value in (("steps", 200), ("vocab", 512), ("dim", 128), ("layers", 2), ("heads", 4),
                        ("batch", 16), ("length", 64), ("top", 16), ("seed", 0), ("every", 20)):
        parser.add_argument(f"--{name}", type=int, default=value, help=f"default {value}")
    parser.add_argument("--temperature", type=float, default=1.5)
    parser.add_argument("--lr", type=float, default=3e-3)
    train(**vars(parser.parse_args(argv)))


if __name__ == "__main__":
    main()
