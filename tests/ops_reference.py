"""Plain 64-bit implementations of the training-step operators (mdq_b200.ops),
on the CPU, written from their formulas, and the error bounds the tests use.

Bounds.  u = 2^-24 is the unit roundoff of fp32, 2^-8 that of bf16.  A sum of n
terms in fp32, in whatever order, is off by at most (n - 1) u times the sum of
the terms' magnitudes (first order); pairwise and lane-wise orders stay far
below.  A result rounded to bf16 adds 2^-8 of its magnitude.
"""
import math

import torch

U32 = 2.0 ** -24
U16 = 2.0 ** -8


def d64(t):
    return None if t is None else t.detach().to("cpu", torch.float64)


def rounding(dtype):
    return U16 if dtype == torch.bfloat16 else 2 * U32


# ----------------------------------------------------------------- embedding

def embedding(ids, table, scale):
    ids, table = ids.cpu().long(), d64(table)
    ok = (ids >= 0) & (ids < table.shape[0])
    out = table[torch.where(ok, ids, 0)] * scale
    return torch.where(ok[..., None], out, 0.0)


def embedding_grad(ids, grad_out, vocab, scale, padding_idx=None):
    """The gradient, and the bound on an fp32 sum's error for each element."""
    ids, g = ids.cpu().long().reshape(-1), d64(grad_out)
    g = g.reshape(ids.numel(), g.shape[-1])
    keep = (ids >= 0) & (ids < vocab)
    if padding_idx is not None:
        keep &= ids != padding_idx
    ids, g = ids[keep], g[keep] * scale
    grad = torch.zeros(vocab, g.shape[-1], dtype=torch.float64).index_add_(0, ids, g)
    mag = torch.zeros_like(grad).index_add_(0, ids, g.abs())
    count = torch.zeros(vocab, dtype=torch.float64).index_add_(0, ids, torch.ones(len(ids)).double())
    return grad, (count[:, None] + 2) * U32 * mag


# ------------------------------------------------------------- residual norm

def norm(v, w, b, eps, kind):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps) * w
    return v if b is None else v + b


def residual_norm(x, h, post_weight, pre_weight, post_bias=None, pre_bias=None, gate=None,
                  residual_scale=1.0, eps=1e-5, kind="rms"):
    """Arguments in float64; x and h are [rows, dim]."""
    new = x
    if h is not None:
        y = norm(h, post_weight, post_bias, eps, kind)
        if gate is not None:
            g = gate.reshape(-1, x.shape[-1])
            y = y * g.repeat_interleave(x.shape[0] // g.shape[0], 0)
        new = residual_scale * x + y
    n = None if pre_weight is None else norm(new, pre_weight, pre_bias, eps, kind)
    return new, n


# -------------------------------------------------------------- distillation

def distill_rows(logits, teacher, index, temperature, weight=None, scale=1.0):
    """Losses of the rows in float64, differentiable in ``logits`` (float64)."""
    n, v = logits.shape
    index, t = index.cpu().long(), d64(teacher) / temperature
    ok = (index >= 0) & (index < v)
    t = torch.where(ok, t, -math.inf)
    w = torch.ones(n, dtype=torch.float64) if weight is None else d64(weight)
    live = (t.max(-1).values > -math.inf) & (w != 0)
    rows = torch.zeros(n, dtype=torch.float64)
    if live.any():
        z, t, at = logits[live] / temperature, t[live], torch.where(ok, index, 0)[live]
        log_q = t - torch.logsumexp(t, -1, keepdim=True)
        q = torch.exp(log_q)
        log_p = (z - torch.logsumexp(z, -1, keepdim=True)).gather(1, at)
        part = torch.where(q > 0, q * (torch.where(q > 0, log_q, 0.0) -
                                       torch.where(q > 0, log_p, 0.0)), 0.0)
        rows = rows.index_put((live.nonzero()[:, 0],),
                              temperature ** 2 * scale * w[live] * part.sum(-1))
    return rows
