"""Cases, plain forms and 64-bit values of the training-step operators.

Three operators, each with what it needs in training and for single tokens:

  embed    scaled embedding lookup and its gradient by sorted tokens
  norm     the norm after a block with its gate and the residual's scale, and
           the norm before the next block, forward and backward
  distill  distillation from a teacher's top logits, loss and gradient

Shapes are those of this repository's models (GPT-2 small: vocabulary 50257,
width 768; LLaMA-7B: vocabulary 32000, width 4096) and generic ones.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "bf16": 2}
_EPS = 1e-5


def _ops():
    """The framework's operators (its package lies beside this folder)."""
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "stream-mm2026_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from mdq_b200 import ops
    return ops


_loaded = None


def _framework():
    global _loaded
    if _loaded is None:
        _loaded = _ops()
    return _loaded


# ------------------------------------------------------------------- cases

def _embed(name, tokens, vocab, dim, table="f32", act="bf16", ids="int64", train=True,
           accumulate=False, pad=0.0, scale=1.0):
    return {"name": name, "op": "embed", "tokens": tokens, "vocab": vocab, "dim": dim,
            "table": table, "act": act, "ids": ids, "train": train, "accumulate": accumulate,
            "pad": pad, "scale": scale}


def _norm(name, rows, dim, kind="rms", x="bf16", h="bf16", params="bf16", gate="vector", seqs=1,
          train=True, residual_scale=1.0):
    return {"name": name, "op": "norm", "rows": rows, "dim": dim, "kind": kind, "x": x, "h": h,
            "params": params, "gate": gate, "seqs": seqs, "train": train,
            "residual_scale": residual_scale}


def _distill(name, rows, vocab, top, logits="bf16", teacher="f32", ids="int64", train=True,
             masked=0.0, temperature=2.0, row_pad=0):
    return {"name": name, "op": "distill", "rows": rows, "vocab": vocab, "top": top,
            "logits": logits, "teacher": teacher, "ids": ids, "train": train, "masked": masked,
            "temperature": temperature, "row_pad": row_pad}


def listed():
    return [
        # Generation: the next token of 8 sequences enters the model.
        _embed("embed 8 tokens", 8, 50257, 768, train=False),
        # A GPT-2 small micro-batch of 8 x 256 tokens; fp32 parameters under autocast.
        _embed("embed 8x256 gpt2", 2048, 50257, 768),
        # The same model at 16 x 1024 tokens, ragged sequences padded at the end.
        _embed("embed 16x1024 gpt2 padded", 16384, 50257, 768, ids="int32", pad=0.2),
        # LLaMA-7B, 4 x 2048 tokens of a later micro-batch: the gradient is added to the buffer.
        _embed("embed 4x2048 llama added", 8192, 32000, 4096, table="f32", accumulate=True,
               scale=64.0),
        # Generation with a LLaMA-7B: one token of 8 sequences passes a block's end.
        _norm("norm 8 tokens llama", 8, 4096, train=False),
        # GPT-2 small, 8 x 256 tokens: layer norms, fp32 residual stream, bf16 blocks.
        _norm("norm 8x256 gpt2 layer", 2048, 768, kind="layer", x="f32", params="f32",
              residual_scale=0.9),
        # LLaMA-7B, 8 x 2048 tokens, all in bf16.
        _norm("norm 8x2048 llama rms", 16384, 4096),
        # An odd width and rows that no tile divides, a gate for each of 3 sequences, fp32.
        _norm("norm 3x341 odd width", 1023, 1601, kind="layer", x="f32", h="f32", params="f32",
              gate="sequence", seqs=3),
        # A few positions (one of each of 8 sequences) against a teacher's best 8.
        _distill("distill 8 rows", 8, 50257, 8),
        # GPT-2 small, 8 x 256 positions less the last, prompts masked; best 64 kept.
        _distill("distill 2047 rows masked", 2047, 50257, 64, masked=0.3, ids="int32"),
        # GPT-2 small at 16 x 1024 positions, best 32: the largest logits of a step.
        _distill("distill 16x1024 gpt2", 16384, 50257, 32),
        # Evaluation of a LLaMA-7B student in fp32 on 1 x 2048 positions: the loss alone.
        _distill("distill llama loss only", 2048, 32000, 16, logits="f32", train=False,
                 temperature=1.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    d = _log_int(rng, lo, hi)
    way = rng.random()
    if way < 0.5:
        d = max(64, d // 64 * 64)
    elif way < 0.75:
        d = max(8, d // 8 * 8)
    return d + 64 if d == 3072 else d


def draw(rng):
    op = rng.choice(["embed", "norm", "distill"])
    train = rng.random() < 0.75
    if op == "embed":
        table = rng.choice(["f32", "f32", "bf16"])
        dim = _width(rng, 64, 8192)
        vocab = _log_int(rng, 256, min(131072, (1 << 28) // dim))
        tokens = _log_int(rng, 1, min(32768, (1 << 27) // dim))
        c = _embed("", tokens, vocab, dim, table=table,
                   act="bf16" if table == "bf16" else rng.choice(["bf16", "bf16", "f32"]),
                   ids=rng.choice(["int64", "int32"]), train=train,
                   accumulate=train and table == "f32" and rng.random() < 0.3,
                   pad=rng.choice([0.0, 0.0, 0.3, 0.9]),
                   scale=rng.choice([1.0, round(math.sqrt(dim), 3)]))
    elif op == "norm":
        dim = _width(rng, 64, 16384)
        seqs = rng.choice([1, 2, 3, 8])
        rows = seqs * max(1, _log_int(rng, 1, min(32768, (1 << 26) // dim)) // seqs)
        x, h, params = rng.choice([("bf16", "bf16", "bf16"), ("f32", "bf16", "f32"),
                                   ("f32", "f32", "f32"), ("bf16", "bf16", "f32")])
        gate = rng.choice(["none", "vector", "vector", "sequence"])
        c = _norm("", rows, dim, kind=rng.choice(["rms", "layer"]), x=x, h=h, params=params,
                  gate=gate, seqs=seqs if gate == "sequence" else 1, train=train,
                  residual_scale=rng.choice([1.0, 0.5, 1.7]))
    else:
        vocab = _log_int(rng, 256, 200000)
        rows = _log_int(rng, 1, min(16384, 16384 * 50257 // (2 * vocab)))
        c = _distill("", rows, vocab, min(_log_int(rng, 1, 200), vocab // 2),
                     logits=rng.choice(["bf16", "bf16", "f32"]),
                     teacher=rng.choice(["f32", "bf16"]), ids=rng.choice(["int64", "int32"]),
                     train=train, masked=rng.choice([0.0, 0.0, 0.25, 0.6]),
                     temperature=rng.choice([1.0, 2.0, 4.0]),
                     row_pad=rng.choice([0, 0, -vocab % 64]))
    del c["name"]
    return c


# ------------------------------------------------------------------- inputs

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, scale=1.0, dtype=torch.float32):
    t = torch.empty(shape, device="cuda", dtype=dtype)
    return t.normal_(0.0, scale, generator=g)


def prepare(case, seed):
    g = _generator(seed)
    s = dict(case)
    if case["op"] == "embed":
        n, v, d = case["tokens"], case["vocab"], case["dim"]
        # Word frequencies: the probability of id k falls as 1 / (k + 1).
        u = torch.rand(n, device="cuda", generator=g, dtype=torch.float64)
        ids = (torch.exp(u * math.log(v + 1.0)).long() - 1).clamp_(0, v - 1)
        s["padding_idx"] = None
        padded = int(case["pad"] * n)
        if padded:
            s["padding_idx"] = v - 1
            ids[n - padded:] = v - 1
        s["ids"] = ids.to(torch.int32 if case["ids"] == "int32" else torch.int64)
        s["weights"] = _randn(g, v, d, scale=0.02, dtype=_DT[case["table"]])
        if case["train"]:
            s["grad_out"] = _randn(g, n, d, scale=1e-3, dtype=_DT[case["act"]])
        if case["accumulate"]:
            s["buffer"] = _randn(g, v, d, scale=1e-3)
    elif case["op"] == "norm":
        n, d, pt = case["rows"], case["dim"], _DT[case["params"]]
        x = _randn(g, n, d, scale=1.5)
        x[:, :: max(1, d // 4)] *= 6.0          # a few channels of a residual stream are large
        s["inp"] = x.to(_DT[case["x"]])
        s["block"] = _randn(g, n, d, scale=0.7, dtype=_DT[case["h"]])
        s["post_weight"] = (1 + _randn(g, d, scale=0.1)).to(pt)
        s["pre_weight"] = (1 + _randn(g, d, scale=0.1)).to(pt)
        layer = case["kind"] == "layer"
        s["post_bias"] = _randn(g, d, scale=0.1).to(pt) if layer else None
        s["pre_bias"] = _randn(g, d, scale=0.1).to(pt) if layer else None
        shape = {"none": None, "vector": (d,), "sequence": (case["seqs"], d)}[case["gate"]]
        s["gate_"] = None if shape is None else (0.5 + _randn(g, *shape, scale=0.2)).to(pt)
        if case["train"]:
            s["grad_new"] = _randn(g, n, d, scale=1e-2, dtype=_DT[case["x"]])
            s["grad_n"] = _randn(g, n, d, scale=1e-2, dtype=_DT[case["h"]])
    else:
        n, v, k = case["rows"], case["vocab"], case["top"]
        lt = _DT[case["logits"]]
        z = _randn(g, n, v + case["row_pad"], scale=1.5, dtype=lt)[:, :v]
        # The teacher's best: K distinct ids, where the student's logits are high as well.
        start = torch.randint(0, v, (n, 1), device="cuda", generator=g)
        step = max(1, v // (k + 1))
        idx = (start + torch.arange(k, device="cuda") * step) % v
        fall = torch.linspace(9.0, 2.0, k, device="cuda")
        t = fall + _randn(g, n, k, scale=0.7)
        z.scatter_(1, idx, (fall + _randn(g, n, k, scale=1.0)).to(lt))
        # Rows whose teacher kept fewer than K: the rest of the row is marked absent.
        kept = torch.randint(max(1, k // 2), k + 1, (n, 1), device="cuda", generator=g)
        idx = torch.where(torch.arange(k, device="cuda") < kept, idx, torch.full_like(idx, -1))
        s["z"] = z
        s["t"] = t.to(_DT[case["teacher"]])
        s["idx"] = idx.to(torch.int32 if case["ids"] == "int32" else torch.int64)
        s["weight"] = None
        out = int(case["masked"] * n)
        if out:
            w = torch.ones(n, device="cuda")
            w[torch.randperm(n, device="cuda", generator=g)[:out]] = 0.0
            s["weight"] = w
        s["factor"] = 1.0 / max(1, n - out)
    return s


# ------------------------------------------------------------------- plain forms

def _plain_embed(s):
    ids, table, scale, v = s["ids"].long(), s["weights"], s["scale"], s["vocab"]
    out = {"out": (table[ids].float() * scale).to(_DT[s["act"]])}
    if s["train"]:
        rows = s["grad_out"].float() * scale
        if s["padding_idx"] is not None:
            rows = torch.where((ids != s["padding_idx"])[:, None], rows, torch.zeros_like(rows))
        grad = torch.zeros(v, s["dim"], device=table.device).index_add_(0, ids, rows)
        if s["accumulate"]:
            out["grad"] = s["buffer"].add_(grad)
        else:
            out["grad"] = grad.to(table.dtype)
    return out


def _plain_stats(x, layer):
    mean = x.mean(-1, keepdim=True) if layer else 0.0
    c = x - mean
    r = torch.rsqrt((c * c).mean(-1, keepdim=True) + _EPS)
    return c * r, r


def _plain_norm_grad(e, hat, r, layer):
    m = (e * hat).mean(-1, keepdim=True)
    e = e - hat * m
    return r * (e - e.mean(-1, keepdim=True) if layer else e)


def _plain_norm(s):
    layer, a = s["kind"] == "layer", s["residual_scale"]
    n, d, seqs = s["rows"], s["dim"], s["seqs"]
    x, h = s["inp"].float(), s["block"].float()
    w1, w2 = s["post_weight"].float(), s["pre_weight"].float()
    b1 = s["post_bias"].float() if layer else 0.0
    b2 = s["pre_bias"].float() if layer else 0.0
    grouped = s["gate"] == "sequence"
    gate = 1.0 if s["gate_"] is None else s["gate_"].float()
    if grouped:
        gate = gate[:, None, :].expand(seqs, n // seqs, d).reshape(n, d)
    hh, r1 = _plain_stats(h, layer)
    y = hh * w1 + b1
    new = a * x + gate * y
    xh, r2 = _plain_stats(new, layer)
    out = {"x": new.to(_DT[s["x"]]), "n": (xh * w2 + b2).to(_DT[s["h"]])}
    if s["train"]:
        pt = _DT[s["params"]]
        dn = s["grad_n"].float()
        t = s["grad_new"].float() + _plain_norm_grad(dn * w2, xh, r2, layer)
        tg = t * gate
        out["dx"] = (a * t).to(_DT[s["x"]])
        out["dh"] = _plain_norm_grad(tg * w1, hh, r1, layer).to(_DT[s["h"]])
        out["dpost"] = (tg * hh).sum(0).to(pt)
        out["dpre"] = (dn * xh).sum(0).to(pt)
        if layer:
            out["dpost_bias"] = tg.sum(0).to(pt)
            out["dpre_bias"] = dn.sum(0).to(pt)
        if s["gate_"] is not None:
            ty = t * y
            ty = ty.view(seqs, n // seqs, d).sum(1) if grouped else ty.sum(0)
            out["dgate"] = ty.to(pt)
    return out


def _plain_distill(s):
    z, temp, v = s["z"].float() / s["temperature"], s["temperature"], s["vocab"]
    idx = s["idx"].long()
    valid = (idx >= 0) & (idx < v)
    at = torch.where(valid, idx, torch.zeros_like(idx))
    t = torch.where(valid, s["t"].float() / temp, torch.full_like(idx, -math.inf, dtype=torch.float32))
    t = t - t.max(-1, keepdim=True).values
    log_q = t - torch.log(torch.exp(t).sum(-1, keepdim=True))
    q = torch.where(valid, torch.exp(log_q), torch.zeros_like(t))
    z = z - z.max(-1, keepdim=True).values
    e = torch.exp(z)
    total = e.sum(-1, keepdim=True)
    log_p = z.gather(1, at) - torch.log(total)
    rows = torch.where(valid, q * (log_q - log_p), torch.zeros_like(q)).sum(-1)
    factor = torch.full_like(rows, s["factor"])
    if s["weight"] is not None:
        factor = factor * s["weight"]
    out = {"rows": temp * temp * factor * rows}
    out["loss"] = out["rows"].sum()
    if s["train"]:
        e = e.mul_(1.0 / total).scatter_add_(1, at, -q)
        out["grad"] = e.mul_(temp * factor[:, None]).to(s["z"].dtype)
    return out


def _own_embed(s):
    ops = _framework()
    out = {"out": ops.scaled_embedding(s["ids"], s["weights"], s["scale"],
                                       out_dtype=_DT[s["act"]])}
    if s["train"]:
        out["grad"] = ops.scaled_embedding_grad(
            s["ids"], s["grad_out"], s["vocab"], s["scale"], dtype=s["weights"].dtype,
            padding_idx=s["padding_idx"], out=s.get("buffer"), accumulate=s["accumulate"])
    return out


def _own_norm(s):
    ops = _framework()
    new, n, stats = ops.residual_norm_forward(
        s["inp"], s["block"], s["post_weight"], s["pre_weight"], post_bias=s["post_bias"],
        pre_bias=s["pre_bias"], gate=s["gate_"], residual_scale=s["residual_scale"], eps=_EPS,
        kind=s["kind"])
    out = {"x": new, "n": n}
    if s["train"]:
        g = ops.residual_norm_backward(
            s["grad_new"], s["grad_n"], s["inp"], s["block"], stats, s["post_weight"],
            s["pre_weight"], post_bias=s["post_bias"], pre_bias=s["pre_bias"], gate=s["gate_"],
            residual_scale=s["residual_scale"], kind=s["kind"])
        out.update(dx=g.x, dh=g.h, dpost=g.post_weight, dpre=g.pre_weight)
        if s["kind"] == "layer":
            out.update(dpost_bias=g.post_bias, dpre_bias=g.pre_bias)
        if s["gate_"] is not None:
            out["dgate"] = g.gate
    return out


def _own_distill(s):
    ops = _framework()
    r = ops.topk_distill(s["z"], s["t"], s["idx"], temperature=s["temperature"],
                         weight=s["weight"], scale=s["factor"], grad=s["train"])
    out = {"rows": r.rows, "loss": r.loss}
    if s["train"]:
        out["grad"] = r.grad
    return out


def run(state):
    op = state["op"]
    if op == "embed":
        return _own_embed(state) if own else _plain_embed(state)
    if op == "norm":
        return _own_norm(state) if own else _plain_norm(state)
    return _own_distill(state) if own else _plain_distill(state)


# ------------------------------------------------------------------- work

def _distinct(vocab, tokens):
    """Expected distinct ids among `tokens` of the distribution of prepare()."""
    k = np.arange(1, vocab + 1, dtype=np.float64)
    p = np.log1p(1.0 / k) / math.log(vocab + 1.0)
    return float(-np.expm1(tokens * np.log1p(-p)).sum())


def work(case):
    if case["op"] == "embed":
        n, v, d = case["tokens"], case["vocab"], case["dim"]
        padded = int(case["pad"] * n)
        rows = _distinct(v, n - padded)
        ts, acts, ids = _SIZE[case["table"]], _SIZE[case["act"]], 4 if case["ids"] == "int32" else 8
        total = n * ids + (rows + bool(padded)) * d * ts + n * d * acts
        flops = n * d
        if case["train"]:
            total += (n - padded) * d * acts
            total += 2 * rows * d * 4 if case["accumulate"] else v * d * ts
            flops += 2 * (n - padded) * d
        return {"bytes": total, "flops": flops}
    if case["op"] == "norm":
        n, d = case["rows"], case["dim"]
        xs, hs, ps = _SIZE[case["x"]], _SIZE[case["h"]], _SIZE[case["params"]]
        vectors = (4 if case["kind"] == "layer" else 2) * d
        vectors += {"none": 0, "vector": d, "sequence": case["seqs"] * d}[case["gate"]]
        total = 2 * n * d * (xs + hs) + vectors * ps
        flops = 12 * n * d
        if case["train"]:
            total += n * d * (xs + hs) + n * d * (xs + hs) + vectors * ps
            flops += 30 * n * d
        return {"bytes": total, "flops": flops}
    n, v, k = case["rows"], case["vocab"], case["top"]
    live = n - int(case["masked"] * n)
    zs, ids = _SIZE[case["logits"]], 4 if case["ids"] == "int32" else 8
    total = live * (v * zs + k * (ids + _SIZE[case["teacher"]])) + 8 * n
    flops = 5 * live * v
    if case["train"]:
        total += n * v * zs
        flops += 3 * live * v
    return {"bytes": total, "flops": flops}


# ------------------------------------------------------------------- 64-bit values

def _exact_embed(s):
    ids = s["ids"].long()
    out = {"out": s["weights"].index_select(0, ids).double().mul_(s["scale"])}
    if s["train"]:
        dy = s["grad_out"].double()
        if s["padding_idx"] is not None:
            keep = ids != s["padding_idx"]
            ids, dy = ids[keep], dy[keep]
        grad = s["buffer"].double() if s["accumulate"] else \
            torch.zeros(s["vocab"], s["dim"], device=dy.device, dtype=torch.float64)
        out["grad"] = grad.index_put_((ids,), dy * s["scale"], accumulate=True)
    return out


def _exact_norm(s):
    layer, a = s["kind"] == "layer", s["residual_scale"]
    n, d, seqs = s["rows"], s["dim"], s["seqs"]

    def leaf(t):
        return None if t is None else t.double().requires_grad_(s["train"])

    x, h, w1, w2, b1, b2, gate = (leaf(s[k]) for k in ("inp", "block", "post_weight", "pre_weight",
                                                       "post_bias", "pre_bias", "gate_"))

    def norm(v, w, b):
        if layer:
            v = v - v.sum(-1, keepdim=True) / d
        v = v / torch.sqrt(v.pow(2).sum(-1, keepdim=True) / d + _EPS) * w
        return v if b is None else v + b

    with torch.enable_grad():
        y = norm(h, w1, b1)
        if gate is not None:
            y = (y.view(-1, n // seqs, d) * gate.view(seqs, 1, d)).view(n, d) \
                if s["gate"] == "sequence" else y * gate
        new = x * a + y
        nn = norm(new, w2, b2)
        out = {"x": new, "n": nn}
        if s["train"]:
            names = {"dx": x, "dh": h, "dpost": w1, "dpre": w2, "dpost_bias": b1, "dpre_bias": b2,
                     "dgate": gate}
            names = {k: t for k, t in names.items() if t is not None}
            got = torch.autograd.grad([new, nn], list(names.values()),
                                      [s["grad_new"].double(), s["grad_n"].double()])
            out.update(zip(names, got))
    return {k: t.detach() for k, t in out.items()}


def _exact_distill(s):
    n, v, temp = s["rows"], s["vocab"], s["temperature"]
    idx = s["idx"].long()
    t = s["t"].double() / temp
    t = t.masked_fill((idx < 0) | (idx >= v), -math.inf)
    log_q = t - torch.logsumexp(t, -1, keepdim=True)
    q = log_q.exp()
    w = s["factor"] * (torch.ones(n, device=idx.device, dtype=torch.float64)
                       if s["weight"] is None else s["weight"].double())
    at = idx.clamp(0, v - 1)
    rows = torch.empty(n, device=idx.device, dtype=torch.float64)
    grad = torch.empty(n, v, device=idx.device, dtype=torch.float64) if s["train"] else None
    for a in range(0, n, 1024):
        b = min(n, a + 1024)
        z = s["z"][a:b].double() / temp
        log_p = z - torch.logsumexp(z, -1, keepdim=True)
        gap = torch.where(q[a:b] > 0, log_q[a:b] - log_p.gather(1, at[a:b]), 0.0)
        rows[a:b] = temp ** 2 * w[a:b] * (q[a:b] * gap).sum(-1)
        if grad is not None:
            g = log_p.exp_().scatter_add_(1, at[a:b], -q[a:b])
            grad[a:b] = g * (temp * w[a:b])[:, None]
    out = {"rows": rows, "loss": rows.sum()}
    if grad is not None:
        out["grad"] = grad
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"embed": _exact_embed, "norm": _exact_norm, "distill": _exact_distill}[case["op"]](s)
