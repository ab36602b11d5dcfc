"""The training-step operators (mdq_b200.ops) on the GPU against plain 64-bit
implementations, at the sizes, strides and masks where they can go wrong.

Every tolerance is derived from the arithmetic, not from a run: see
ops_reference.py for the bound of a sum.  Values of a norm and of a softmax come
from a few roundings and sums of non-negative terms held lane-wise, so their
relative error is a small multiple of u (64 u is allowed, 256 u where two row
sums of mixed sign enter); it is applied to the magnitudes that enter the value.
"""
import math

import pytest
import torch

import ops_reference as ref
from mdq_b200 import ops
from ops_reference import U32, d64, rounding

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape, scale=1.0, dtype=F32):
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def within(got, want, bound, what=""):
    """|got - want| <= bound everywhere (a bound for each element)."""
    got, bound = d64(got), bound.expand_as(want)
    off = (got - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} values; worst "
                           f"{float((off / bound.clamp_min(1e-300))[bad].max()):.3g} of its bound")


def bits(t):
    return t.view(torch.int16 if t.dtype == BF16 else torch.int32)


# ----------------------------------------------------------------- embedding

EMBED = [  # tokens, vocab, dim
    (0, 7, 16), (1, 1, 1), (1, 50257, 768), (2, 5, 3), (31, 257, 40), (33, 300, 8), (64, 17, 1600),
    (257, 1000, 77), (1000, 3, 64), (1024, 1 << 17, 16), (2049, 513, 130), (4097, 70001, 24),
]


@pytest.mark.parametrize("tokens,vocab,dim", EMBED)
@pytest.mark.parametrize("table_dtype,out_dtype,ids_dtype", [
    (F32, BF16, torch.int64), (BF16, BF16, torch.int32), (F32, F32, torch.int32),
    (BF16, F32, torch.int64)])
def test_embedding(cuda_device, tokens, vocab, dim, table_dtype, out_dtype, ids_dtype):
    g = gen(tokens + dim)
    table = randn(g, vocab, dim, dtype=table_dtype)
    ids = torch.randint(-2, vocab + 2, (tokens,), generator=g).to(ids_dtype)
    got = ops.scaled_embedding(ids.to(cuda_device), table.to(cuda_device), 3.7, out_dtype=out_dtype)
    assert got.dtype == out_dtype and got.shape == (tokens, dim)
    want = ref.embedding(ids, table, 3.7)
    # scale rounded to fp32, one product, one rounding
    within(got, want, (2 * U32 + rounding(out_dtype)) * want.abs())


def _ids(kind, n, vocab, g, dtype=torch.int64):
    if kind == "uniform":
        t = torch.randint(0, vocab, (n,), generator=g)
    elif kind == "same":
        t = torch.full((n,), vocab // 2)
    elif kind == "words":
        t = (torch.exp(torch.rand(n, generator=g).double() * math.log(vocab + 1.0)).long() - 1)
    elif kind == "outside":
        t = torch.randint(-5, vocab + 5, (n,), generator=g)
    elif kind == "none":
        t = torch.full((n,), -1)
    else:   # ascending runs of unequal lengths
        t = (torch.arange(n).double().sqrt() * 3).long()
    return t.clamp(-5, vocab + 5).to(dtype) if kind in ("outside", "none") \
        else t.clamp(0, vocab - 1).to(dtype)


@pytest.mark.parametrize("tokens,vocab,dim", EMBED + [(16384, 997, 32), (16385, 4099, 20),
                                                     (40000, 50257, 8), (70001, 300000, 4)])
@pytest.mark.parametrize("kind", ["uniform", "same", "words", "outside", "none", "runs"])
def test_embedding_grad(cuda_device, tokens, vocab, dim, kind):
    g = gen(tokens * 3 + dim)
    way = (tokens + vocab + dim + len(kind)) % 4
    go_dtype, w_dtype = ((F32, F32), (BF16, F32), (BF16, BF16), (F32, BF16))[way]
    ids = _ids(kind, tokens, vocab, g, torch.int32 if way % 2 else torch.int64)
    go = randn(g, tokens, dim, dtype=go_dtype)
    want, bound = ref.embedding_grad(ids, go, vocab, 0.3)
    dev_ids, dev_go = ids.to(cuda_device), go.to(cuda_device)
    got = ops.scaled_embedding_grad(dev_ids, dev_go, vocab, 0.3, dtype=w_dtype)
    within(got, want, bound + rounding(w_dtype) * want.abs(), "dense")
    again = ops.scaled_embedding_grad(dev_ids, dev_go, vocab, 0.3, dtype=w_dtype)
    assert torch.equal(bits(got), bits(again))
    start = randn(g, vocab, dim)
    buf = start.clone().to(cuda_device)
    same = ops.scaled_embedding_grad(dev_ids, dev_go, vocab, 0.3, out=buf, accumulate=True)
    assert same is buf
    total = want + start.double()
    within(buf, total, bound + U32 * (total.abs() + want.abs()), "added")
    absent = torch.ones(vocab, dtype=torch.bool)
    absent[ids.long()[(ids >= 0) & (ids < vocab)]] = False
    assert torch.equal(buf.cpu()[absent], start[absent]), "rows that do not occur are not touched"


def test_embedding_grad_overwrites_and_pads(cuda_device):
    g = gen(5)
    ids = torch.randint(0, 50, (400,), generator=g)
    go = randn(g, 400, 96, dtype=BF16)
    go[ids == 7] = float("nan")          # masked by padding_idx
    want, bound = ref.embedding_grad(ids, go, 50, 1.0, padding_idx=7)
    out = torch.full((50, 96), float("nan"), device=cuda_device)
    ops.scaled_embedding_grad(ids.to(cuda_device), go.to(cuda_device), 50, out=out, padding_idx=7)
    within(out, want, bound + U32 * want.abs())
    assert bool((out[7] == 0).all())
    # NaN and infinity of a token stay in its row
    go = randn(g, 400, 96)
    go[ids == 3] = float("inf")
    go[ids == 4, 5] = float("nan")
    got = ops.scaled_embedding_grad(ids.to(cuda_device), go.to(cuda_device), 50).cpu()
    assert bool(torch.isinf(got[3]).all()) and bool(torch.isnan(got[4, 5]))
    got[3] = 0
    got[4, 5] = 0
    assert bool(torch.isfinite(got).all())


def test_embedding_strides_shapes_and_autograd(cuda_device):
    g = gen(6)
    wide = randn(g, 90, 128).to(cuda_device)
    table = wide[:, 3:103]                      # rows 128 apart, not 16-byte aligned
    ids = torch.randint(0, 90, (5, 7), generator=g).to(cuda_device)
    got = ops.scaled_embedding(ids, table, 2.0)
    want = ref.embedding(ids.reshape(-1), table, 2.0).reshape(5, 7, 100)
    within(got, want, 4 * U32 * want.abs())
    for dtype, cols in ((F32, slice(1, 34)), (BF16, slice(8, 40)), (BF16, slice(1, 34))):
        go = randn(g, 5, 7, 48, dtype=dtype).to(cuda_device)[:, :, cols]
        got = ops.scaled_embedding_grad(ids, go, 90)
        want, bound = ref.embedding_grad(ids, go, 90, 1.0)
        within(got, want, bound + U32 * want.abs())
    # autograd, an expanded (stride 0) incoming gradient, and another stream
    side = torch.cuda.Stream()
    leaf = randn(g, 90, 33).to(cuda_device).requires_grad_()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = ops.scaled_embedding(ids, leaf, 0.5, out_dtype=BF16, padding_idx=2)
        y.float().sum().backward()
    torch.cuda.current_stream().wait_stream(side)
    want, bound = ref.embedding_grad(ids, torch.ones(5, 7, 33), 90, 0.5, padding_idx=2)
    within(leaf.grad, want, bound + U32 * want.abs())


def test_embedding_large_offsets(cuda_device):
    """Rows whose element offsets pass 2^31, in the table and its gradient."""
    vocab, dim = 40000, 65536
    table = torch.zeros(vocab, dim, dtype=BF16, device=cuda_device)
    table[vocab - 1] = torch.arange(dim, device=cuda_device).remainder(64).to(BF16)
    ids = torch.tensor([vocab - 1, 3, vocab - 1], device=cuda_device)
    got = ops.scaled_embedding(ids, table, 2.0)
    assert torch.equal(got[0], table[vocab - 1] * 2) and torch.equal(got[2], got[0])
    assert not bool(got[1].any())
    grad = ops.scaled_embedding_grad(ids, got, vocab, dtype=BF16, out=table)
    assert torch.equal(grad[vocab - 1].float(), got[0].float() * 2)
    assert not bool(grad[:vocab - 1].any())


# ------------------------------------------------------------- residual norm

NORM_SIZES = [(1, 1), (1, 7), (1, 4096), (2, 768), (3, 8), (5, 33), (8, 1024), (13, 1600),
              (301, 768), (7, 1601), (64, 2050), (30, 5120), (6, 8192), (9, 12288), (4, 16384),
              (3, 20001), (2, 40000), (1200, 96)]
NORM_TYPES = [(F32, F32, F32), (F32, BF16, F32), (BF16, BF16, BF16), (BF16, BF16, F32),
              (BF16, F32, F32)]


def _norm_args(g, rows, dim, kind, types, gate_rows, bias):
    xt, ht, pt = types
    a = {"x": randn(g, rows, dim, scale=2.0, dtype=xt), "h": randn(g, rows, dim, dtype=ht) + 0.3}
    a["h"] = a["h"].to(ht)
    a["post_weight"] = (1 + randn(g, dim, scale=0.2)).to(pt)
    a["pre_weight"] = (1 + randn(g, dim, scale=0.2)).to(pt)
    a["post_bias"] = randn(g, dim, scale=0.2).to(pt) if bias else None
    a["pre_bias"] = randn(g, dim, scale=0.2).to(pt) if bias else None
    a["gate"] = None
    if gate_rows is not None:
        a["gate"] = (0.5 + randn(g, *((dim,) if gate_rows == 0 else (gate_rows, dim)),
                                 scale=0.3)).to(pt)
    return a


def _check_norm(dev, a, kind, alpha, seed, grads=("new", "n")):
    g = gen(seed)
    rows, dim = a["x"].shape
    eps = 1e-5
    on = {k: None if v is None else v.to(dev) for k, v in a.items()}
    pars = {k: on[k] for k in ("post_bias", "pre_bias", "gate")}
    new, n, stats = ops.residual_norm_forward(on["x"], on["h"], on["post_weight"],
                                              on["pre_weight"], residual_scale=alpha, eps=eps,
                                              kind=kind, **pars)
    leaves = {k: None if v is None else d64(v).requires_grad_() for k, v in a.items()}
    w_new, w_n = ref.residual_norm(**leaves, residual_scale=alpha, eps=eps, kind=kind)
    c = 64 * U32
    r_n = rounding(on["x"].dtype if on["h"] is None else on["h"].dtype)
    with torch.no_grad():
        # magnitudes that enter x_new: the residual, and the block's part with its mean removed
        size = w_new.abs() + abs(alpha) * leaves["x"].abs()
        if a["h"] is not None:
            gate = 1.0 if a["gate"] is None else leaves["gate"].abs().reshape(-1, dim)
            hm = leaves["h"].abs()
            sc = 1 / torch.sqrt(leaves["h"].var(-1, correction=0, keepdim=True) + eps) \
                if kind == "layer" else \
                1 / torch.sqrt(leaves["h"].pow(2).mean(-1, keepdim=True) + eps)
            part = (hm + hm.mean(-1, keepdim=True)) * sc * leaves["post_weight"].abs()
            if a["post_bias"] is not None:
                part = part + leaves["post_bias"].abs()
            if a["gate"] is not None:
                part = part * gate.repeat_interleave(rows // gate.shape[0], 0)
            size = size + part
            within(new, w_new, c * size + rounding(on["x"].dtype) * w_new.abs(), "x_new")
        else:
            assert new is on["x"]
        if n is not None:
            dev_new = torch.sqrt(w_new.var(-1, correction=0, keepdim=True) + eps) \
                if kind == "layer" else torch.sqrt(w_new.pow(2).mean(-1, keepdim=True) + eps)
            rel = (size + size.mean(-1, keepdim=True) + w_new.abs()) / dev_new
            rel = rel * leaves["pre_weight"].abs()
            # the deviation's own error, from the row's
            rel = rel + (w_n.abs() + leaves["pre_weight"].abs()) * \
                ((size * w_new.abs()).mean(-1, keepdim=True) / dev_new ** 2)
            within(n, w_n, c * rel + (r_n + c) * w_n.abs() +
                   (0 if a["pre_bias"] is None else c * leaves["pre_bias"].abs()), "n")
    # gradients against the formula's (64-bit autograd)
    gn = randn(g, rows, dim, dtype=on["x"].dtype) if "new" in grads else None
    gg = randn(g, rows, dim, dtype=on["x"].dtype if a["h"] is None else on["h"].dtype) \
        if "n" in grads and n is not None else None
    got = ops.residual_norm_backward(None if gn is None else gn.to(dev),
                                     None if gg is None else gg.to(dev), on["x"], on["h"], stats,
                                     on["post_weight"], on["pre_weight"], residual_scale=alpha,
                                     kind=kind, **pars)
    outs = [(t, d64(v)) for t, v in ((w_new, gn), (w_n, gg)) if v is not None]
    names = [k for k in leaves if leaves[k] is not None]
    want = torch.autograd.grad([t for t, _ in outs], [leaves[k] for k in names],
                               [v for _, v in outs], allow_unused=True)
    for k, w in zip(names, want):
        v = getattr(got, k)
        w = torch.zeros_like(leaves[k]) if w is None else w
        assert v.shape == a[k].shape and v.dtype == a[k].dtype
        # Row gradients: two row sums of mixed sign.  Parameters: sums over the rows, whose
        # terms are of the size of the largest; both against the magnitudes' root mean square.
        if k in ("x", "h"):
            scale = w.pow(2).mean(-1, keepdim=True).sqrt() + w.abs()
            if k == "h":
                scale = scale + 4.0 / torch.sqrt(leaves["h"].var(-1, correction=0, keepdim=True)
                                                 + eps if kind == "layer" else
                                                 leaves["h"].pow(2).mean(-1, keepdim=True) + eps)
            else:
                scale = scale + 4.0 * max(1.0, abs(alpha))
            if n is not None:
                scale = scale * (1 + (size.pow(2).mean(-1, keepdim=True).sqrt() /
                                      dev_new).detach())
            scale = scale * (1 + math.sqrt(dim) / 16)
        else:
            per = rows if v.dim() == 1 else rows // v.shape[0]
            scale = 16.0 * per + w.abs()
        within(v, w.detach(), 256 * U32 * scale + rounding(v.dtype) * w.abs().detach(), "grad " + k)
    return got


@pytest.mark.parametrize("rows,dim", NORM_SIZES)
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_residual_norm(cuda_device, rows, dim, kind):
    if kind == "layer" and dim == 1:
        pytest.skip("the layer norm of one value has no deviation")
    k = rows + dim
    for i, types in enumerate(NORM_TYPES):
        gate_rows = (0, None, rows if rows % 2 else 2, 1, 0)[(k + i) % 5]
        if gate_rows and rows % gate_rows:
            gate_rows = 1
        a = _norm_args(gen(k + i), rows, dim, kind, types, gate_rows, bias=(k + i) % 2 == 0)
        _check_norm(cuda_device, a, kind, (1.0, 0.5, -1.7)[(k + i) % 3], k)


@pytest.mark.parametrize("part", ["first", "last", "first layer", "last layer", "no grad_new",
                                  "no grad_n"])
@pytest.mark.parametrize("dim", [40, 768, 1601, 5000])
def test_residual_norm_parts(cuda_device, part, dim):
    kind = "layer" if "layer" in part else "rms"
    for i, types in enumerate(NORM_TYPES[:4]):
        a = _norm_args(gen(dim + i), 37, dim, kind, types, 0, bias="layer" in part)
        if part.startswith("first"):
            a["h"] = a["post_weight"] = a["post_bias"] = a["gate"] = None
        if part.startswith("last"):
            a["pre_weight"] = a["pre_bias"] = None
        grads = {"no grad_new": ("n",), "no grad_n": ("new",)}.get(part, ("new", "n"))
        _check_norm(cuda_device, a, kind, 1.0, dim, grads)


@pytest.mark.parametrize("groups,per", [(1, 50), (2, 1), (5, 7), (3, 341), (64, 2), (300, 1), (1, 1)])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_residual_norm_gate_groups(cuda_device, groups, per, kind):
    for dim in (24, 1030):
        a = _norm_args(gen(groups), groups * per, dim, kind, NORM_TYPES[groups % 3], groups,
                       bias=kind == "layer")
        _check_norm(cuda_device, a, kind, 0.9, dim)


def test_residual_norm_empty(cuda_device):
    w = torch.ones(16, device=cuda_device)
    x = torch.zeros(0, 16, device=cuda_device)
    new, n, stats = ops.residual_norm_forward(x, x, w, w, gate=w)
    assert new.shape == n.shape == (0, 16)
    g = ops.residual_norm_backward(x, x, x, x, stats, w, w, gate=w)
    for t in (g.post_weight, g.pre_weight, g.gate):
        assert not bool(t.any())


def test_residual_norm_hard_values(cuda_device):
    """Rows of zeros, of one value, huge and tiny ones, and rows with NaN or
    infinity, which stay in their rows."""
    g = gen(9)
    for dim in (64, 769, 4096):
        x, h = randn(g, 9, dim), randn(g, 9, dim)
        x[0], h[0] = 0, 0
        h[1] = 5.0                       # no deviation: layer norm gives the bias
        x[2], h[2] = x[2] * 1e15, h[2] * 1e15
        h[3] = h[3] * 1e-12
        x[4] += 1000.0                   # a mean far above the deviation
        x[5, 3] = float("nan")
        h[6, 5] = float("inf")
        w = 1 + randn(g, dim, scale=0.1)
        for kind in ("rms", "layer"):
            new, n, _ = (None if t is None else t.cpu() for t in ops.residual_norm_forward(
                x.to(cuda_device), h.to(cuda_device), w.to(cuda_device), w.to(cuda_device),
                kind=kind))
            w_new, w_n = ref.residual_norm(*(t.double() for t in (x, h, w, w)), kind=kind)
            assert bool(torch.isnan(n[5]).all()) and bool(torch.isnan(n[6]).all())
            keep = [0, 1, 2, 3, 7, 8]
            size = w_new[keep].abs() + x[keep].abs().double()
            # row 1 under layer norm: h - mean(h) is rounding, at most 4 u of h over sqrt(eps)
            slack = 64 * U32 * (size + 1) + (4 * U32 * 5 / math.sqrt(1e-5) if kind == "layer" else 0)
            within(new[keep], w_new[keep], slack, f"{kind} x_new")
            dev = torch.sqrt(w_new[keep].pow(2).mean(-1, keepdim=True) + 1e-5)
            within(n[keep], w_n[keep], 8 * slack / dev * 2 + 64 * U32 * (1 + w_n[keep].abs()),
                   f"{kind} n")
            # row 4: values near 1000 carry 1000 u, over a deviation of about 1.4
            within(n[4:5], w_n[4:5], torch.tensor(64 * U32 * 1010.0), f"{kind} large mean")


def test_residual_norm_strides_autograd_streams(cuda_device):
    g = gen(10)
    wide_x = randn(g, 3, 11, 150).to(cuda_device)
    wide_h = randn(g, 33, 131, dtype=BF16).to(cuda_device)
    w = [(1 + randn(g, 97, scale=0.1)).to(cuda_device).requires_grad_() for _ in range(3)]
    x = wide_x[:, :, 2:99].clone().requires_grad_()
    xs = wide_x[:, :, 2:99]                    # rows 150 apart, off a 16-byte boundary
    hs = wide_h[:, 1:98].unflatten(0, (3, 11))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        h = hs.clone().requires_grad_()
        a_new, a_n = ops.residual_norm(xs, hs, w[0].detach(), w[1].detach(), gate=w[2].detach())
        new, n = ops.residual_norm(x, h, w[0], w[1], gate=w[2])
        (new.sum() + n.float().sum()).backward()       # expanded gradients
    torch.cuda.current_stream().wait_stream(side)
    # strided inputs give what their copies give, up to the order of the sums
    within(a_new, d64(new), 64 * U32 * (d64(new).abs() + 2))
    within(a_n, d64(n), (2 * rounding(BF16)) * (d64(n).abs() + 1e-3))
    assert new.shape == (3, 11, 97) and n.dtype == BF16
    leaves = [d64(t).requires_grad_() for t in (x.reshape(33, 97), h.reshape(33, 97), *w)]
    w_new, w_n = ref.residual_norm(leaves[0], leaves[1], leaves[2], leaves[3], gate=leaves[4])
    want = torch.autograd.grad(w_new.sum() + w_n.sum(), leaves)
    for t, v in zip((x, h, *w), want):
        v = v.reshape(t.shape)
        within(t.grad, v, rounding(t.dtype) * v.abs() + 256 * U32 * 33 * 8)
    # only one of the results used; the first norm and the last
    for pick in (0, 1):
        x.grad = None
        ops.residual_norm(x, h, w[0], w[1])[pick].float().square().sum().backward()
        assert bool(torch.isfinite(x.grad).all()) and bool(x.grad.any())
    x.grad = None
    same, n = ops.residual_norm(x, None, None, w[1], kind="layer")
    assert same is x
    n.square().sum().backward()
    assert bool(torch.isfinite(x.grad).all())
    new, none = ops.residual_norm(x, h, w[0], None)
    assert none is None and new.shape == x.shape


def test_residual_norm_gradient_by_differences(cuda_device):
    """<gradient, direction> against a central difference of the 64-bit loss.
    The difference's own error is of the order step^2 (third derivatives of order
    one); the kernel's is fp32."""
    g = gen(11)
    rows, dim, step = 6, 50, 1e-4
    for kind in ("rms", "layer"):
        a = _norm_args(g, rows, dim, kind, NORM_TYPES[0], 3, bias=True)
        co = randn(g, rows, dim), randn(g, rows, dim)
        on = {k: v.to(cuda_device) for k, v in a.items()}
        pars = {k: on[k] for k in ("post_bias", "pre_bias", "gate")}
        stats = ops.residual_norm_forward(on["x"], on["h"], on["post_weight"], on["pre_weight"],
                                          residual_scale=0.8, kind=kind, **pars)[2]
        got = ops.residual_norm_backward(co[0].to(cuda_device), co[1].to(cuda_device), on["x"],
                                         on["h"], stats, on["post_weight"], on["pre_weight"],
                                         residual_scale=0.8, kind=kind, **pars)

        def loss(args):
            new, n = ref.residual_norm(**args, residual_scale=0.8, kind=kind)
            return float((new * co[0].double()).sum() + (n * co[1].double()).sum())

        for k in a:
            v = randn(g, *a[k].shape).double()
            plus, minus = ({**{j: t.double() for j, t in a.items()}} for _ in range(2))
            plus[k], minus[k] = plus[k] + step * v, minus[k] - step * v
            diff = (loss(plus) - loss(minus)) / (2 * step)
            dot = float((d64(getattr(got, k)) * v).sum())
            size = float((d64(getattr(got, k)) * v).abs().sum())
            assert abs(dot - diff) <= 2e-5 * size + 1e-5, (kind, k, dot, diff)


# -------------------------------------------------------------- distillation

DISTILL = [(1, 1, 1), (1, 50257, 8), (2, 2, 2), (3, 7, 5), (5, 257, 16), (4, 1000, 1000),
           (9, 4097, 33), (130, 8191, 7), (7, 50257, 64), (3, 50304, 100), (2, 100003, 20),
           (3, 128256, 50), (2, 262147, 12), (600, 300, 4), (0, 50, 3)]


def _distill_case(g, rows, vocab, top, dtype, t_dtype, i_dtype):
    z = randn(g, rows, vocab, scale=2.0, dtype=dtype)
    idx = torch.rand(rows, vocab if vocab <= 4096 else 4096, generator=g).argsort(-1)[:, :top] \
        if rows else torch.zeros(0, top, dtype=torch.int64)
    if vocab > 4096:
        idx = idx * (vocab // 4096) + vocab % 4096
    t = randn(g, rows, top, scale=2.0, dtype=t_dtype)
    return z, t, idx.to(i_dtype)


def _check_distill(dev, z, t, idx, temp, weight, scale):
    on = [None if v is None else v.to(dev) for v in (z, t, idx, weight)]
    got = ops.topk_distill(on[0], on[1], on[2], temperature=temp, weight=on[3], scale=scale)
    leaf = d64(z).requires_grad_()
    rows = ref.distill_rows(leaf, t, idx, temp, weight, scale)
    (grad,) = torch.autograd.grad(rows.sum(), leaf) if rows.requires_grad else (torch.zeros_like(leaf),)
    rows = rows.detach()
    w = torch.ones(len(z), dtype=torch.float64) if weight is None else d64(weight)
    c = temp * temp * scale * w.abs()
    # A row's loss: log-probabilities of magnitude up to the spread of z / T, each with a few
    # roundings; the exponents' own error is u times their magnitude, at most the spread.
    spread = 1 + 2 * leaf.detach().abs().max(-1).values / temp if z.numel() else torch.zeros(len(z))
    within(got.rows, rows, 64 * U32 * c * (spread + 1), "rows")
    assert got.loss.shape == () and got.rows.shape == z.shape[:-1]
    within(got.loss, rows.sum(), (64 * U32 * c * (spread + 1)).sum() + 4 * U32 * rows.sum().abs())
    if z.numel():
        # p and q to a relative (spread + 64) u each
        mag = grad.abs() + (temp * scale * w.abs())[:, None] * _mass(leaf.detach(), t, idx, temp)
        bound = (spread[:, None] + 64) * U32 * 2 * mag + rounding(z.dtype) * grad.abs()
        within(got.grad, grad, bound + 1e-37, "grad")
    only = ops.topk_distill(on[0], on[1], on[2], temperature=temp, weight=on[3], scale=scale,
                            grad=False)
    assert only.grad is None
    within(only.rows, d64(got.rows), 128 * U32 * c * (spread + 1))
    again = ops.topk_distill(on[0], on[1], on[2], temperature=temp, weight=on[3], scale=scale)
    for x, y in zip(got, again):
        assert torch.equal(bits(x), bits(y)), "the same call gives the same bits"
    return got


def _mass(z, t, idx, temp):
    """p + the q's at each index: the magnitudes that a gradient is the difference of."""
    idx, v = idx.long(), z.shape[1]
    ok = (idx >= 0) & (idx < v)
    q = torch.softmax(torch.where(ok, d64(t) / temp, -math.inf), -1)
    q = torch.where(ok, q, 0.0).nan_to_num(0.0)
    return torch.softmax(z / temp, -1).scatter_add_(1, torch.where(ok, idx, 0), q)


@pytest.mark.parametrize("rows,vocab,top", DISTILL)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_distill(cuda_device, rows, vocab, top, dtype):
    g = gen(vocab + rows)
    k = (rows + vocab + top) % 3
    t_dtype, i_dtype = (F32, BF16)[k % 2], (torch.int64, torch.int32)[k // 2]
    z, t, idx = _distill_case(g, rows, vocab, top, dtype, t_dtype, i_dtype)
    for temp, weight, scale in ((1.0, None, 1.0), (2.5, (torch.rand(rows, generator=g) > 0.4).float()
                                                   * 1.5, 0.01)):
        _check_distill(cuda_device, z, t, idx, temp, weight, scale)


@pytest.mark.parametrize("vocab", [40, 3001, 50257])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_distill_absent_repeated_and_empty_rows(cuda_device, vocab, dtype):
    g = gen(21)
    z, t, idx = _distill_case(g, 10, vocab, 12, dtype, F32, torch.int64)
    idx[0, 5:] = -1
    idx[1, :7] = vocab                 # outside
    idx[2] = -1                        # nothing present
    idx[3] = idx[3, 0]                 # one index twelve times
    idx[4, 6:] = idx[4, :6]            # pairs
    t[5, 3:] = -math.inf               # entries of probability 0
    t[6] = -math.inf                   # present, but without probability: an empty row
    t[0, 5:] = float("nan")            # masked values are not used
    t[1, :7] = float("inf")
    weight = torch.ones(10)
    weight[7] = 0.0
    got = _check_distill(cuda_device, z, t, idx, 1.5, weight, 0.5)
    for r in (2, 6, 7):
        assert float(got.rows[r]) == 0.0 and not bool(got.grad[r].any())
    # Rows that do not count may hold anything.
    for r in (2, 6, 7):
        z[r] = float("nan")
    z[7, 0] = float("inf")
    dirty = ops.topk_distill(z.to(cuda_device), t.to(cuda_device), idx.to(cuda_device),
                             temperature=1.5, weight=weight.to(cuda_device), scale=0.5)
    assert torch.equal(dirty.rows, got.rows) and torch.equal(dirty.grad, got.grad)
    assert bool(torch.isfinite(dirty.loss))


@pytest.mark.parametrize("vocab", [33, 50257])
def test_distill_masked_vocabulary_and_special_values(cuda_device, vocab):
    g = gen(22)
    z, t, idx = _distill_case(g, 7, vocab, 4, F32, F32, torch.int32)
    z[0, ::2] = -math.inf                       # half of the vocabulary masked away
    idx[0] = torch.tensor([1, 3, 5, 7])
    z[1, 1::2] = torch.finfo(F32).min           # the type's lowest value
    idx[1] = torch.tensor([0, 2, 4, 6])
    z[2] = 12.5                                 # a flat row
    z[3] = z[3] * 1000                          # one token has all probability
    z[4, idx[4, 0].long()] = -math.inf          # the teacher's token is masked: infinite loss
    z[5, 2] = float("nan")
    z[6, 2] = math.inf
    out = ops.topk_distill(z.to(cuda_device), t.to(cuda_device), idx.to(cuda_device))
    rows, grad = out.rows.cpu(), out.grad.cpu()
    keep = [0, 1, 2, 3]
    leaf = z[keep].double().requires_grad_()
    want = ref.distill_rows(leaf, t[keep], idx[keep], 1.0)
    spread = torch.tensor([16.0, 16.0, 16.0, 2e4])
    within(rows[keep], want.detach(), 64 * U32 * spread)
    p = torch.softmax(leaf.detach(), -1)
    q = torch.softmax(t[keep].double(), -1)
    exact = p.scatter_add(1, idx[keep].long(), -q)
    within(grad[keep], exact, (spread[:, None] + 64) * 2 * U32 * (exact.abs() + p + 1e-3))
    assert not bool(grad[0, ::2].any())
    assert math.isinf(float(rows[4])) and bool(torch.isfinite(grad[4]).all())
    for r in (5, 6):
        assert math.isnan(float(rows[r]))


def test_distill_is_cross_entropy_with_one_entry(cuda_device):
    g = gen(23)
    z = randn(g, 50, 1000, scale=3.0)
    label = torch.randint(0, 1000, (50,), generator=g)
    label[10] = -100
    got = ops.topk_distill(z.to(cuda_device), torch.zeros(50, 1, device=cuda_device),
                           label[:, None].to(cuda_device))
    want = torch.nn.functional.cross_entropy(z.double(), label, ignore_index=-100, reduction="sum")
    within(got.loss, want, torch.tensor(64 * U32 * 50 * 24.0))


def test_distill_strides_in_place_autograd_streams(cuda_device):
    g = gen(24)
    for dtype in (F32, BF16):
        wide = randn(g, 12, 1100, dtype=dtype).to(cuda_device)
        z = wide[:, 3:1004]                       # rows 1100 apart, off a 16-byte boundary
        _, t, idx = _distill_case(g, 12, 1001, 9, dtype, F32, torch.int64)
        t, idx = t.to(cuda_device), idx.to(cuda_device)
        plain = ops.topk_distill(z.contiguous(), t, idx, temperature=2.0)
        got = ops.topk_distill(z, t, idx, temperature=2.0)
        scale = float(plain.rows.abs().max())
        within(got.rows, d64(plain.rows), torch.tensor(64 * U32 * (scale + 8)))
        within(got.grad, d64(plain.grad), 2 * rounding(dtype) * d64(plain.grad).abs() + 256 * U32)
        # a gradient buffer of other strides and alignment; the rest of it stays
        buf = torch.full((12, 1300), 7.0, dtype=dtype, device=cuda_device)
        ops.topk_distill(z, t, idx, temperature=2.0, out=buf[:, 5:1006])
        assert torch.equal(buf[:, 5:1006], got.grad)
        assert bool((buf[:, :5] == 7).all()) and bool((buf[:, 1006:] == 7).all())
        # in place
        keep = wide.clone()
        ops.topk_distill(z, t, idx, temperature=2.0, out=z)
        assert torch.equal(z, got.grad)
        assert torch.equal(wide[:, :3], keep[:, :3]) and torch.equal(wide[:, 1004:], keep[:, 1004:])
        wide.copy_(keep)
        # autograd: upstream scalars and upstream rows, on another stream
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            leaf = z.reshape(3, 4, 1001).clone().requires_grad_()
            args = (t.reshape(3, 4, 9), idx.reshape(3, 4, 9))
            (ops.topk_distill_loss(leaf, *args, temperature=2.0) * 3.0).backward()
            whole = leaf.grad
            leaf.grad = None
            rows = ops.topk_distill_loss(leaf, *args, temperature=2.0, reduction="none")
            (rows * torch.arange(12.0, device=cuda_device).view(3, 4)).sum().backward()
        torch.cuda.current_stream().wait_stream(side)
        want = d64(plain.grad)
        within(whole.view(12, 1001), 3 * want, (4 * rounding(dtype)) * 3 * want.abs() + 256 * U32)
        up = torch.arange(12.0).double()[:, None]
        within(leaf.grad.view(12, 1001), up * want, (4 * rounding(dtype)) * up * want.abs() + 2e-5)
        assert rows.shape == (3, 4)


def test_distill_gradient_by_differences(cuda_device):
    g = gen(25)
    z, t, idx = _distill_case(g, 6, 200, 10, F32, F32, torch.int64)
    idx[:, 7:] = idx[:, :3]
    got = ops.topk_distill(z.to(cuda_device), t.to(cuda_device), idx.to(cuda_device),
                           temperature=1.7, scale=0.25)
    v, step = randn(g, 6, 200).double(), 1e-4
    plus, minus = (float(ref.distill_rows(z.double() + s * v, t, idx, 1.7, None, 0.25).sum())
                   for s in (step, -step))
    dot = float((d64(got.grad) * v).sum())
    assert abs(dot - (plus - minus) / (2 * step)) <= 1e-6 * float((d64(got.grad) * v).abs().sum()) + 1e-6


def test_distill_large_offsets(cuda_device):
    """Rows whose element offsets pass 2^31."""
    rows, vocab = 44000, 50257
    z = torch.zeros(rows, vocab, dtype=BF16, device=cuda_device)
    z[rows - 1, 100] = 3.0
    idx = torch.full((rows, 1), -1, dtype=torch.int64, device=cuda_device)
    idx[0, 0] = 5
    idx[rows - 1, 0] = 100
    got = ops.topk_distill(z, torch.zeros(rows, 1, device=cuda_device), idx, out=z)
    total = vocab - 1 + math.exp(3.0)
    # one row flat, one with a raised token: log-sum-exp minus the token's logit
    within(got.rows[0], torch.tensor(math.log(vocab)).double(), torch.tensor(64 * U32 * 11))
    within(got.rows[-1], torch.tensor(math.log(total) - 3.0).double(), torch.tensor(64 * U32 * 14))
    assert not bool(got.grad[1:rows - 1].any())
    p = math.exp(3.0) / total - 1
    assert abs(float(got.grad[rows - 1, 100]) - p) <= 2 ** -8


# ------------------------------------------------------------------ refusals

def test_front_end_refuses(cuda_device):
    x = torch.zeros(4, 8, device=cuda_device)
    w = torch.ones(8, device=cuda_device)
    ids = torch.zeros(4, dtype=torch.int64, device=cuda_device)
    idx = torch.zeros(4, 2, dtype=torch.int64, device=cuda_device)
    t = torch.zeros(4, 2, device=cuda_device)
    stats = torch.zeros(4, 4, device=cuda_device)
    half = torch.float16
    bad = [
        ("ids must be", lambda: ops.scaled_embedding(ids.float(), x)),
        ("ids must be on", lambda: ops.scaled_embedding(ids.cpu(), x)),
        ("contiguous", lambda: ops.scaled_embedding(ids[::2], x)),
        ("float32 or bfloat16", lambda: ops.scaled_embedding(ids, x.to(half))),
        ("out_dtype", lambda: ops.scaled_embedding(ids, x, out_dtype=half)),
        ("table must be", lambda: ops.scaled_embedding(ids, w)),
        ("table must be", lambda: ops.scaled_embedding(ids, x[:0])),
        ("contiguous", lambda: ops.scaled_embedding(ids, x.t())),
        ("padding_idx", lambda: ops.scaled_embedding(ids, x, padding_idx=4)),
        ("grad_out must be", lambda: ops.scaled_embedding_grad(ids[:3], x, 9)),
        ("positive", lambda: ops.scaled_embedding_grad(ids, x, 0)),
        ("accumulate needs out", lambda: ops.scaled_embedding_grad(ids, x, 9, accumulate=True)),
        ("accumulate needs a float32",
         lambda: ops.scaled_embedding_grad(ids, x, 4, out=x.bfloat16(), accumulate=True)),
        ("out must be", lambda: ops.scaled_embedding_grad(ids, x, 5, out=x)),
        ("padding_idx", lambda: ops.scaled_embedding_grad(ids, x, 5, padding_idx=-1)),
        ("float32 or bfloat16", lambda: ops.scaled_embedding_grad(ids, x, 5, dtype=half)),
        ("kind", lambda: ops.residual_norm(x, x, w, w, kind="batch")),
        ("h must have", lambda: ops.residual_norm(x, x[:3], w, w)),
        ("h must be on", lambda: ops.residual_norm(x, x.cpu(), w, w)),
        ("needs post_weight", lambda: ops.residual_norm(x, x, None, w)),
        ("need h", lambda: ops.residual_norm(x, None, None, w, gate=w)),
        ("either", lambda: ops.residual_norm(x, None, None, None)),
        ("residual_scale", lambda: ops.residual_norm(x, None, None, w, residual_scale=0.5)),
        ("pre_bias", lambda: ops.residual_norm(x, x, w, None, pre_bias=w)),
        ("one dtype", lambda: ops.residual_norm(x, x, w, w.bfloat16())),
        ("post_weight must be", lambda: ops.residual_norm(x, x, w[:7], w)),
        ("gate must be", lambda: ops.residual_norm(x, x, w, w, gate=w[:7])),
        ("divide", lambda: ops.residual_norm(x, x, w, w, gate=x[:3].contiguous())),
        ("float32 or bfloat16", lambda: ops.residual_norm(x.to(half), x, w, w)),
        ("stats", lambda: ops.residual_norm_backward(x, x, x, x, None, w, w)),
        ("stats", lambda: ops.residual_norm_backward(x, x, x, x, stats[:3], w, w)),
        ("grad_new must", lambda: ops.residual_norm_backward(x[:3], x, x, x, stats, w, w)),
        ("grad_n must", lambda: ops.residual_norm_backward(x, x.bfloat16(), x, x, stats, w, w)),
        ("grad_n needs", lambda: ops.residual_norm_backward(x, x, x, x, stats, w, None)),
        ("teacher_index must be", lambda: ops.topk_distill(x, t, idx.float())),
        ("teacher_logits and", lambda: ops.topk_distill(x, t, idx[:3])),
        ("contiguous", lambda: ops.topk_distill(x, t.expand(4, 2)[:, :1], idx[:, :1])),
        ("top must", lambda: ops.topk_distill(x, t[:, :0], idx[:, :0])),
        ("temperature", lambda: ops.topk_distill(x, t, idx, temperature=0.0)),
        ("temperature", lambda: ops.topk_distill(x, t, idx, temperature=float("nan"))),
        ("weight", lambda: ops.topk_distill(x, t, idx, weight=w)),
        ("weight", lambda: ops.topk_distill(x, t, idx, weight=w[:4].double())),
        ("out must", lambda: ops.topk_distill(x, t, idx, out=x.bfloat16())),
        ("overlap", lambda: ops.topk_distill(x, t, idx, out=w.expand(4, 8))),
        ("out needs", lambda: ops.topk_distill(x, t, idx, out=x, grad=False)),
        ("float32 or bfloat16", lambda: ops.topk_distill(x.to(half), t, idx)),
        ("reduction", lambda: ops.topk_distill_loss(x, t, idx, reduction="mean")),
    ]
    for match, call in bad:
        with pytest.raises(RuntimeError, match=match):
            call()
