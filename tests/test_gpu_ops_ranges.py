"""The training-step operators (mdq_b200.ops) on the GPU beyond ordinary sizes:
long lists of teacher entries over many rows, rows that no shared memory holds,
more tokens than one sort takes, wide residual streams, rows that neighbours with
NaN surround, and gradient buffers that overlap the logits.

The bounds are those of test_gpu_ops.py, whose checks these tests call.
"""
import math

import pytest
import torch

import ops_reference as ref
import test_gpu_ops as base
from mdq_b200 import ops
from ops_reference import U32, d64, rounding
from test_gpu_ops import BF16, F32, bits, gen, randn, within

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------ distillation

MANY = [  # rows, vocab, top
    (149, 257, 257), (160, 3001, 100), (301, 700, 1024), (160, 33, 64), (500, 4096, 33),
    (200, 50257, 40), (149, 130001, 5), (2, 460003, 50), (3, 300001, 300), (148, 20011, 64),
    (1500, 1, 3), (1481, 7, 2), (1600, 1031, 8),
]


def _entries(g, rows, vocab, top, i_dtype):
    """Indices with absent and repeated entries, rows without any, rows of one index."""
    idx = torch.randint(-1, vocab + 1, (rows, top), generator=g)
    if top > 1:
        idx[1::5, top // 2:] = idx[1::5, :top - top // 2]
    idx[2::7] = idx[2::7, :1].clamp(0, vocab - 1)
    idx[3::11] = -1
    return idx.to(i_dtype)


@pytest.mark.parametrize("rows,vocab,top", MANY)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_distill_many_rows_and_entries(cuda_device, rows, vocab, top, dtype):
    g = gen(rows + vocab + top)
    idx = _entries(g, rows, vocab, top, (torch.int32, torch.int64)[rows % 2])
    z = randn(g, rows, vocab, scale=2.0, dtype=dtype)
    t = randn(g, rows, top, scale=2.0, dtype=(F32, BF16)[top % 2])
    weight = (torch.rand(rows, generator=g) > 0.3).float() * torch.rand(rows, generator=g)
    got = base._check_distill(cuda_device, z, t, idx, 1.3, weight, 0.7)
    dead = (weight == 0) | (((idx < 0) | (idx >= vocab)).all(-1))
    assert not bool(got.grad.cpu()[dead].any()) and not bool(got.rows.cpu()[dead].any())
    # rows that do not count hold anything; in place; weights of 1 by their absence
    dirty = z.clone()
    dirty[dead] = float("nan")
    on = [v.to(cuda_device) for v in (dirty, t, idx, weight)]
    same = ops.topk_distill(on[0], on[1], on[2], temperature=1.3, weight=on[3], scale=0.7, out=on[0])
    assert same.grad is on[0]
    for a, b in zip(got, same):
        assert torch.equal(bits(a), bits(b))
    if rows <= 200:
        base._check_distill(cuda_device, z, t, idx, 1.0, None, 1.0)


def test_distill_more_rows_than_are_listed(cuda_device):
    g = gen(31)
    rows = 66000
    z, t = randn(g, rows, 40, dtype=BF16), randn(g, rows, 3)
    idx = _entries(g, rows, 40, 3, torch.int32)
    base._check_distill(cuda_device, z, t, idx, 2.0, (torch.rand(rows, generator=g) > 0.5).float(), 1e-3)


@pytest.mark.parametrize("vocab", [1001, 50257, 130001])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_distill_many_rows_off_alignment(cuda_device, vocab, dtype):
    """Rows at an odd distance off 16 bytes, between columns of NaN that stay as
    they are, for more rows than the device holds at once."""
    g = gen(vocab)
    rows = 310 if vocab < 100000 else 160
    wide = randn(g, rows, vocab + 14, scale=2.0, dtype=dtype)
    wide[:, :5] = wide[:, vocab + 5:] = float("nan")
    t, idx = randn(g, rows, 9), _entries(g, rows, vocab, 9, torch.int64)
    on = wide.to(cuda_device)
    z = on[:, 5:vocab + 5]
    want = ops.topk_distill(z.contiguous(), t.to(cuda_device), idx.to(cuda_device), temperature=0.7)
    got = ops.topk_distill(z, t.to(cuda_device), idx.to(cuda_device), temperature=0.7, out=z)
    spread = 1 + 2 * d64(wide[:, 5:vocab + 5]).abs().max(-1).values / 0.7
    # each is within its bound of the exact result
    within(got.rows, d64(want.rows), 2 * 64 * U32 * 0.49 * (spread + 1))
    within(z, d64(want.grad), 2 * rounding(dtype) * d64(want.grad).abs() +
           4 * (spread[:, None] + 64) * U32 * 2 * 0.7)
    assert bool(torch.isnan(on[:, :5]).all()) and bool(torch.isnan(on[:, vocab + 5:]).all())


def test_distill_refuses_an_overlapping_gradient(cuda_device):
    big = torch.zeros(4, 64, device=cuda_device)
    t, idx = torch.zeros(4, 1, device=cuda_device), torch.zeros(4, 1, dtype=torch.int32, device=cuda_device)
    for logits, out in ((big[:, :32], big[:, 8:40]), (big[:, :32], big[:, 16:48]),
                        (big[1:, :32], big[:3, :32]), (big.view(-1)[:80].view(4, 20), big[:, :20])):
        k = logits.shape[0]
        with pytest.raises(RuntimeError, match="overlap"):
            ops.topk_distill(logits, t[:k], idx[:k], out=out)
    for logits, out in ((big[:, :32], big[:, :32]), (big[:, :32], big[:, 32:]), (big[:2], big[2:]),
                        (big[:, 40:], big[:, :24])):
        k = logits.shape[0]
        logits.zero_()
        got = ops.topk_distill(logits, t[:k], idx[:k], out=out)
        v = logits.shape[1]
        within(got.rows, torch.full((k,), math.log(v), dtype=torch.float64), torch.tensor(64 * U32 * 8))
        assert abs(float(out[0, 1]) - 1 / v) <= 64 * U32


# --------------------------------------------------------------- embedding

@pytest.mark.parametrize("tokens,vocab,dim,kind", [
    (131072, 50257, 8, "uniform"), (131073, 1009, 12, "words"), (262145, 300, 9, "runs"),
    (300000, 70001, 4, "words"), (140000, 5003, 33, "same"), (140001, 5003, 32, "outside"),
    (131500, 257, 64, "uniform"), (131501, 257, 66, "words"),
    # chunks of every length, and rows cut into slices
    (16384, 50257, 768, "words"), (32768, 4001, 1024, "runs"), (8192, 9001, 4096, "words"),
    (4097, 300, 2052, "same"), (2000, 300, 20011, "words"), (9785, 300, 64, "runs"),
    (70, 40, 5000, "words"), (600, 7, 1030, "uniform"),
])
def test_embedding_grad_long_lists(cuda_device, tokens, vocab, dim, kind):
    base.test_embedding_grad(cuda_device, tokens, vocab, dim, kind)


@pytest.mark.parametrize("tokens", [32, 33, 48, 63, 64, 65, 100, 128, 129, 512, 513, 1000])
@pytest.mark.parametrize("dim", [4, 40, 520])
def test_embedding_grad_few_tokens(cuda_device, tokens, dim):
    for vocab in (3, 5000):
        for kind in ("words", "outside"):
            base.test_embedding_grad(cuda_device, tokens, vocab, dim, kind)


# ------------------------------------------------------------ residual norm

WIDE = [  # rows, dim, groups (0: one gate, None: none)
    (160, 4100, 0), (37, 6000, 37), (10, 8191, 2), (300, 5121, 3), (450, 8192, None),
    (12, 9000, 4), (9, 16383, 3), (150, 12288, 0), (149, 10001, None), (40, 32768, 8),
    (3, 66000, 3), (2, 65536, 0),
]


@pytest.mark.parametrize("rows,dim,groups", WIDE)
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_residual_norm_wide(cuda_device, rows, dim, groups, kind):
    for i in range(2):
        types = base.NORM_TYPES[(rows + dim + i) % 5]
        a = base._norm_args(gen(dim + i), rows, dim, kind, types, groups, bias=(rows + i) % 2 == 0)
        base._check_norm(cuda_device, a, kind, (0.5, -1.7)[i], rows)


def _surrounded(t, dev, before=3, after=6):
    """`t` [rows, dim] on the device in rows among columns of NaN, off 16 bytes."""
    wide = torch.full((t.shape[0], t.shape[1] + before + after), float("nan"), dtype=t.dtype, device=dev)
    wide[:, before:before + t.shape[1]] = t.to(dev)
    return wide[:, before:before + t.shape[1]]


@pytest.mark.parametrize("dim", [1, 7, 33, 148, 769, 1600, 4095, 4101, 8191, 9003])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_residual_norm_among_nan(cuda_device, dim, kind):
    if kind == "layer" and dim == 1:
        pytest.skip("the layer norm of one value has no deviation")
    rows = 700 if dim < 1000 else 170
    for types in base.NORM_TYPES[:3]:
        a = base._norm_args(gen(dim), rows, dim, kind, types, 0, bias=kind == "layer")
        a["h"] = a["h"] + (2 * torch.randint(0, 2, (rows, 1), generator=gen(1)) - 1).to(a["h"].dtype)
        on = {k: None if v is None else v.to(cuda_device) for k, v in a.items()}
        pars = {k: on[k] for k in ("post_bias", "pre_bias", "gate")}
        g_new, g_n = (randn(gen(2 + i), rows, dim, dtype=types[i]).to(cuda_device) for i in (0, 1))

        def both(x, h, gn, gg):
            new, n, stats = ops.residual_norm_forward(x, h, on["post_weight"], on["pre_weight"],
                                                      kind=kind, **pars)
            return (new, n) + tuple(ops.residual_norm_backward(gn, gg, x, h, stats,
                                                               on["post_weight"], on["pre_weight"],
                                                               kind=kind, **pars))

        plain = both(on["x"], on["h"], g_new, g_n)
        got = both(*(_surrounded(t, cuda_device) for t in (on["x"], on["h"], g_new, g_n)))
        for p, v in zip(plain, got):
            if p is None:
                continue
            # the same formula in another order of sums: 256 u of the terms, whose sizes stay
            # below 64 in a row (and 64 a row in a parameter's sum), and a rounding each
            per = rows if v.dim() == 1 else 1
            size = 64.0 * (1 + math.sqrt(dim) / 16) * per
            within(v, d64(p), 2 * (256 * U32 * size + rounding(v.dtype) * d64(p).abs()))


@pytest.mark.parametrize("dim", [40, 1601, 4096, 9000])
def test_residual_norm_rows_of_stride_zero(cuda_device, dim):
    """One row of the block for all rows, and an expanded incoming gradient."""
    g = gen(dim)
    w = (1 + randn(g, dim, scale=0.2)).to(cuda_device)
    x, h = randn(g, 200, dim).to(cuda_device), randn(g, 1, dim).to(cuda_device)
    up = randn(g, 1, dim).to(cuda_device)
    args = (x, h.expand(200, dim), up.expand(200, dim))
    results = []
    for xs, hs, gs in (args, [t.contiguous() for t in args]):
        new, n, stats = ops.residual_norm_forward(xs, hs, w, w)
        b = ops.residual_norm_backward(gs, gs, xs, hs, stats, w, w)
        results.append((new, n, b.x, b.h, b.post_weight, b.pre_weight))
    for got, want in zip(*results):
        assert torch.equal(got, want)


def test_operators_in_a_captured_graph(cuda_device):
    """The operators record into a CUDA graph, and a replay on new values gives
    the direct calls' bits."""
    g = gen(77)
    tokens, vocab, dim, top = 300, 1000, 96, 8
    table = randn(g, vocab, dim, dtype=BF16).to(cuda_device)
    w = (1 + randn(g, dim, scale=0.1)).to(cuda_device)
    ids = torch.randint(0, vocab, (tokens,), generator=g).to(cuda_device)
    z = randn(g, tokens, vocab, dtype=BF16).to(cuda_device)
    t = randn(g, tokens, top).to(cuda_device)
    at = torch.randint(0, vocab, (tokens, top), generator=g).to(cuda_device)

    def step():
        x = ops.scaled_embedding(ids, table, 2.0)
        new, n, stats = ops.residual_norm_forward(x, x, w, w)
        d = ops.topk_distill(z, t, at)
        b = ops.residual_norm_backward(new, n, x, x, stats, w, w)
        e = ops.scaled_embedding_grad(ids, b.x, vocab, 2.0)
        return new, n, b.h, b.post_weight, d.loss, d.grad, e

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    ids.copy_(ids.flip(0))
    z.copy_(z.flip(1))
    table.mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(held, step()):
        assert torch.equal(a, b)


def test_embedding_long_activations(cuda_device):
    """Activations and incoming gradients of more than 2^31 elements."""
    tokens, vocab, dim = 70000, 64, 32768
    g = gen(61)
    table = randn(g, vocab, dim, dtype=BF16).to(cuda_device)
    ids = torch.randint(0, vocab - 1, (tokens,), generator=g).to(cuda_device)
    ids[-1] = vocab - 1
    out = ops.scaled_embedding(ids, table, 1.0)
    for n in (0, 65535, 65536, tokens - 2, tokens - 1):
        assert torch.equal(out[n], table[ids[n]])
    out[:-1] = 0
    grad = ops.scaled_embedding_grad(ids, out, vocab, 2.0)
    assert torch.equal(grad[-1], table[-1].float() * 2) and not bool(grad[:-1].any())


def test_residual_norm_long_activations(cuda_device):
    """Rows whose element offsets pass 2^31: the last rows against the same rows
    alone, and the parameters' gradients when only they have an upstream one."""
    rows, dim, last = 66000, 32768, 3
    g = gen(62)
    w1, w2, gate = ((1 + randn(g, dim, scale=0.1)).to(cuda_device) for _ in range(3))
    x = torch.zeros(rows, dim, dtype=BF16, device=cuda_device)
    h = torch.zeros(rows, dim, dtype=BF16, device=cuda_device)
    up = torch.zeros(rows, dim, dtype=BF16, device=cuda_device)
    parts = [randn(g, last, dim, dtype=BF16).to(cuda_device) for _ in range(3)]
    for t, p in zip((x, h, up), parts):
        t[-last:] = p
    new, n, stats = ops.residual_norm_forward(x, h, w1, w2, gate=gate)
    b = ops.residual_norm_backward(up, up, x, h, stats, w1, w2, gate=gate)
    leaves = [d64(t).requires_grad_() for t in (*parts[:2], w1, w2, gate)]
    want = ref.residual_norm(leaves[0], leaves[1], leaves[2], leaves[3], gate=leaves[4])
    grads = torch.autograd.grad(want, leaves, [d64(parts[2])] * 2)
    u16 = rounding(BF16)
    for got, w in zip((new, n), want):
        w = w.detach()
        within(got[-last:], w, u16 * w.abs() + 64 * U32 * 16)
        assert not bool(got[:-last].any())
    for got, w in zip((b.x[-last:], b.h[-last:], b.post_weight, b.pre_weight, b.gate), grads):
        # sums over a row of 32768: 256 u of terms below 16, as many as sqrt(32768) of one sign
        within(got, w, rounding(got.dtype) * w.abs() + 256 * U32 * 16 * 12)
    assert not bool(b.x[:-last].any())


def test_distill_indices_beyond_32_bits(cuda_device):
    g = gen(63)
    z, t = randn(g, 5, 300), randn(g, 5, 4)
    idx = torch.randint(0, 300, (5, 4), generator=g)
    idx[0, 1], idx[1, 2], idx[2, 0] = 1 << 32, (1 << 40) + 7, -(1 << 33)
    idx[3] = torch.tensor([1 << 31, (1 << 32) + 1, -1, 1 << 62])
    got = base._check_distill(cuda_device, z, t, idx, 1.0, None, 1.0)
    assert float(got.rows[3]) == 0.0
    ids = torch.tensor([1, 1 << 32, (1 << 33) + 1, -(1 << 40), 2], device=cuda_device)
    table = randn(g, 4, 24).to(cuda_device)
    out = ops.scaled_embedding(ids, table)
    assert torch.equal(out[[0, 4]], table[[1, 2]]) and not bool(out[1:4].any())
    grad = ops.scaled_embedding_grad(ids, out + 1, 4)
    assert torch.equal(grad[[1, 2]], table[[1, 2]] + 1) and not bool(grad[[0, 3]].any())
    long = ids.repeat(300)
    grad = ops.scaled_embedding_grad(long, torch.ones(1500, 24, device=cuda_device), 4)
    assert torch.equal(grad[:, 0].cpu(), torch.tensor([0.0, 300.0, 300.0, 0.0]))
