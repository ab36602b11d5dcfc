"""Residual norm (mdq_b200.ops) on the paths that only very wide rows reach:
rows off 16 bytes of more than 32768 columns, whose backward pass holds a row in
a cluster's registers, and rows that no cluster holds (more than 65536 columns
off 16 bytes, with means, biases or a gate of groups in the backward pass; more
than 131072 otherwise), which plain kernels read several times.

The bounds are those of test_gpu_ops.py, whose checks these tests call.
"""
import math

import pytest
import torch

import test_gpu_ops as base
from mdq_b200 import ops
from ops_reference import U32, d64, rounding
from test_gpu_ops import gen, randn, within
from test_gpu_ops_ranges import _surrounded

pytestmark = pytest.mark.gpu

PATHS = [  # rows, dim, groups (0: one gate, None: none)
    # a cluster's registers, off 16 bytes: two chunks a thread, four chunks
    (37, 33001, 0), (40, 33001, 4), (3, 33001, None), (24, 40001, 3), (5, 50001, 5), (50, 65535, 0),
    (20, 131069, None), (3, 98307, 0),
    # no cluster: forward alone (rows on 16 bytes of 65537 to 131072 have one), or both passes
    (40, 70001, 0), (24, 70001, 4), (3, 70001, None), (6, 70000, 3), (1, 131080, 0), (33, 131080, 11),
    (2, 200003, None),
]


@pytest.mark.parametrize("rows,dim,groups", PATHS)
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_residual_norm_very_wide(cuda_device, rows, dim, groups, kind):
    for i in range(2):
        types = base.NORM_TYPES[(rows + dim + 2 * i) % 5]
        a = base._norm_args(gen(dim + i), rows, dim, kind, types, groups, bias=(rows + i) % 2 == 0)
        base._check_norm(cuda_device, a, kind, (0.5, -1.7)[i], rows)


@pytest.mark.parametrize("part", ["first", "last", "no grad_new", "no grad_n"])
@pytest.mark.parametrize("dim", [33001, 70001, 131080])
def test_residual_norm_very_wide_parts(cuda_device, part, dim):
    for kind, types in (("rms", base.NORM_TYPES[2]), ("layer", base.NORM_TYPES[0])):
        a = base._norm_args(gen(dim), 5, dim, kind, types, 0, bias=kind == "layer")
        if part == "first":
            a["h"] = a["post_weight"] = a["post_bias"] = a["gate"] = None
        if part == "last":
            a["pre_weight"] = a["pre_bias"] = None
        grads = {"no grad_new": ("n",), "no grad_n": ("new",)}.get(part, ("new", "n"))
        base._check_norm(cuda_device, a, kind, 1.0, dim, grads)


@pytest.mark.parametrize("dim", [33000, 33001, 65540, 70001])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_residual_norm_very_wide_among_nan(cuda_device, dim, kind):
    """Rows off 16 bytes, surrounded by columns of NaN, against the same rows alone."""
    rows = 21
    for types in base.NORM_TYPES[:3]:
        a = base._norm_args(gen(dim), rows, dim, kind, types, 0, bias=kind == "layer")
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
            # as in test_residual_norm_among_nan: the same formula in another order of sums
            size = 64.0 * (1 + math.sqrt(dim) / 16) * (rows if v.dim() == 1 else 1)
            within(v, d64(p), 2 * (256 * U32 * size + rounding(v.dtype) * d64(p).abs()))
