"""The operators' host side on a machine without a GPU: refusals of the C ABI
and of the torch front end, and the packing of the descriptors."""
import ctypes

import pytest
import torch

from mdq_b200 import _lib, ops
from mdq_b200._lib import MDQ_ERR_INVALID_ARG, MDQ_ERR_TOO_LARGE, MDQ_ERR_UNSUPPORTED

PTR = 0x1000


def _embed(**kw):
    d = _lib.EmbedDesc(PTR, PTR, PTR, 10, 100, 64, 64, 1.0, _lib.MDQ_F32, _lib.MDQ_F32,
                       _lib.MDQ_I64)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def _embed_grad(**kw):
    d = _lib.EmbedGradDesc(PTR, PTR, PTR, PTR, 1 << 40, 10, 100, 64, 64, -1, 1.0, _lib.MDQ_F32,
                           _lib.MDQ_F32, _lib.MDQ_I64, 0, 0)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def _norm(**kw):
    d = _lib.ResidualNormDesc(x=PTR, h=PTR, x_new=PTR, n=PTR, stats=PTR, post_weight=PTR,
                              pre_weight=PTR, rows=8, dim=64, x_stride=64, h_stride=64,
                              gate_rows=1, residual_scale=1.0, eps=1e-5)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def _norm_grad(f=None, **kw):
    d = _lib.ResidualNormGradDesc(f=_norm(**(f or {})), grad_new=PTR, grad_n=PTR, grad_x=PTR,
                                  grad_h=PTR, workspace=PTR, workspace_bytes=1 << 40,
                                  grad_new_stride=64, grad_n_stride=64)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def _distill(**kw):
    d = _lib.TopkDistillDesc(logits=PTR, teacher=PTR, index=PTR, row_loss=PTR, grad=PTR, rows=4,
                             vocab=100, logits_stride=100, grad_stride=100, top=8, temperature=1.0,
                             scale=1.0, index_dtype=_lib.MDQ_I64)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


I, U, T = MDQ_ERR_INVALID_ARG, MDQ_ERR_UNSUPPORTED, MDQ_ERR_TOO_LARGE


@pytest.mark.parametrize("name,make,kw,status,msg", [
    ("mdq_embed", _embed, dict(tokens=-1), I, "size"),
    ("mdq_embed", _embed, dict(vocab=0), I, "size"),
    ("mdq_embed", _embed, dict(dim=0), I, "size"),
    ("mdq_embed", _embed, dict(tokens=1 << 31), T, "2^31"),
    ("mdq_embed", _embed, dict(table_dtype=_lib.MDQ_I8), U, "MDQ_F32"),
    ("mdq_embed", _embed, dict(out_dtype=99), U, "MDQ_F32"),
    ("mdq_embed", _embed, dict(ids_dtype=_lib.MDQ_I16), U, "MDQ_I32"),
    ("mdq_embed", _embed, dict(table=None), I, "null"),
    ("mdq_embed_grad", _embed_grad, dict(tokens=-1), I, "size"),
    ("mdq_embed_grad", _embed_grad, dict(padding_idx=-2), I, "size"),
    ("mdq_embed_grad", _embed_grad, dict(grad=None), I, "null"),
    ("mdq_embed_grad", _embed_grad, dict(ids=None), I, "null"),
    ("mdq_embed_grad", _embed_grad, dict(grad_dtype=_lib.MDQ_U8), U, "MDQ_F32"),
    ("mdq_embed_grad", _embed_grad, dict(ids_dtype=_lib.MDQ_F32), U, "MDQ_I32"),
    ("mdq_embed_grad", _embed_grad, dict(grad_dtype=_lib.MDQ_BF16, accumulate=1), U, "accumulate"),
    ("mdq_embed_grad", _embed_grad, dict(tokens=1 << 31), T, "2^31"),
    ("mdq_residual_norm", _norm, dict(rows=-1), I, "size"),
    ("mdq_residual_norm", _norm, dict(dim=0), I, "size"),
    ("mdq_residual_norm", _norm, dict(gate_rows=0), I, "size"),
    ("mdq_residual_norm", _norm, dict(gate=PTR, gate_rows=3), I, "gate_rows"),
    ("mdq_residual_norm", _norm, dict(gate_rows=2), I, "gate_rows"),
    ("mdq_residual_norm", _norm, dict(kind=2), I, "kind"),
    ("mdq_residual_norm", _norm, dict(x=None), I, "null"),
    ("mdq_residual_norm", _norm, dict(x_new=None), I, "null"),
    ("mdq_residual_norm", _norm, dict(h=None), I, "block"),
    ("mdq_residual_norm", _norm, dict(post_weight=None), I, "post_weight"),
    ("mdq_residual_norm", _norm, dict(h=None, post_weight=None, pre_weight=None), I, "neither"),
    ("mdq_residual_norm", _norm, dict(pre_weight=None, pre_bias=PTR), I, "pre_bias"),
    ("mdq_residual_norm", _norm, dict(x_dtype=_lib.MDQ_I8), U, "MDQ_F32"),
    ("mdq_residual_norm", _norm, dict(param_dtype=_lib.MDQ_I8), U, "MDQ_F32"),
    ("mdq_residual_norm", _norm, dict(rows=1 << 31), T, "2^31"),
    ("mdq_residual_norm_grad", _norm_grad, dict(grad_n_stride=-1), I, "size"),
    ("mdq_residual_norm_grad", _norm_grad, dict(grad_x=None), I, "null"),
    ("mdq_residual_norm_grad", _norm_grad, dict(grad_h=None), I, "null"),
    ("mdq_residual_norm_grad", _norm_grad, dict(f=dict(stats=None)), I, "null"),
    ("mdq_residual_norm_grad", _norm_grad, dict(f=dict(pre_weight=None)), I, "grad_n"),
    ("mdq_residual_norm_grad", _norm_grad, dict(workspace_bytes=0), I, "workspace"),
    ("mdq_topk_distill", _distill, dict(rows=-1), I, "size"),
    ("mdq_topk_distill", _distill, dict(vocab=0), I, "size"),
    ("mdq_topk_distill", _distill, dict(top=0), I, "size"),
    ("mdq_topk_distill", _distill, dict(top=1025), T, "1024"),
    ("mdq_topk_distill", _distill, dict(temperature=0.0), I, "temperature"),
    ("mdq_topk_distill", _distill, dict(temperature=float("nan")), I, "temperature"),
    ("mdq_topk_distill", _distill, dict(temperature=float("inf")), I, "temperature"),
    ("mdq_topk_distill", _distill, dict(upstream_stride=2), I, "upstream"),
    ("mdq_topk_distill", _distill, dict(logits=None), I, "null"),
    ("mdq_topk_distill", _distill, dict(row_loss=None, loss=PTR), I, "row_loss"),
    ("mdq_topk_distill", _distill, dict(grad_stride=99), I, "overlap"),
    ("mdq_topk_distill", _distill, dict(logits_dtype=_lib.MDQ_I8), U, "MDQ_F32"),
    ("mdq_topk_distill", _distill, dict(index_dtype=_lib.MDQ_F32), U, "MDQ_I32"),
    ("mdq_topk_distill", _distill, dict(vocab=1 << 31, grad_stride=1 << 31), T, "2^31"),
])
def test_c_entry_points_refuse(name, make, kw, status, msg):
    lib = _lib.load()
    assert getattr(lib, name)(ctypes.byref(make(**kw)), None) == status
    assert msg in lib.mdq_last_error().decode()
    assert getattr(lib, name)(None, None) == MDQ_ERR_INVALID_ARG


def test_workspace_queries_refuse():
    lib = _lib.load()
    need = ctypes.c_int64(-1)
    for name in ("mdq_embed_grad_workspace_bytes", "mdq_residual_norm_grad_workspace_bytes"):
        fn = getattr(lib, name)
        assert fn(-1, 10, 10, ctypes.byref(need)) == MDQ_ERR_INVALID_ARG
        assert fn(1, 0, 10, ctypes.byref(need)) == MDQ_ERR_INVALID_ARG
        assert fn(1, 10, 0, ctypes.byref(need)) == MDQ_ERR_INVALID_ARG
        assert fn(1, 10, 10, None) == MDQ_ERR_INVALID_ARG
        assert fn(4, 4, 4, ctypes.byref(need)) == 0 and need.value >= 0


def test_empty_calls_need_no_device():
    lib = _lib.load()
    assert lib.mdq_embed(ctypes.byref(_embed(tokens=0)), None) == 0
    assert lib.mdq_residual_norm(ctypes.byref(_norm(rows=0)), None) == 0
    assert lib.mdq_topk_distill(ctypes.byref(_distill(rows=0)), None) == 0


@pytest.mark.parametrize("fmt,mirror", [
    (ops._EMBED, _lib.EmbedDesc), (ops._EMBED_GRAD, _lib.EmbedGradDesc),
    (ops._NORM, _lib.ResidualNormDesc), (ops._NORM_GRAD, _lib.ResidualNormGradDesc),
    (ops._DISTILL, _lib.TopkDistillDesc)])
def test_descriptors_pack_as_their_mirrors(fmt, mirror):
    """Distinct values packed in order land in the mirror's fields in order."""
    assert fmt.size == ctypes.sizeof(mirror)
    codes = "".join(c * int(n or 1) for n, c in __import__("re").findall(r"(\d*)([Qqfi])", fmt.format))
    values = [float(i + 1) if c == "f" else i + 1 for i, c in enumerate(codes)]
    d = mirror.from_buffer_copy(fmt.pack(*values))

    def flat(s):
        for name, kind in s._fields_:
            v = getattr(s, name)
            yield from flat(v) if isinstance(v, ctypes.Structure) else (v,)

    assert list(flat(d)) == values


def test_front_end_refuses_cpu_tensors():
    x, w, ids = torch.zeros(4, 8), torch.ones(8), torch.zeros(4, dtype=torch.int64)
    for call in (lambda: ops.scaled_embedding(ids, x),
                 lambda: ops.scaled_embedding_grad(ids, x, 10),
                 lambda: ops.residual_norm(x, x, w, w),
                 lambda: ops.residual_norm_backward(x, x, x, x, torch.zeros(4, 4), w, w),
                 lambda: ops.topk_distill(x, x, ids),
                 lambda: ops.topk_distill_loss(x, x, ids)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_row_strides():
    t = torch.zeros(6, 4, 10)
    assert ops._row_stride(t, "t") == 10
    assert ops._row_stride(t[:, :, :7], "t") == 10
    assert ops._row_stride(t[:, 1], "t") == 40
    assert ops._row_stride(t[0, 0, :7], "t") == 7
    assert ops._row_stride(torch.zeros(10).expand(5, 10), "t") == 0
    with pytest.raises(RuntimeError, match="evenly strided"):
        ops._row_stride(t[:, :3], "t")
    with pytest.raises(RuntimeError, match="contiguous"):
        ops._row_stride(torch.zeros(5, 10).t(), "t")
