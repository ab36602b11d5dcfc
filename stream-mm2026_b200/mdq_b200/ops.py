"""Training-step operators beside the optimizer: the memory-bound parts of a
language model's step, as CUDA kernels behind the C ABI of ``include/mdq_ops.h``.

  scaled_embedding, scaled_embedding_grad
      out = scale * table[ids], and the table's gradient by sorted tokens
  residual_norm, residual_norm_forward, residual_norm_backward
      x_new = residual_scale * x + gate * norm(h), n = norm(x_new)
  topk_distill, topk_distill_loss
      distillation from a teacher's top logits, loss and gradient in one pass

``scaled_embedding``, ``residual_norm`` and ``topk_distill_loss`` take part in
autograd; the others are the passes themselves, for programs that run their own
backward.  There is no forward-mode derivative: dual tensors are refused.  Every
call works on the current stream of its tensors' device, allocates its results and
scratch through torch's caching allocator and does not wait for the device.
Tensors are float32 or bfloat16; the last dimension is contiguous and rows may be
strided.  CPU tensors are refused.
"""
from __future__ import annotations

import ctypes
import struct
from functools import lru_cache
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from . import _lib

_FLOAT = {torch.float32: _lib.MDQ_F32, torch.bfloat16: _lib.MDQ_BF16}
_IDS = {torch.int32: _lib.MDQ_I32, torch.int64: _lib.MDQ_I64}
_KINDS = {"rms": _lib.NORM_RMS, "layer": _lib.NORM_LAYER}

# The descriptors of mdq_ops.h as packed bytes: one pack costs far less host
# time than one ctypes store a field (tests check the mirrors' offsets).
_EMBED = struct.Struct("=3Q4qf3i")
_EMBED_GRAD = struct.Struct("=4Q6qf5i")
_NORM = struct.Struct("=10Q5q2f4i")
_NORM_GRAD = struct.Struct("=10Q5q2f4i10Q3q")
_DISTILL = struct.Struct("=8Q5qi2f3i")


# These checks run on every call, beside kernels of a few microseconds: they ask
# for a device's index rather than compare devices, and look sizes up once.


def _float_code(t: torch.Tensor, what: str) -> int:
    code = _FLOAT.get(t.dtype)
    if code is None:
        raise RuntimeError(f"{what} must be float32 or bfloat16")
    return code


def _device(t: torch.Tensor, what: str) -> int:
    """Index of the device a tensor is on."""
    index = t.get_device()
    if index < 0 or not t.is_cuda:
        raise RuntimeError(f"{what} must be CUDA")
    return index


def _on(t: torch.Tensor, index: int, what: str) -> None:
    if t.get_device() != index:
        raise RuntimeError(f"{what} must be on cuda:{index}")


def _no_tangents(*tensors: Optional[torch.Tensor]) -> None:
    """Refuses tensors with a forward-mode tangent, which the kernels do not see."""
    if forward_ad._current_level < 0 or not torch._C._is_fwd_grad_enabled():
        return
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError("the operators have no forward-mode derivative")


def _row_stride(t: torch.Tensor, what: str) -> int:
    """Elements from one row (last dimension) of ``t`` to the next."""
    if t.is_contiguous():
        return t.shape[-1]
    if t.dim() > 2:
        try:
            t = t.view(-1, t.shape[-1])
        except RuntimeError:
            raise RuntimeError(f"{what}: rows must be evenly strided") from None
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise RuntimeError(f"{what}: the last dimension must be contiguous")
    return t.stride(0) if t.dim() == 2 else t.shape[-1]


def _row_count(t: torch.Tensor) -> int:
    """Rows of ``t``, also when its rows or columns are none."""
    shape = t.shape
    if len(shape) == 2:
        return shape[0]
    n = 1
    for k in shape[:-1]:
        n *= k
    return n


def _like(t: torch.Tensor) -> torch.Tensor:
    """An uninitialised contiguous tensor of ``t``'s shape and dtype."""
    if t.is_contiguous():
        return torch.empty_like(t)
    return torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _usable(t: torch.Tensor) -> torch.Tensor:
    """An incoming gradient in a layout the kernels take."""
    if t.is_contiguous():
        return t
    try:
        _row_stride(t, "gradient")
        return t
    except RuntimeError:
        return t.contiguous()


def _empty(shape, strides, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    """torch.empty in two thirds of its host time (1.5 us against 2.3)."""
    return torch.empty_strided(shape, strides, dtype=dtype, device=device)


def _run(fn, index: int, desc: bytes) -> None:
    """One entry point of the library on the current stream of a device."""
    if torch._C._cuda_getDevice() == index:
        st = fn(desc, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            st = fn(desc, torch._C._cuda_getCurrentRawStream(index))
    if st:
        _lib.check(st)


@lru_cache(maxsize=None)
def _entry(name: str):
    return getattr(_lib.load(), name)


@lru_cache(maxsize=1024)
def _workspace_bytes(name: str, a: int, b: int, c: int) -> int:
    need = ctypes.c_int64(0)
    _lib.check(_entry(name)(a, b, c, ctypes.byref(need)))
    return need.value


def _workspace(name: str, index: int, a: int, b: int, c: int):
    need = _workspace_bytes(name, a, b, c)
    if need == 0:
        return None, 0, 0
    ws = _empty((need,), (1,), torch.uint8, _cuda(index))
    return ws, ws.data_ptr(), need


@lru_cache(maxsize=None)
def _cuda(index: int) -> torch.device:
    return torch.device("cuda", index)


# --------------------------------------------------------------- embedding

def _check_ids(ids: torch.Tensor, dev: int) -> int:
    code = _IDS.get(ids.dtype)
    if code is None:
        raise RuntimeError("ids must be int32 or int64")
    _on(ids, dev, "ids")
    if not ids.is_contiguous():
        raise RuntimeError("ids must be contiguous")
    return code


def _embedding_forward(ids, table, scale, out_dtype):
    dev = _device(table, "table")
    _no_tangents(table)
    if table.dim() != 2 or table.numel() == 0:
        raise RuntimeError("table must be [vocab, dim], neither of them 0")
    ids_code, table_code = _check_ids(ids, dev), _float_code(table, "table")
    stride = _row_stride(table, "table")
    vocab, dim = table.shape
    out = torch.empty((*ids.shape, dim), dtype=out_dtype or table.dtype, device=table.device)
    out_code = _float_code(out, "out_dtype")
    _run(_entry("mdq_embed"), dev, _EMBED.pack(
        table.data_ptr(), ids.data_ptr(), out.data_ptr(), ids.numel(), vocab, dim, stride,
        scale, table_code, out_code, ids_code))
    return out


def scaled_embedding_grad(ids: torch.Tensor, grad_out: torch.Tensor, vocab: int,
                          scale: float = 1.0, *, dtype: torch.dtype = torch.float32,
                          padding_idx: Optional[int] = None, out: Optional[torch.Tensor] = None,
                          accumulate: bool = False) -> torch.Tensor:
    """Gradient of ``scaled_embedding`` with respect to its table: the rows of
    ``grad_out`` [*ids.shape, dim] summed by id, times ``scale``, as a dense
    [vocab, dim] tensor.  Sums run in fp32 in a fixed order, so repeated calls
    give the same bits.  Ids outside [0, vocab) and ``padding_idx`` contribute
    nothing.

    ``out`` (contiguous, [vocab, dim]) receives the result; with ``accumulate``
    (fp32) the sums are added to it, and only the rows that occur are touched (by
    additions that take subnormal values as zero).  To autograd that is an in-place
    operation on ``out``.
    """
    dev = _device(grad_out, "grad_out")
    _no_tangents(grad_out, out)
    ids_code, go_code = _check_ids(ids, dev), _float_code(grad_out, "grad_out")
    if grad_out.dim() < 1 or grad_out.shape[:-1] != ids.shape:
        raise RuntimeError("grad_out must be [*ids.shape, dim]")
    dim = grad_out.shape[-1]
    if vocab < 1 or dim < 1:
        raise RuntimeError("vocab and dim must be positive")
    if padding_idx is not None and not 0 <= padding_idx < vocab:
        raise RuntimeError("padding_idx must lie in [0, vocab)")
    stride = _row_stride(grad_out, "grad_out")
    given = out is not None
    if not given:
        if accumulate:
            raise RuntimeError("accumulate needs out")
        out = _empty((vocab, dim), (dim, 1), dtype, grad_out.device)
    else:
        _on(out, dev, "out")
        if out.shape != (vocab, dim) or not out.is_contiguous():
            raise RuntimeError("out must be contiguous [vocab, dim]")
        if accumulate and out.dtype != torch.float32:
            raise RuntimeError("accumulate needs a float32 out")
    out_code, tokens = _float_code(out, "gradient"), ids.numel()
    ws, ws_ptr, ws_bytes = _workspace("mdq_embed_grad_workspace_bytes", dev, tokens, vocab, dim)
    _run(_entry("mdq_embed_grad"), dev, _EMBED_GRAD.pack(
        grad_out.data_ptr(), ids.data_ptr(), out.data_ptr(), ws_ptr, ws_bytes, tokens, vocab, dim,
        stride, -1 if padding_idx is None else padding_idx, scale, go_code, out_code, ids_code,
        1 if accumulate else 0, 0))
    if given:
        increment_version(out)   # backward passes that need its former values refuse
    return out


class _ScaledEmbedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, ids, scale, out_dtype, padding_idx):
        ctx.save_for_backward(ids)
        ctx.args = (table.shape[0], scale, table.dtype, padding_idx)
        return _embedding_forward(ids, table, scale, out_dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        (ids,) = ctx.saved_tensors
        vocab, scale, dtype, padding_idx = ctx.args
        grad = scaled_embedding_grad(ids, _usable(grad_out), vocab, scale, dtype=dtype,
                                     padding_idx=padding_idx)
        return grad, None, None, None, None


def scaled_embedding(ids: torch.Tensor, table: torch.Tensor, scale: float = 1.0, *,
                     out_dtype: Optional[torch.dtype] = None,
                     padding_idx: Optional[int] = None) -> torch.Tensor:
    """``scale * table[ids]`` as [*ids.shape, dim] in ``out_dtype`` (the table's
    by default).  ids: int32 or int64, contiguous; an id outside [0, vocab)
    gives zeros.  The row of ``padding_idx`` is looked up as any other and gets
    no gradient."""
    if padding_idx is not None and not 0 <= padding_idx < table.shape[0]:
        raise RuntimeError("padding_idx must lie in [0, vocab)")
    if table.requires_grad and torch.is_grad_enabled():
        return _ScaledEmbedding.apply(table, ids, scale, out_dtype, padding_idx)
    return _embedding_forward(ids, table, scale, out_dtype)


# ----------------------------------------------------------- residual norm

class ResidualNormGrads(NamedTuple):
    """Gradients of ``residual_norm``'s arguments (None where there was none)."""

    x: torch.Tensor
    h: Optional[torch.Tensor]
    post_weight: Optional[torch.Tensor]
    pre_weight: Optional[torch.Tensor]
    post_bias: Optional[torch.Tensor]
    pre_bias: Optional[torch.Tensor]
    gate: Optional[torch.Tensor]


def _ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _parameter(t, shape, dtype, dev, what) -> int:
    if t.shape != shape:
        raise RuntimeError(f"{what} must be [dim]")
    if t.dtype != dtype or not t.is_contiguous():
        raise RuntimeError(f"{what}: parameters must be contiguous and of one dtype")
    if t.get_device() != dev:
        raise RuntimeError(f"{what} must be on cuda:{dev}")
    return t.data_ptr()


def _norm_fields(x, h, post_weight, pre_weight, post_bias, pre_bias, gate, residual_scale, eps,
                 kind, x_new, n, stats):
    """Checks the arguments and returns the fields of mdq_residual_norm_desc."""
    dev = _device(x, "x")
    x_code = _float_code(x, "x")
    code = _KINDS.get(kind)
    if code is None:
        raise RuntimeError("kind must be 'rms' or 'layer'")
    shape = x.shape
    if not shape or shape[-1] < 1:
        raise RuntimeError("x must be [..., dim]")
    dim, rows = shape[-1], _row_count(x)
    if h is not None:
        _on(h, dev, "h")
        h_code = _float_code(h, "h")
        if h.shape != shape:
            raise RuntimeError("h must have x's shape")
        h_stride = _row_stride(h, "h")
        if post_weight is None:
            raise RuntimeError("h needs post_weight")
    else:
        h_code, h_stride = x_code, 0
        if post_weight is not None or post_bias is not None or gate is not None:
            raise RuntimeError("gate and post parameters need h")
        if pre_weight is None:
            raise RuntimeError("either h or pre_weight is needed")
        if residual_scale != 1.0:
            raise RuntimeError("residual_scale needs h")
    if pre_weight is None and pre_bias is not None:
        raise RuntimeError("pre_bias needs pre_weight")
    first = pre_weight if post_weight is None else post_weight
    dtype, one = first.dtype, (dim,)
    p_code = _FLOAT.get(dtype)
    if p_code is None:
        raise RuntimeError("parameters must be float32 or bfloat16")
    post_w = post_b = pre_w = pre_b = 0
    if post_weight is not None:
        post_w = _parameter(post_weight, one, dtype, dev, "post_weight")
    if post_bias is not None:
        post_b = _parameter(post_bias, one, dtype, dev, "post_bias")
    if pre_weight is not None:
        pre_w = _parameter(pre_weight, one, dtype, dev, "pre_weight")
    if pre_bias is not None:
        pre_b = _parameter(pre_bias, one, dtype, dev, "pre_bias")
    gate_rows = 1
    if gate is not None:
        _on(gate, dev, "gate")
        if gate.dtype != dtype or not gate.is_contiguous():
            raise RuntimeError("gate: parameters must be contiguous and of one dtype")
        if gate.dim() not in (1, 2) or gate.shape[-1] != dim:
            raise RuntimeError("gate must be [dim] or [groups, dim]")
        if gate.dim() == 2:
            gate_rows = gate.shape[0]
            if gate_rows < 1 or rows % gate_rows:
                raise RuntimeError("gate's groups must divide the rows")
    return dev, (x.data_ptr(), _ptr(h), _ptr(x_new), _ptr(n), _ptr(stats), post_w, post_b, pre_w,
                 pre_b, _ptr(gate), rows, dim, _row_stride(x, "x"), h_stride, gate_rows, residual_scale, eps, x_code, h_code,
                 p_code, code)


def residual_norm_forward(x, h, post_weight, pre_weight, *, post_bias=None, pre_bias=None,
                          gate=None, residual_scale: float = 1.0, eps: float = 1e-5,
                          kind: str = "rms", want_stats: bool = True):
    """The forward pass of ``residual_norm``: (x_new, n, stats).  stats ([rows,
    4] fp32) is what ``residual_norm_backward`` needs, None without
    ``want_stats``."""
    _device(x, "x")
    _no_tangents(x, h, post_weight, pre_weight, post_bias, pre_bias, gate)
    x_new = x if h is None else _like(x)
    n = None
    if pre_weight is not None:
        n = _like(x if h is None else h)
    stats = None
    if want_stats:
        stats = _empty((_row_count(x), 4), (4, 1), torch.float32, x.device)
    dev, fields = _norm_fields(x, h, post_weight, pre_weight, post_bias, pre_bias, gate,
                               residual_scale, eps, kind, None if h is None else x_new, n, stats)
    if x.numel():
        _run(_entry("mdq_residual_norm"), dev, _NORM.pack(*fields))
    return x_new, n, stats


def residual_norm_backward(grad_new, grad_n, x, h, stats, post_weight, pre_weight, *,
                           post_bias=None, pre_bias=None, gate=None, residual_scale: float = 1.0,
                           kind: str = "rms") -> ResidualNormGrads:
    """Gradients of ``residual_norm`` from its arguments and the forward pass's
    stats.  ``grad_new`` / ``grad_n``: the gradients of x_new (x's dtype) and n
    (h's dtype), None for zero.  x_new itself is recomputed, so it need not be
    kept."""
    if stats is None or stats.dtype != torch.float32 or not stats.is_contiguous() or \
            stats.numel() != 4 * _row_count(x):
        raise RuntimeError("stats must be the forward pass's")
    _no_tangents(grad_new, grad_n, x, h, stats, post_weight, pre_weight, post_bias, pre_bias, gate)
    dev, fields = _norm_fields(x, h, post_weight, pre_weight, post_bias, pre_bias, gate,
                               residual_scale, 0.0, kind, None, None, stats)
    _on(stats, dev, "stats")
    strides = []
    for t, like, what in ((grad_new, x, "grad_new"), (grad_n, x if h is None else h, "grad_n")):
        if t is None:
            strides.append(0)
            continue
        _on(t, dev, what)
        if t.shape != x.shape or t.dtype != like.dtype:
            raise RuntimeError(f"{what} must have its result's shape and dtype")
        strides.append(_row_stride(t, what))
    if grad_n is not None and pre_weight is None:
        raise RuntimeError("grad_n needs pre_weight")

    new = torch.empty_like
    gx, gh = _like(x), None if h is None else _like(h)
    g = ResidualNormGrads(gx, gh, None if post_weight is None else new(post_weight),
                          None if pre_weight is None else new(pre_weight),
                          None if post_bias is None else new(post_bias),
                          None if pre_bias is None else new(pre_bias),
                          None if gate is None else new(gate))
    if not x.numel():
        for t in g:
            if t is not None:
                t.zero_()
        return g
    ws, ws_ptr, ws_bytes = _workspace("mdq_residual_norm_grad_workspace_bytes", dev, fields[10],
                                      fields[11], fields[14])
    _run(_entry("mdq_residual_norm_grad"), dev, _NORM_GRAD.pack(
        *fields, _ptr(grad_new), _ptr(grad_n), gx.data_ptr(), _ptr(gh), _ptr(g.post_weight),
        _ptr(g.post_bias), _ptr(g.pre_weight), _ptr(g.pre_bias), _ptr(g.gate), ws_ptr, ws_bytes,
        *strides))
    return g


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, h, post_weight, pre_weight, post_bias, pre_bias, gate, residual_scale,
                eps, kind):
        ctx.set_materialize_grads(False)
        x_new, n, stats = residual_norm_forward(
            x, h, post_weight, pre_weight, post_bias=post_bias, pre_bias=pre_bias, gate=gate,
            residual_scale=residual_scale, eps=eps, kind=kind)
        ctx.save_for_backward(x, h, stats, post_weight, pre_weight, post_bias, pre_bias, gate)
        ctx.args = (residual_scale, kind)
        return (n,) if h is None else (x_new,) if n is None else (x_new, n)

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        x, h, stats, post_weight, pre_weight, post_bias, pre_bias, gate = ctx.saved_tensors
        grads = [None if t is None else _usable(t) for t in grads]
        grad_new, grad_n = (None, grads[0]) if h is None else (*grads, None)[:2]
        if grad_new is None and grad_n is None:
            return (None,) * 10
        g = residual_norm_backward(grad_new, grad_n, x, h, stats, post_weight, pre_weight,
                                   post_bias=post_bias, pre_bias=pre_bias, gate=gate,
                                   residual_scale=ctx.args[0], kind=ctx.args[1])
        return (*g, None, None, None)


def residual_norm(x, h, post_weight, pre_weight, *, post_bias=None, pre_bias=None, gate=None,
                  residual_scale: float = 1.0, eps: float = 1e-5, kind: str = "rms"):
    """The end of a block and the beginning of the next, in one pass:

        x_new = residual_scale * x + gate * (norm(h) * post_weight + post_bias)
        n     = norm(x_new) * pre_weight + pre_bias

    and returns (x_new, n).  x [..., dim] is the residual stream, h the block's
    output; they may differ in dtype (an fp32 stream with bf16 blocks); x_new has
    x's dtype, n has h's.  kind: "rms" or "layer".  gate: None, [dim], or
    [groups, dim] with one row for each run of rows / groups consecutive rows (an
    adaptive gate of every sequence of a batch).  Before the first block pass
    h = post_weight = None: n = norm(x) and x_new is x.  After the last one pass
    pre_weight = None: n is None."""
    args = (x, h, post_weight, pre_weight, post_bias, pre_bias, gate)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in args):
        out = _ResidualNorm.apply(*args, residual_scale, eps, kind)
        return (x, out[0]) if h is None else (out[0], out[1] if len(out) > 1 else None)
    x_new, n, _ = residual_norm_forward(
        x, h, post_weight, pre_weight, post_bias=post_bias, pre_bias=pre_bias, gate=gate,
        residual_scale=residual_scale, eps=eps, kind=kind, want_stats=False)
    return x_new, n


# ------------------------------------------------------------ distillation

class TopkDistill(NamedTuple):
    """``topk_distill``'s result: total loss [], loss of each row, and the
    gradient of the logits (None when it was not asked for)."""

    loss: torch.Tensor
    rows: torch.Tensor
    grad: Optional[torch.Tensor]


def _distill(logits, teacher, index, temperature, weight, scale, grad, upstream=None,
             want_loss=True):
    dev = _device(logits, "logits")
    _no_tangents(logits, teacher, weight, grad, upstream)
    code, t_code = _float_code(logits, "logits"), _float_code(teacher, "teacher_logits")
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise RuntimeError("logits must be [..., vocab]")
    lead, vocab, rows = logits.shape[:-1], logits.shape[-1], _row_count(logits)
    _on(teacher, dev, "teacher_logits")
    _on(index, dev, "teacher_index")
    i_code = _IDS.get(index.dtype)
    if i_code is None:
        raise RuntimeError("teacher_index must be int32 or int64")
    if teacher.shape != index.shape or teacher.dim() < 1 or teacher.shape[:-1] != lead:
        raise RuntimeError("teacher_logits and teacher_index must be [*logits.shape[:-1], top]")
    if not (teacher.is_contiguous() and index.is_contiguous()):
        raise RuntimeError("teacher_logits and teacher_index must be contiguous")
    top = teacher.shape[-1]
    if not 1 <= top <= _lib.DISTILL_MAX_TOP:
        raise RuntimeError(f"top must lie in 1..{_lib.DISTILL_MAX_TOP}")
    if weight is not None:
        _on(weight, dev, "weight")
        if weight.dtype != torch.float32 or weight.shape != lead or not weight.is_contiguous():
            raise RuntimeError("weight must be contiguous float32 [*logits.shape[:-1]]")
    if not 0.0 < temperature < float("inf"):
        raise RuntimeError("temperature must be positive and finite")
    stride = _row_stride(logits, "logits")
    losses = total = None
    if want_loss:
        device = logits.device
        losses = _empty(lead, (1,), torch.float32, device) if len(lead) == 1 else \
            torch.empty(lead, dtype=torch.float32, device=device)
        total = _empty((), (), torch.float32, device)
    up_stride = 0
    if upstream is not None and upstream.dim() > 0:
        up_stride = 1
    _run(_entry("mdq_topk_distill"), dev, _DISTILL.pack(
        logits.data_ptr(), teacher.data_ptr(), index.data_ptr(), _ptr(weight), _ptr(upstream),
        _ptr(losses), _ptr(total), _ptr(grad), rows, vocab, stride,
        0 if grad is None else _row_stride(grad, "out"), up_stride, top, temperature, scale, code,
        t_code, i_code))
    return total, losses


def _entangled(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two [..., vocab] tensors of one shape and dtype share elements
    without being the same: a row of one would be written before another reads it."""
    rows, vocab, size = _row_count(a), a.shape[-1], a.element_size()
    if rows == 0:
        return False
    off = b.data_ptr() - a.data_ptr()
    sa, sb = ((_row_stride(t, what) if rows > 1 else 0) * size
              for t, what in ((a, "logits"), (b, "out")))
    if off >= (rows - 1) * sa + vocab * size or -off >= (rows - 1) * sb + vocab * size:
        return False
    if sa != sb:
        return True
    # the same distance between rows: side by side in one matrix, or the same rows
    return off != 0 and (rows == 1 or not vocab * size <= off % sa <= sa - vocab * size)


def topk_distill(logits: torch.Tensor, teacher_logits: torch.Tensor, teacher_index: torch.Tensor,
                 *, temperature: float = 1.0, weight: Optional[torch.Tensor] = None,
                 scale: float = 1.0, grad: bool = True,
                 out: Optional[torch.Tensor] = None) -> TopkDistill:
    """Distillation from a teacher's top logits: loss and, in the same pass over
    the logits, their gradient.

    For every row, with q = softmax(teacher_logits / temperature) over the row's
    entries and p = softmax(logits / temperature) over the vocabulary,

        loss_row = scale * weight * temperature^2 * sum_k q_k (log q_k - log p[index_k])

    and the total is their sum (pass scale = 1 / positions for a mean).  An entry
    with an index outside [0, vocab) (-1, say) is absent.  A row of weight 0, or
    without an entry above -infinity, has loss and gradient 0, whatever its logits
    hold.  top = 1 with temperature 1 is the cross-entropy against the index.

    ``out`` receives the gradient (logits' shape and dtype, evenly strided rows), to
    autograd an in-place operation on it; it may be ``logits``, which are then
    overwritten, but share nothing else with them.  Without ``grad`` only the loss is
    computed."""
    given = out is not None
    if given:
        if not grad:
            raise RuntimeError("out needs grad")
        _on(out, _device(logits, "logits"), "out")
        if out.shape != logits.shape or out.dtype != logits.dtype:
            raise RuntimeError("out must have logits' shape and dtype")
        if _row_count(out) > 1 and _row_stride(out, "out") < out.shape[-1]:
            raise RuntimeError("out's rows must not overlap")
        if _entangled(logits, out):
            raise RuntimeError("out must be logits itself or not overlap them")
    elif grad:
        _device(logits, "logits")
        out = _like(logits)
    total, losses = _distill(logits, teacher_logits, teacher_index, temperature, weight,
                             scale, out)
    if given:
        increment_version(out)   # backward passes that need its former values refuse
    return TopkDistill(total, losses, out)


class _TopkDistillLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, teacher, index, temperature, weight, scale, reduction):
        total, losses = _distill(logits, teacher, index, temperature, weight, scale, None)
        ctx.save_for_backward(logits, teacher, index, weight)
        ctx.args = (temperature, scale)
        return total if reduction == "sum" else losses

    @staticmethod
    @once_differentiable
    def backward(ctx, upstream):
        logits, teacher, index, weight = ctx.saved_tensors
        grad = _like(logits)
        _distill(logits, teacher, index, ctx.args[0], weight, ctx.args[1], grad,
                 upstream.float().contiguous(), want_loss=False)
        return grad, None, None, None, None, None, None


def topk_distill_loss(logits, teacher_logits, teacher_index, *, temperature: float = 1.0,
                      weight: Optional[torch.Tensor] = None, scale: float = 1.0,
                      reduction: str = "sum") -> torch.Tensor:
    """``topk_distill``'s loss as a differentiable function of ``logits``:
    the total (reduction "sum") or every row's ("none").  The backward pass reads
    the logits again and writes their gradient; ``topk_distill`` does both in one
    pass where the upstream gradient is known to be 1."""
    if reduction not in ("sum", "none"):
        raise RuntimeError("reduction must be 'sum' or 'none'")
    if logits.requires_grad and torch.is_grad_enabled():
        return _TopkDistillLoss.apply(logits, teacher_logits, teacher_index, temperature, weight,
                                      scale, reduction)
    total, losses = _distill(logits, teacher_logits, teacher_index, temperature, weight, scale,
                             None)
    return total if reduction == "sum" else losses


__all__ = ["scaled_embedding", "scaled_embedding_grad", "residual_norm", "residual_norm_forward",
           "residual_norm_backward", "ResidualNormGrads", "topk_distill", "topk_distill_loss",
           "TopkDistill"]
