"""What callers of the training-step operators rely on beside the values: calls
without rows through the C ABI, results written into a caller's tensor,
which autograd has to learn of, and forward-mode tangents.
"""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from mdq_b200 import _lib, ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("groups", [1, 3, 300])
@pytest.mark.parametrize("kind", [_lib.NORM_RMS, _lib.NORM_LAYER])
@pytest.mark.parametrize("dim", [64, 1601, 9000])
def test_residual_norm_grad_without_rows(cuda_device, groups, kind, dim):
    """No rows: every parameter's gradient is zero, the gate's of all groups too,
    whatever the workspace held."""
    lib = _lib.load()
    need = ctypes.c_int64(0)
    assert lib.mdq_residual_norm_grad_workspace_bytes(0, dim, groups, ctypes.byref(need)) == 0

    def filled(*shape):
        return torch.full(shape, float("nan"), device=cuda_device)

    workspace, w, gate = filled(need.value // 4 + 1), filled(dim), filled(groups, dim)
    grads = {k: filled(dim) for k in ("post_weight", "post_bias", "pre_weight", "pre_bias")}
    grads["gate"] = filled(groups, dim)
    p = w.data_ptr()
    f = _lib.ResidualNormDesc(x=p, h=p, stats=p, post_weight=p, post_bias=p, pre_weight=p,
                              pre_bias=p, gate=gate.data_ptr(), rows=0, dim=dim, x_stride=dim,
                              h_stride=dim, gate_rows=groups, residual_scale=1.0, eps=1e-5,
                              kind=kind)
    g = _lib.ResidualNormGradDesc(f=f, grad_new=p, grad_n=p, grad_x=p, grad_h=p,
                                  workspace=workspace.data_ptr(), workspace_bytes=need.value,
                                  grad_new_stride=dim, grad_n_stride=dim,
                                  **{f"grad_{k}": t.data_ptr() for k, t in grads.items()})
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.mdq_residual_norm_grad(ctypes.byref(g), stream) == 0
    for k, t in grads.items():
        assert bool((t == 0).all()), k


def _distill_into(out, dev):
    rows = out.shape[0]
    return ops.topk_distill(out, torch.zeros(rows, 2, device=dev),
                            torch.zeros(rows, 2, dtype=torch.int64, device=dev), out=out).grad


def _sums_into(accumulate):
    def write(out, dev):
        ids = torch.arange(out.shape[0], device=dev)
        return ops.scaled_embedding_grad(ids, torch.ones_like(out), out.shape[0], out=out,
                                         accumulate=accumulate)
    return write


@pytest.mark.parametrize("write", [_distill_into, _sums_into(False), _sums_into(True)],
                         ids=["distill", "embedding", "embedding added"])
def test_results_in_a_callers_tensor_raise_its_version(cuda_device, write):
    """As an in-place operation of torch: a backward pass that needs the values
    that were overwritten refuses."""
    leaf = torch.randn(6, 40, device=cuda_device, requires_grad=True)
    saved = torch.exp(leaf)            # its backward pass reads the result
    out = saved.detach()
    version = out._version
    assert write(out, cuda_device) is out
    assert out._version == version + 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        saved.sum().backward()
    # the logits that the loss's own backward pass reads
    logits = torch.randn(6, 40, device=cuda_device, requires_grad=True)
    loss = ops.topk_distill_loss(logits, torch.zeros(6, 1, device=cuda_device),
                                 torch.zeros(6, 1, dtype=torch.int64, device=cuda_device))
    write(logits.detach(), cuda_device)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    # a refused call has written nothing; inference tensors have no version
    version = out._version
    with pytest.raises(RuntimeError, match="temperature"):
        ops.topk_distill(out, out[:, :2].contiguous(),
                         torch.zeros(6, 2, dtype=torch.int64, device=cuda_device),
                         temperature=0.0, out=out)
    assert out._version == version
    with torch.inference_mode():
        assert bool(torch.isfinite(write(torch.randn(6, 40, device=cuda_device), cuda_device)).all())


def _calls_with(dev):
    """Every front end, as a function of one of its floating-point arguments."""
    x, h = torch.randn(6, 40, device=dev), torch.randn(6, 40, device=dev)
    w, ids = torch.ones(40, device=dev), torch.arange(6, device=dev)
    t, at = torch.zeros(6, 2, device=dev), torch.zeros(6, 2, dtype=torch.int64, device=dev)
    weight = torch.ones(6, device=dev)
    stats = ops.residual_norm_forward(x, h, w, w)[2]
    return {
        "embedding": (x, lambda v: ops.scaled_embedding(ids, v)),
        "embedding grad": (x, lambda v: ops.scaled_embedding_grad(ids, v, 6)),
        "embedding grad out": (x, lambda v: ops.scaled_embedding_grad(ids, x, 6, out=v)),
        "norm x": (x, lambda v: ops.residual_norm(v, h, w, w)),
        "norm h": (x, lambda v: ops.residual_norm(x, v, w, w)),
        "norm first": (x, lambda v: ops.residual_norm(v, None, None, w)),
        "norm weight": (w, lambda v: ops.residual_norm(x, h, v, w)),
        "norm bias": (w, lambda v: ops.residual_norm(x, h, w, w, pre_bias=v)),
        "norm gate": (w, lambda v: ops.residual_norm_forward(x, h, w, w, gate=v)),
        "norm backward": (x, lambda v: ops.residual_norm_backward(v, x, x, h, stats, w, w)),
        "norm backward stats": (stats, lambda v: ops.residual_norm_backward(x, x, x, h, v, w, w)),
        "distill": (x, lambda v: ops.topk_distill(v, t, at)),
        "distill teacher": (t, lambda v: ops.topk_distill_loss(x, v, at)),
        "distill weight": (weight, lambda v: ops.topk_distill(x, t, at, weight=v)),
        "distill out": (x, lambda v: ops.topk_distill(x, t, at, out=v)),
        "distill loss": (x, lambda v: ops.topk_distill_loss(v, t, at)),
    }


def test_forward_mode_tangents_are_refused(cuda_device):
    """No operator has a forward-mode derivative: a dual tensor is refused, with or
    without reverse mode, and not taken for its primal."""
    for name, (value, call) in _calls_with(cuda_device).items():
        call(value.clone())
        with forward_ad.dual_level():
            call(value.clone())                   # no tangent: as ever
            for grad in (False, True):
                dual = forward_ad.make_dual(value.clone().requires_grad_(grad),
                                            torch.ones_like(value))
                with pytest.raises(RuntimeError, match="forward"):
                    call(dual)
                    pytest.fail(name)
                with torch.no_grad(), pytest.raises(RuntimeError, match="forward"):
                    call(dual)
                    pytest.fail(name)
    # and under torch.func, whose tensors have no memory of their own
    x, w = torch.randn(6, 40, device=cuda_device), torch.ones(40, device=cuda_device)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda v: ops.residual_norm(v, None, None, w)[1], (x,), (x,))
