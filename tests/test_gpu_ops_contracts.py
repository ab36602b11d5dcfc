"""What callers of the training-step operators rely on beside the values: calls
without rows through the C ABI.
"""
import ctypes

import pytest
import torch

from mdq_b200 import _lib

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
