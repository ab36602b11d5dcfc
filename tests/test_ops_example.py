"""The example that trains on all operators together."""
import importlib.util
import math
import subprocess
import sys
from pathlib import Path

import pytest
import torch

PATH = Path(__file__).resolve().parents[1] / "stream-mm2026_b200" / "examples" / "distill_lm.py"


def _example():
    spec = importlib.util.spec_from_file_location("distill_lm", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_example_describes_itself():
    said = subprocess.run([sys.executable, str(PATH), "--help"], capture_output=True, text=True)
    assert said.returncode == 0 and "--temperature" in said.stdout


@pytest.mark.gpu
def test_example_learns(cuda_device):
    losses = _example().train(steps=150, every=0)
    assert all(math.isfinite(v) for v in losses)
    # A teacher of 16 entries at random places among 512: the untrained model's
    # divergence is T^2 log(512 / 16) at least; a bigram table is learnt to well below half.
    assert sum(losses[-10:]) < 0.5 * sum(losses[:10])


@pytest.mark.gpu
def test_example_trains_one_layer(cuda_device):
    losses = _example().train(steps=2, vocab=32, dim=32, layers=1, heads=2, batch=3, length=16, top=4, every=0)
    assert len(losses) == 2 and all(math.isfinite(v) for v in losses)


@pytest.mark.gpu
@pytest.mark.parametrize("length", [1, 7, 9, 60, 64])
def test_example_weights_add_up_to_one(cuda_device, length, monkeypatch):
    """The loss is a mean: the weights of the positions that count, times the scale, sum to 1."""
    m, seen = _example(), []

    def look(*args, weight, scale, **kw):
        seen.append(float(weight.sum()) * scale)
        return distill(*args, weight=weight, scale=scale, **kw)

    distill = m.ops.topk_distill
    monkeypatch.setattr(m.ops, "topk_distill", look)
    losses = m.train(steps=1, vocab=32, dim=32, layers=1, heads=2, batch=3, length=length, top=4, every=0)
    assert math.isfinite(losses[0]) and seen == [pytest.approx(1.0, rel=1e-6)]


@pytest.mark.gpu
def test_example_gradients(cuda_device):
    """The model's gradients on the operators against the same model on plain
    fp32 torch operations (bf16 products in both)."""
    m = _example()
    torch.manual_seed(3)
    model = m.SmallLM(64, 32, 2, 2).to(cuda_device)
    teacher = m.Teacher(64, 5, cuda_device)
    ids = torch.randint(0, 64, (3, 9), device=cuda_device)
    t, at = teacher(ids)

    def norm(v, w):
        v = v.float()
        return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-5) * w

    def plain():
        x = model.table[ids] * math.sqrt(32)
        n = norm(x, model.pre[0])
        with torch.autocast("cuda", torch.bfloat16):
            for k, block in enumerate(model.blocks):
                h = block(n)
                x = x + model.gate[k] * norm(h, model.post[k])
                n = norm(x, model.pre[k + 1]).to(h.dtype)
            return n @ model.table.t()

    logits = plain()
    z, q = logits.float() / 1.5, torch.softmax(t / 1.5, -1)
    log_p = torch.log_softmax(z, -1).gather(-1, at)
    (1.5 ** 2 * (q * (q.log() - log_p)).sum()).backward()
    want = [p.grad.clone() for p in model.parameters()]
    model.zero_grad()
    logits = model(ids)
    logits.backward(m.ops.topk_distill(logits.detach(), t, at, temperature=1.5).grad)
    for p, w in zip(model.parameters(), want):
        # bf16 activations round differently in a few places: 2^-8 each, a dozen in a row
        assert float((p.grad - w).norm()) <= 12 * 2 ** -8 * float(w.norm())
