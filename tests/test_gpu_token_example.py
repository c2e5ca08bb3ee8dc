"""The token-classifier example: its gradients against torch's differentiation
of the same model in 64 bits (the activation's slope taken where the 8-bit
tape has it), and a few steps of training."""
import importlib.util
import math
import os

import pytest
import torch

import token_ref as R

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _example():
    spec = importlib.util.spec_from_file_location(
        "token_experts", os.path.join(ROOT, "examples", "token_experts.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


class _TapedGelu(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, tape):
        ctx.save_for_backward(torch.from_numpy(R.act_slope("gelu", tape.numpy())))
        return 0.5 * x * (1 + torch.erf(x / math.sqrt(2)))

    @staticmethod
    def backward(ctx, g):
        return g * ctx.saved_tensors[0], None


def _reference(model, ids, target, eps):
    """Loss and gradients in Float64 on the CPU; the tape's values come from the
    run under test, whose hidden layer they belong to."""
    n_s, n_v, n_d, n_e, n_f, n_h, n_o = model.size
    p = {k: v.detach().cpu().double().requires_grad_() for k, v in model.p.items()}
    ids = ids.cpu()
    order = torch.argsort(ids % n_e, stable=True)
    tape = torch.empty(n_s, n_f, dtype=torch.float64)
    tape[order] = torch.from_numpy(R.tape8_values(model.q.cpu().numpy().reshape(n_s, n_f),
                                                  model.e.cpu().numpy().reshape(n_s, -1)))

    def norm(x, w, b):
        d = x - x.mean(1, keepdim=True)
        return d / torch.sqrt((d * d).mean(1, keepdim=True) + eps) * w + b

    emb = p["table"][ids] * math.sqrt(n_d)
    x = norm(emb, p["norm_w"], p["norm_b"])
    up = torch.einsum("sd,sdf->sf", x, p["up"][ids % n_e])
    y = torch.einsum("sf,sfd->sd", _TapedGelu.apply(up, tape), p["down"][ids % n_e])
    out = norm(emb + y, p["out_w"], p["out_b"])
    z = torch.tanh(out @ p["w1"] + p["b1"]) @ p["w2"] + p["b2"]
    loss = -(torch.log_softmax(z, 1) * target.cpu()).sum() / n_s
    loss.backward()
    return loss.item(), {k: v.grad for k, v in p.items()}


@pytest.mark.parametrize("sizes", [(200, 60, 64, 4, 96, 32, 10), (333, 1000, 40, 5, 72, 24, 7)])
def test_gradients_in_float32(sizes):
    m = _example()
    model = m.TokenExperts(*sizes, dtype=torch.float32)
    g = torch.Generator().manual_seed(3)
    ids = torch.randint(0, sizes[1], (sizes[0],), generator=g)
    target = torch.nn.functional.one_hot(torch.randint(0, sizes[6], (sizes[0],), generator=g), sizes[6])
    loss = model.gradient(ids.cuda(), target.cuda()).item()
    ref, grads = _reference(model, ids, target, m.EPS)
    # a chain of some ten operators, each within a few 1e-6 of its own scale
    assert abs(loss - ref) < 1e-4 * abs(ref)
    for k, v in grads.items():
        err = (model.g[k].cpu().double() - v).norm() / v.norm()
        assert err < 1e-4, f"{k}: {err:.2e}"


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
def test_training_lowers_the_loss(dt):
    m = _example()
    model = m.TokenExperts(512, 200, 64, 4, 128, 32, 10, dtype=dt)
    g = torch.Generator(device="cuda").manual_seed(1)
    labels = torch.randint(0, 10, (200,), generator=g, device="cuda")
    losses = []
    for _ in range(60):
        ids = torch.randint(0, 200, (512,), generator=g, device="cuda")
        target = torch.nn.functional.one_hot(labels[ids], 10)
        losses.append(model.step(ids, target, 1.0).item())
    assert all(math.isfinite(v) for v in losses)
    assert losses[-1] < 0.5 * losses[0]
