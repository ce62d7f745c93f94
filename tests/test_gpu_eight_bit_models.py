"""A model's training pass on 8-bit blocks, call by call: each Linear, LayerNorm and GELU of each block against its formula in 64 bits, on
the input and the gradient that it had in the pass.  Bounds as in test_gpu_eight_bit; gradients of a module that is called twice add up."""
import math

import pytest
import torch
from torch import nn

from tests import eight_bit_reference as ref
from tests.test_gpu_eight_bit import HALF, WALK, _deit, _pvt, _within

pytestmark = pytest.mark.gpu
F32 = HALF[torch.float32]


def _sum(n):
    return WALK * (8 + 2 * math.sqrt(n))


def _linear(m, x, y, dx, dy):
    w8, x8, g = ref.q(m.weight), ref.q(x), dy.to(torch.bfloat16).cpu().double()
    b = torch.zeros(w8.shape[0], dtype=torch.float64) if m.bias is None else m.bias.detach().cpu().double()
    want = x8 @ w8.t() + b
    _within(y, want, 1.01 * (_sum(x8.shape[1]) * (x8.abs() @ w8.abs().t()) + 2 * WALK * b.abs() + F32 * want.abs()), "y")
    want = g @ w8
    _within(dx, want, 1.01 * (_sum(g.shape[1]) * (g.abs() @ w8.abs()) + F32 * want.abs()) + 1e-38, "dx")
    return [(m.weight, g.t() @ x8, _sum(g.shape[0]) * (g.abs().t() @ x8.abs()))] + ([] if m.bias is None else [(m.bias, g.sum(0), _sum(g.shape[0]) * g.abs().sum(0))])


def _gelu(m, x, y, dx, dy):
    x64, g = x.cpu().double(), dy.cpu().double()
    slope = ref.gelu_slope(ref.q(x))
    _within(y, ref.gelu(x64), 1.01 * (4e-7 * x64.abs() + F32 * ref.gelu(x64).abs()) + 1e-38, "y")
    _within(dx, g * slope, 1.01 * (4e-7 * g.abs() + F32 * (g * slope).abs()) + 1e-38, "dx")
    return []


def _layer_norm(m, x, y, dx, dy):
    n, rows = x.shape[1], x.shape[0]
    want, grads = ref.layer_norm(x, m.weight, m.bias, m.eps, dy)
    _within(y, want, 1.01 * (16 * WALK * (1 + want.abs() + m.bias.detach().cpu().double().abs()) + F32 * want.abs()), "y")
    x64, w64, g64 = x.cpu().double(), m.weight.detach().cpu().double(), dy.cpu().double()
    c = x64 - x64.mean(1, keepdim=True)
    r = 1 / torch.sqrt((c * c).mean(1, keepdim=True) + m.eps)
    h, gw = (ref.q(x.cpu() - x64.mean(1, keepdim=True).float()) * r).abs(), (g64 * w64).abs()
    size = r * (gw + gw.mean(1, keepdim=True) + h * (gw * h).mean(1, keepdim=True))
    _within(dx, grads[0], 1.01 * (WALK * (16 + 2 * math.sqrt(n)) * size + F32 * grads[0].abs()) + 1e-38, "dx")
    return [(m.weight, grads[1], WALK * (16 + 2 * math.sqrt(rows)) * (g64.abs() * h).sum(0)), (m.bias, grads[2], _sum(rows) * g64.abs().sum(0))]


CHECKS = {nn.Linear: _linear, nn.GELU: _gelu, nn.LayerNorm: _layer_norm}


@pytest.mark.parametrize("make,size,count", [(_deit, 64, 2 * 9), (_pvt, 128, 4 * 9 + 3)])
def test_every_call_of_a_training_pass(dev, monkeypatch, make, size, count):
    from vtpack_amd.layers.eight_bit import call_8bit
    from vtpack_amd.models.dge import deit_dge, pvt_dge
    from vtpack_amd.synthetic import synthetic_images
    calls = []

    def seen(module, x):
        x = x.view_as(x)                                 # a place of its own for this call's gradient
        x.retain_grad()
        y = call_8bit(module, x)
        y.retain_grad()
        calls.append((module, x, y))
        return y

    for models in (deit_dge, pvt_dge):
        monkeypatch.setattr(models, "call_8bit", seen)
    m = make(dev).set_eight_bit()
    images, target = synthetic_images(4, size, seed=1).to(dev), torch.tensor([1, 0, 3, 2], device=dev)
    torch.manual_seed(5)                                 # the gates are sampled
    m(images, target).backward()
    assert len(calls) == count
    flat = lambda t: t.detach().reshape(-1, t.shape[-1])                                            # noqa: E731
    sums = {}
    for module, x, y in calls:
        for p, want, bound in CHECKS[type(module)](module, flat(x), flat(y), flat(x.grad), flat(y.grad)):
            so_far = sums.setdefault(p, (torch.zeros_like(want), torch.zeros_like(want), torch.zeros_like(want)))
            # (each call's gradient is rounded, and so is the sum of two)
            sums[p] = so_far[0] + want, so_far[1] + bound + F32 * want.abs(), so_far[2] + want.abs()
    names = {p: n for n, p in m.named_parameters()}
    for p, (want, bound, parts) in sums.items():
        _within(p.grad, want, 1.01 * (bound + F32 * parts) + 1e-38, names[p])
    blocks = [b for b in m.modules() if type(b).__name__ == "Block"]
    inside = {p for b in blocks for part in (b.norm1, b.norm2, b.mlp, b.attn.q, b.attn.kv, b.attn.proj) for p in part.parameters()}
    assert inside <= set(sums)
