"""GELU of the 8-bit operators over the whole range of its type, against the formula in 64 bits: what is far out on the negative side is
small, and zero where it is no number of the type.

Bounds, relative to the value.  A result in bf16 is rounded once, 2^-8 at most.  bf16: what stands for Phi is 7.2e-5 off up to
4, 2.9e-4 up to 10 (2^-13 and 2^-11 with the rounding of its argument), a quarter behind that, where the value is below 8e-23.  fp32: 4e-7 for the fit, the reciprocal, the exponential and the products, and the exponent 0.72 x^2, rounded
three times, 2^-23 x^2.  An exponential that is no normal number is zero: 14 2^-126, where |x| <= 14."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16]
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
NONE = 14 * 2.0 ** -126


def phi(x):
    return 0.5 * torch.erfc(-x * math.sqrt(0.5))        # (torch.special.ndtr has nothing left below -8.3)


def gelu(x):
    return x * phi(x)


def _all_of_bf16():
    return torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)


def _is_gelu(got, x64):
    dtype = got.dtype
    got, want = got.detach().cpu().double(), gelu(x64)
    assert torch.equal(got.isnan(), want.isnan())
    there = torch.isfinite(want)
    assert torch.equal(got[~there & ~want.isnan()], want[~there & ~want.isnan()])
    got, want, x64 = got[there], want[there], x64[there]
    if dtype == torch.bfloat16:
        off = torch.full_like(x64, 2.0 ** -13)
        off[x64 < -4], off[x64 < -10] = 2.0 ** -11, 0.26
    else:
        off = 4e-7 + 2.0 ** -23 * x64.clamp(-14, 0) ** 2
    over = (got - want).abs() - 1.01 * (off + HALF[dtype]) * want.abs() - NONE
    assert float(over.max()) <= 0, (float(x64[over.argmax()]), float(got[over.argmax()]), float(want[over.argmax()]))


@pytest.mark.parametrize("dtype", DTYPES)
def test_gelu_of_every_number(dev, dtype):
    from vtpack_amd.layers import gelu_8bit
    x = _all_of_bf16().to(dtype)
    y = gelu_8bit(x.to(dev).view(512, 128)).view(-1)
    _is_gelu(y, x.double())
    far = torch.tensor([-1e30, -1000.0, -100.0, -30.0], dtype=dtype).to(dev)
    assert not gelu_8bit(far).any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 40])
def test_gelu_of_every_bias(dev, dtype, rows):
    """act="gelu" of the Linear, in few rows and by tiles: sums of zeros and a bias of every number."""
    from vtpack_amd.layers import linear_8bit
    bias = _all_of_bf16().to(dtype)
    x, w = torch.zeros(rows, 8, dtype=dtype, device=dev), torch.ones(bias.numel(), 8, dtype=dtype, device=dev)
    y = linear_8bit(x, w, bias.to(dev), act="gelu")
    for r in (0, rows - 1):
        _is_gelu(y[r], bias.double())


def _numbers_of_four_bits():
    """Both signs of 8 to 15 times 2^k: a block of its own holds each as it is."""
    m = torch.arange(8, 16, dtype=torch.float64)
    c = torch.cat([m * 2.0 ** k for k in range(-100, 117)])
    return torch.cat([c, -c, torch.zeros(1, dtype=torch.float64)])


@pytest.mark.parametrize("dtype", DTYPES)
def test_slope_of_every_number_of_four_bits(dev, dtype):
    """dx = dy (Phi(c) + c phi(c)): nothing far out on the negative side, dy on the positive one.

    bf16: 3.8e-5 (|S| + 0.05 e), S the slope of -|c| and e = exp(-c^2 / 2), is 2^-14 |S| + 2e-6 e; |S| <= |d|, or <= 1/2 <= d on the positive side;
    twice as much with the roundings of the terms, whose size is |c| e.  fp32: the terms are (|c| + 1) e, off by 4e-7 and 2^-23 c^2 as Phi is;
    the result's own rounding, and 1 - S, are half a step each."""
    from vtpack_amd.layers import gelu_8bit, quantize_blocks
    c = _numbers_of_four_bits()
    x = c.to(dtype).to(dev).view(-1, 1)
    assert torch.equal(quantize_blocks(x).dequantize(), x.float())
    x.requires_grad_()
    e = torch.exp(-c * c / 2)
    d = phi(c) + c * e * (0.5 / math.pi) ** 0.5
    for g in (1.0, -1.1484375):
        dx, = torch.autograd.grad(gelu_8bit(x), x, torch.full_like(x, g))
        got, want = dx.view(-1).cpu().double(), g * d
        if dtype == torch.bfloat16:
            off = 2.0 ** -13 * d.abs() + 4e-6 * e
        else:
            off = (4e-7 + 2.0 ** -23 * c.clamp(-14, 14) ** 2) * (c.abs() + 1) * e + 2.0 ** -24 * (c >= 0)
        over = (got - want).abs() - 1.01 * (off * abs(g) + HALF[dtype] * want.abs() + NONE * 14)
        assert float(over.max()) <= 0, (float(c[over.argmax()]), float(got[over.argmax()]), float(want[over.argmax()]))
        assert not got[c <= -16].any() and torch.equal(got[c >= 16], torch.full_like(got[c >= 16], g))
