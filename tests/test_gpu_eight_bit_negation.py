"""Operands whose negation is still to be made (the imaginary part of a conjugate is such a view of the complex numbers' memory)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _negated(dev, *shape, seed=0):
    z = torch.randn(*shape, dtype=torch.complex64, generator=torch.Generator().manual_seed(seed)).to(dev)
    t = z.conj().imag
    assert t.is_neg()
    return t, t.clone()


def test_operands_with_a_negation_to_be_made(dev):
    from vtpack_amd.layers import gelu_8bit, layer_norm_8bit, linear_8bit, quantize_blocks
    for n in (1, 40):
        (x, x_), (w, w_), (b, b_), (v, v_) = (_negated(dev, *s, seed=k) for k, s in enumerate(((30, n), (1, n), (1,), (n,))))
        assert torch.equal(quantize_blocks(x).dequantize(), quantize_blocks(x_).dequantize())
        assert torch.equal(gelu_8bit(x), gelu_8bit(x_))
        assert torch.equal(layer_norm_8bit(x, v, v), layer_norm_8bit(x_, v_, v_))
        assert torch.equal(linear_8bit(x, w, b), linear_8bit(x_, w_, b_))
        assert torch.equal(linear_8bit(x, quantize_blocks(w), b), linear_8bit(x_, w_, b_))


def test_gradients_with_a_negation_to_be_made(dev):
    """As a function of complex numbers hands them back."""
    from vtpack_amd.layers import gelu_8bit, layer_norm_8bit, linear_8bit
    for n in (1, 40):
        dy, dy_ = _negated(dev, 30, n, seed=7)
        x, w, b, v = (torch.randn(*s, device=dev).requires_grad_() for s in ((30, n), (n, n), (n,), (n,)))
        for op, leaves in ((lambda: linear_8bit(x, w, b), (x, w, b)), (lambda: gelu_8bit(x), (x,)), (lambda: layer_norm_8bit(x, v, b, 0.5), (x, v, b))):
            for got, want in zip(torch.autograd.grad(op(), leaves, dy), torch.autograd.grad(op(), leaves, dy_)):
                assert torch.equal(got, want)
        # the weight of a norm, kept for its gradients
        u, u_ = _negated(dev, n, seed=9)
        got, want = (torch.autograd.grad(layer_norm_8bit(x, t, b, 0.5), x, dy_)[0] for t in (u, u_))
        assert torch.equal(got, want)
