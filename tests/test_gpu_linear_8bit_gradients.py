"""Some of the gradients of linear_8bit without the others: the same bits, and no memory for those that nobody asked for."""
import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16]


def _leaves(dev, rows, out, width, dtype):
    g = torch.Generator(dev).manual_seed(rows + out)
    new = lambda *s, scale=1.0: (torch.randn(*s, device=dev, generator=g) * scale).to(dtype)       # noqa: E731
    return (new(rows, width), new(out, width, scale=width ** -0.5), new(out)), new(rows, out, scale=1e-3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,out,width", [(1, 64, 8), (33, 70, 50), (70, 128, 300), (4112, 384, 384), (3000, 64, 64), (8192, 2048, 2048)])
def test_any_of_the_gradients(dev, dtype, rows, out, width):
    from vtpack_amd.layers import linear_8bit
    operands, dy = _leaves(dev, rows, out, width, dtype)
    whole = [t.clone().requires_grad_() for t in operands]
    want = torch.autograd.grad(linear_8bit(*whole), whole, dy)
    for asked in itertools.product((False, True), repeat=3):
        if not any(asked):
            continue
        leaves = [t.clone().requires_grad_(a) for t, a in zip(operands, asked)]
        got = torch.autograd.grad(linear_8bit(*leaves), [t for t in leaves if t.requires_grad], dy)
        for a, b in zip(got, (w for w, on in zip(want, asked) if on)):
            assert torch.equal(a, b), asked


def test_memory_of_a_backward_pass(dev):
    """Beside the result: the second operand in bf16 (and parts of dweight, 64 MB at most here), and no place for sums that are not cut."""
    from vtpack_amd.layers import linear_8bit
    rows, out, width = 32768, 512, 4096
    operands, dy = _leaves(dev, rows, out, width, torch.bfloat16)
    for k, second in ((0, out * width), (1, rows * width)):
        leaves = [t.clone().requires_grad_(i == k) for i, t in enumerate(operands)]
        y = linear_8bit(*leaves)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        grad, = torch.autograd.grad(y, leaves[k], dy)
        more = torch.cuda.max_memory_allocated() - before
        assert more <= grad.numel() * 2 + second * 2 + (64 << 20) * (k == 1) + (1 << 20), (k, more)
        del y, grad
