"""Blocks of 8-bit numbers and the operators on them against their definitions in float64 on the CPU.

Bounds.  Blocks: none, bytes are equal.  Sums: every fp32 step is off by half a step of a partial sum, which is sum |p| at most; their
errors walk: 2^-24 (8 + 2 sqrt(n)) sum |p| for n terms.  A result in bf16 is rounded once, 2^-8 of it at most.  In bf16 the Linear's
forward product runs on the 8-bit matrix instructions, which cut the products of a group off below the largest one's 13th bit: 2^-12
sum |p|.  GELU in bf16 is a polynomial, 1.4e-4 of |x| away from the formula at most."""
import math

import pytest
import torch

from tests import eight_bit_reference as ref

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16]
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
WALK = 2.0 ** -24


def _numbers(dev, *shape, dtype=torch.float32, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed * 7919 + sum(shape))
    x = torch.randn(*shape, generator=g) * torch.exp(0.6 * torch.randn(shape[-1], generator=g)) + 0.3 * torch.randn(shape[-1], generator=g)
    return (x * scale).to(dev, dtype)


def _within(got, want, bound, what=""):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, what
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    fine = ~torch.isnan(want)
    over = ((got - want).abs() / (bound + 1e-300))[fine]
    assert over.numel() == 0 or float(over.max()) <= 1, f"{what}: {float(over.max())} of what it may be off"


# ------------------------------------------------------------------------------------------------ blocks
def _same_blocks(blocks, x):
    numbers, e = ref.blocks_of(x)
    assert blocks.values.dtype == torch.float8_e4m3fn and blocks.values.shape == x.shape
    assert torch.equal(blocks.scales.view(torch.uint8).cpu().double() - 127, e)
    per_value = e.repeat_interleave(128, -1)[..., :x.shape[-1]]
    assert torch.equal((blocks.values.cpu().double() * torch.exp2(per_value)).nan_to_num(nan=-1.5), numbers.nan_to_num(nan=-1.5))
    for dtype in DTYPES:
        back = blocks.dequantize(dtype)
        assert back.dtype == dtype and back.is_contiguous()
        assert torch.equal(back.cpu().double().nan_to_num(nan=-1.5), numbers.nan_to_num(nan=-1.5))
    # what fills the rows up
    n, data = x.shape[-1], blocks._data
    rows, pitch = x.numel() // n, -(-n // 128) * 128
    assert not data[:rows * pitch].view(rows, pitch)[:, n:].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (1, 7), (3, 8), (5, 127), (2, 128), (7, 129), (1, 4096), (33, 384), (4, 5, 200), (2057, 192), (17, 1000), (9, 513), (6,)])
def test_blocks(dev, dtype, shape):
    from vtpack_amd.layers import quantize_blocks
    x = _numbers(dev, *shape, dtype=dtype)
    _same_blocks(quantize_blocks(x), x)


@pytest.mark.parametrize("dtype", DTYPES)
def test_blocks_of_rows_that_lie_anyhow(dev, dtype):
    from vtpack_amd.layers import quantize_blocks
    base = _numbers(dev, 40, 301, dtype=dtype)
    for x in (base[:, :256], base[:, 1:257], base[3::2, 5:], base.t(), base[:1, 7:], base[:, :1], base[5], base[:, None, :160].expand(40, 3, 160),
              base[:, ::2]):
        _same_blocks(quantize_blocks(x), x)


@pytest.mark.parametrize("dtype", DTYPES)
def test_blocks_at_the_borders(dev, dtype):
    """Zeros, the least scale, the largest numbers, ties, maxima beside 448, infinities and NaN."""
    from vtpack_amd.layers import quantize_blocks
    most = torch.finfo(dtype).max
    x = torch.zeros(24, 256)
    x[1, 3] = 1e-45
    x[2] = 2.0 ** -119
    x[3, :4] = torch.tensor([2.0 ** -120, 2.0 ** -121, -(2.0 ** -119) * 1.5, 2.0 ** -126])
    x[4, 0], x[4, 1], x[4, 2] = most, -most / 3, 1e30
    x[5, 0], x[5, 200] = 2.0 ** 127, 1.75 * 2.0 ** 127
    for row, top in enumerate((448.0, 448.0 * (1 + torch.finfo(dtype).eps), 448.0 * (1 - torch.finfo(dtype).eps), 1.75 * 2.0 ** 100, 447.0, 449.0), 6):
        x[row, 77], x[row, 200] = top, -top
    # ties between neighbours, normal and not, both ways
    steps = torch.tensor([256.0 + 16, 288 + 16, 1 + 1 / 16, 1 + 3 / 16, 2.0 ** -6 + 2.0 ** -10, 2.0 ** -10, 3 * 2.0 ** -10, 2.0 ** -9 * 7.5])
    x[12, :8], x[12, 8:16], x[12, 16] = steps, -steps, 448.0
    x[13, 0], x[13, 1], x[13, 2] = float("inf"), 1.0, float("-inf")
    x[14] = float("nan")
    x[15, 130], x[15, 0] = float("nan"), 5.0
    x[16] = float("inf")
    x[17, 64] = -0.0
    x[18, 0], x[18, 1] = float("inf"), most
    x = x.to(dtype)
    _same_blocks(quantize_blocks(x.to(dev)), x)


def test_blocks_from_a_pair(dev):
    """A copy, whatever the pair's strides; scales that quantize_blocks never makes."""
    from vtpack_amd.layers import Blocks, linear_8bit, quantize_blocks
    x = _numbers(dev, 6, 5, 300)
    a = quantize_blocks(x)
    b = Blocks(a.values, a.scales)
    assert torch.equal(a._data, b._data) and a._data.data_ptr() != b._data.data_ptr() and b.shape == x.shape
    wide = torch.empty(6, 5, 600, dtype=torch.uint8, device=dev)[..., ::2].copy_(a.values.view(torch.uint8)).view(6, 5, 300)
    values = torch.empty(30, 301, dtype=torch.float8_e4m3fn, device=dev)[:, 1:]
    values.view(torch.uint8).copy_(wide.reshape(30, 300))
    c = Blocks(values, a.scales.reshape(30, 3))
    assert torch.equal(c._data, a._data)
    scales = torch.tensor([[0], [1], [254], [255], [127]], dtype=torch.uint8, device=dev).view(torch.float8_e8m0fnu)
    ones = torch.ones(5, 3, device=dev).to(torch.float8_e4m3fn)
    odd = Blocks(ones, scales).dequantize()
    assert torch.equal(odd[[0, 1, 2, 4], 0].cpu().double(), torch.tensor([2.0 ** -127, 2.0 ** -126, 2.0 ** 127, 1.0], dtype=torch.float64))
    assert torch.isnan(odd[3]).all()
    y = linear_8bit(torch.ones(2, 3, device=dev), Blocks(ones, scales))
    assert torch.isnan(y[:, 3]).all() and torch.equal(y[:, 4].cpu(), torch.full((2,), 3.0))
    assert quantize_blocks(x[:0]).dequantize().shape == (0, 5, 300)


def test_blocks_from_a_pair_without_rows(dev):
    from vtpack_amd.layers import Blocks, quantize_blocks
    a = quantize_blocks(_numbers(dev, 0, 5, 300))
    b = Blocks(a.values, a.scales)
    assert b.shape == (0, 5, 300) and b._data.numel() == 0 and b.dequantize().shape == (0, 5, 300)


# ------------------------------------------------------------------------------------------------ Linear
def _linear_bound(x8, w8, b, y, dtype, act="none"):
    sums = x8.abs() @ w8.abs().t()
    bound = (WALK * (8 + 2 * math.sqrt(x8.shape[1])) + (2.0 ** -12 if dtype == torch.bfloat16 else 0.0)) * sums
    if b is not None:
        bound = bound + WALK * 2 * b.abs()
    if act == "gelu":
        bound = 1.13 * bound + (1.4e-4 if dtype == torch.bfloat16 else 2e-7) * y.abs()
        y = ref.gelu(y)
    return bound * 1.01 + HALF[dtype] * (y.abs() + bound) + 1e-38, y


def _operands(dev, rows, out, width, dtype, bias=True, seed=0):
    x = _numbers(dev, rows, width, dtype=dtype, seed=seed)
    w = _numbers(dev, out, width, dtype=dtype, seed=seed + 1, scale=0.7 / math.sqrt(width))
    return x, w, _numbers(dev, out, dtype=dtype, seed=seed + 2) if bias else None


SIZES = [(1, 1, 1), (1, 5, 8), (2, 130, 127), (3, 64, 128), (17, 33, 129), (1, 1000, 384), (16, 257, 640), (31, 2049, 192), (64, 64, 64), (65, 129, 1027),
         (255, 384, 384), (300, 257, 200), (1021, 768, 192), (2057, 1536, 384), (513, 4100, 72), (5, 300, 4200)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,out,width", SIZES)
def test_linear(dev, dtype, rows, out, width):
    from vtpack_amd.layers import linear_8bit, quantize_blocks
    x, w, b = _operands(dev, rows, out, width, dtype)
    x8, w8, b64 = ref.q(x), ref.q(w), b.cpu().double()
    for bias, act in ((b, "none"), (None, "gelu"), (b, "gelu")):
        y = x8 @ w8.t() + (0 if bias is None else b64)
        bound, want = _linear_bound(x8, w8, None if bias is None else b64, y, dtype, act)
        got = linear_8bit(x, w, bias, act=act)
        assert got.dtype == dtype
        _within(got, want, bound, act)
        assert torch.equal(linear_8bit(x, quantize_blocks(w), bias, act=act), got)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,out,width", SIZES)
@pytest.mark.parametrize("bias", [True, False])
def test_linear_gradients(dev, dtype, rows, out, width, bias):
    from vtpack_amd.layers import linear_8bit
    x, w, b = _operands(dev, rows, out, width, dtype, bias, seed=3)
    dy = _numbers(dev, rows, out, dtype=dtype, seed=7, scale=1e-3)
    leaves = [None if t is None else t.requires_grad_() for t in (x, w, b)]
    y = linear_8bit(*leaves)
    x8, w8, g = ref.q(x), ref.q(w), dy.to(torch.bfloat16).cpu().double()
    bound, want = _linear_bound(x8, w8, None if b is None else b.detach().cpu().double(), x8 @ w8.t() + (0 if b is None else b.detach().cpu().double()), dtype)
    _within(y, want, bound, "y")
    grads = torch.autograd.grad(y, [t for t in leaves if t is not None], dy)
    wants = [(g @ w8, g.abs() @ w8.abs(), out), (g.t() @ x8, g.abs().t() @ x8.abs(), rows), (g.sum(0), g.abs().sum(0), rows)]
    for name, got, (want, sums, n) in zip("xwb", grads, wants):
        assert got.dtype == dtype and got.is_contiguous()
        _within(got, want, WALK * (8 + 2 * math.sqrt(n)) * sums * 1.01 + HALF[dtype] * want.abs() * 1.01 + 1e-38, name)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,out,width", [(4099, 2049, 200), (8200, 4100, 700), (2999, 1301, 777)])
def test_linear_by_large_tiles(dev, dtype, rows, out, width):
    """Ragged ones of 128 x 128 and 256 x 256."""
    test_linear(dev, dtype, rows, out, width)
    test_linear_gradients(dev, dtype, rows, out, width, True)


@pytest.mark.parametrize("out", [1000, 1024])
def test_offsets_beyond_32_bits(dev, out):
    """Operands of more than 2^31 numbers: whole numbers, whose sums are exact, and rows, each of which is its own."""
    from vtpack_amd.layers import gelu_8bit, layer_norm_8bit, linear_8bit, quantize_blocks
    rows, width, tail = (1 << 21) + 333, 1024, 200
    g = torch.Generator(dev).manual_seed(out)
    whole = lambda *s: torch.randint(-1, 2, s, device=dev, generator=g, dtype=torch.int8).to(torch.bfloat16)
    x, w, dy = whole(rows, width).requires_grad_(), whole(out, width).requires_grad_(), whole(rows, out)
    b = torch.ones(out, device=dev, dtype=torch.bfloat16, requires_grad=True)
    y = linear_8bit(x, w, b)
    with torch.no_grad():
        assert torch.equal(y[-tail:], (x[-tail:].float() @ w.float().t() + 1).bfloat16())
        at = (1 << 31) // out                              # around the 2^31st result
        assert torch.equal(y[at - 50:at + 50], (x[at - 50:at + 50].float() @ w.float().t() + 1).bfloat16())
    del y
    dx, dw, db = torch.autograd.grad(linear_8bit(x, w, b), (x, w, b), dy)
    with torch.no_grad():
        assert torch.equal(dx[-tail:], (dy[-tail:].float() @ w.float()).bfloat16())
        want, sums = torch.zeros(out, width, device=dev), torch.zeros(out, device=dev)
        for k in range(0, rows, 1 << 17):
            piece = dy[k:k + (1 << 17)].float()
            want += piece.t().contiguous() @ x[k:k + (1 << 17)].float()
            sums += piece.sum(0)
        assert torch.equal(dw, want.bfloat16()) and torch.equal(db, sums.bfloat16())
        del dx, dw, want
    if out == 1024:
        return
    n = torch.ones(width, device=dev, dtype=torch.bfloat16, requires_grad=True)
    end = x.detach()[-tail:].clone().requires_grad_()
    kept = quantize_blocks(x.detach())
    assert torch.equal(kept.dequantize(torch.bfloat16)[-tail:], quantize_blocks(end.detach()).dequantize(torch.bfloat16))
    del kept, dy
    for op in (gelu_8bit, lambda t: layer_norm_8bit(t, n, n)):
        y, z = op(x), op(end)
        assert torch.equal(y[-tail:], z)
        assert torch.equal(torch.autograd.grad(y, x, y.detach())[0][-tail:], torch.autograd.grad(z, end, z.detach())[0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_of_one_tensor_twice(dev, dtype):
    """x is its own weight, and the gradients add up."""
    from vtpack_amd.layers import linear_8bit
    x = _numbers(dev, 96, 96, dtype=dtype, scale=0.1).requires_grad_()
    other = x.detach().clone().requires_grad_()
    dy = _numbers(dev, 96, 96, dtype=dtype, seed=5)
    y, z = linear_8bit(x, x), linear_8bit(x.detach().clone().requires_grad_(), other)
    assert torch.equal(y, z)
    got = torch.autograd.grad(y, x, dy)[0]
    left = x.detach().clone().requires_grad_()
    parts = torch.autograd.grad(linear_8bit(left, other), (left, other), dy)
    assert torch.equal(got, parts[0] + parts[1])


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_of_any_layout(dev, dtype):
    """Leading dimensions, strides, gradients that are broadcast or lie anyhow; some of the gradients alone."""
    from vtpack_amd.layers import linear_8bit
    base, w0 = _numbers(dev, 40, 301, dtype=dtype), _numbers(dev, 300, 301, dtype=dtype, scale=0.05)
    b = _numbers(dev, 600, dtype=dtype)[::2]
    for x, w in ((base[:, 1:257], w0[:64, 7:263]), (base[3::2, :200], w0[::3, :200]), (base[:, None, :160].expand(40, 3, 160), w0[:, :160]),
                 (base[:, :40].t(), w0[:100, :40]), (base[0, :128], w0[:, 100:228]), (base[:1, 5:], w0[:, 5:])):
        out = w.shape[0]
        plain = linear_8bit(x.reshape(-1, x.shape[-1]).contiguous(), w.contiguous(), b[:out].contiguous())
        leaves = [t.detach().requires_grad_() for t in (x, w, b[:out])]
        y = linear_8bit(*leaves)
        assert y.shape == (*x.shape[:-1], out) and torch.equal(y.reshape(-1, out), plain)
        for dy in (torch.ones((), dtype=dtype, device=dev).expand(y.shape), _numbers(dev, *y.shape[:-1], 2 * out, dtype=dtype)[..., ::2],
                   _numbers(dev, *y.shape[:-1], out + 8, dtype=dtype)[..., 3:out + 3]):
            flat = [t.detach().contiguous().requires_grad_() for t in (x.reshape(-1, x.shape[-1]), w, b[:out])]
            want = torch.autograd.grad(linear_8bit(*flat), flat, dy.reshape(-1, out).contiguous())
            got = torch.autograd.grad(y, leaves, dy, retain_graph=True)
            for k, (g, r) in enumerate(zip(got, want)):
                assert g.shape == leaves[k].shape
                assert torch.equal(g.reshape(r.shape), r), k
                assert torch.equal(torch.autograd.grad(y, leaves[k], dy, retain_graph=True)[0], g), k


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_that_are_not_finite_reach_their_own_results(dev, dtype):
    """An infinity or NaN in x makes its row of y NaN; one in the gradient reaches its row of dx and the sums that it is in."""
    from vtpack_amd.layers import linear_8bit
    x, w, b = _operands(dev, 70, 90, 200, dtype)
    clean = linear_8bit(x, w, b)
    x[3, 7], x[69, 199] = float("inf"), float("nan")
    y = linear_8bit(x, w, b)
    bad = torch.zeros(70, dtype=torch.bool, device=dev)
    bad[3] = bad[69] = True
    assert torch.isnan(y[bad]).all() and torch.equal(y[~bad], clean[~bad])
    x = _operands(dev, 70, 90, 200, dtype)[0].requires_grad_()
    wl = w.clone().requires_grad_()
    dy = _numbers(dev, 70, 90, dtype=dtype)
    want = torch.autograd.grad(linear_8bit(x, wl, b), (x, wl), dy)
    dy[69, 89] = float("inf")
    dx, dw = torch.autograd.grad(linear_8bit(x, wl, b), (x, wl), dy)
    assert not torch.isfinite(dx[69]).all() and torch.equal(dx[:69], want[0][:69])
    assert not torch.isfinite(dw[89]).all() and torch.equal(dw[:89], want[1][:89])


def test_no_rows(dev):
    from vtpack_amd.layers import gelu_8bit, layer_norm_8bit, linear_8bit
    x, w, b = (t.requires_grad_() for t in _operands(dev, 2, 30, 64, torch.float32))
    empty = x.detach()[:0].reshape(0, 3, 64).requires_grad_()
    y = linear_8bit(empty, w, b)
    assert y.shape == (0, 3, 30)
    dx, dw, db = torch.autograd.grad(y.sum(), (empty, w, b))
    assert dx.shape == empty.shape and dw.shape == w.shape and not dw.any() and not db.any()
    y = gelu_8bit(empty)
    assert torch.autograd.grad(y.sum(), empty)[0].shape == empty.shape
    n = [torch.ones(64, device=dev).requires_grad_() for _ in range(2)]
    grads = torch.autograd.grad(layer_norm_8bit(empty, *n).sum(), (empty, *n))
    assert grads[0].shape == empty.shape and not grads[1].any() and not grads[2].any()


# ------------------------------------------------------------------------------------------------ GELU, LayerNorm
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (2, 128), (5, 129), (33, 1536), (4, 3, 200), (1021, 768), (1, 8), (2, 5000)])
def test_gelu(dev, dtype, shape):
    from vtpack_amd.layers import gelu_8bit
    x = _numbers(dev, *shape, dtype=dtype, scale=1.5).requires_grad_()
    dy = _numbers(dev, *shape, dtype=dtype, seed=5)
    x64, c, g = x.detach().cpu().double(), ref.q(x), dy.cpu().double()
    poly = 1.4e-4 if dtype == torch.bfloat16 else 4e-7
    y = gelu_8bit(x)
    _within(y, ref.gelu(x64), poly * x64.abs() + HALF[dtype] * ref.gelu(x64).abs() * 1.01 + 1e-38, "y")
    slope = ref.gelu_slope(c)
    dx, = torch.autograd.grad(y, x, dy)
    _within(dx, g * slope, (poly * g.abs() + HALF[dtype] * (g * slope).abs()) * 1.01 + 1e-38, "dx")
    assert torch.equal(gelu_8bit(x.detach()), y)


@pytest.mark.parametrize("dtype", DTYPES)
def test_gelu_far_out(dev, dtype):
    from vtpack_amd.layers import gelu_8bit
    x = torch.tensor([[-1e30, -40.0, -13.0, -6.0, -0.0, 0.0, 1e-30, 6.0, 13.0, 40.0, 1e30], [float("inf"), 1.0, -1.0] + [0.5] * 8,
                      [float("nan")] * 11], dtype=dtype).to(dev).requires_grad_()
    y = gelu_8bit(x)
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    want = ref.gelu(x.detach().cpu().double())
    assert torch.equal(torch.isnan(y.cpu()), torch.isnan(want)) and float(y[1, 0]) == float("inf")
    slope = ref.gelu_slope(ref.q(x))
    _within(dx, slope, (1.4e-4 if dtype == torch.bfloat16 else 4e-7) + HALF[dtype] * slope.abs() * 1.01, "dx")


WIDTHS = [1, 7, 8, 64, 127, 128, 129, 384, 512, 513, 1000, 1024, 1025, 2048, 4100, 8192]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", WIDTHS)
@pytest.mark.parametrize("rows", [1, 3, 70])
def test_layer_norm(dev, dtype, n, rows):
    from vtpack_amd.layers import layer_norm_8bit
    x = _numbers(dev, rows, n, dtype=dtype).requires_grad_()
    w = (1 + 0.2 * _numbers(dev, n, seed=1)).to(dtype).requires_grad_()
    b = _numbers(dev, n, dtype=dtype, seed=2).requires_grad_()
    dy = _numbers(dev, rows, n, dtype=dtype, seed=3)
    want, grads = ref.layer_norm(x, w, b, 1e-6, dy)
    y = layer_norm_8bit(x, w, b)
    big = want.abs() + b.detach().cpu().double().abs()
    _within(y, want, (16 * WALK * (1 + big) + HALF[dtype] * want.abs()) * 1.01, "y")
    got = torch.autograd.grad(y, (x, w, b), dy)
    # each term of a sum is off by a few half steps, and the sums walk
    x64, w64, g64 = x.detach().cpu().double(), w.detach().cpu().double(), dy.cpu().double()
    c = x64 - x64.mean(1, keepdim=True)
    r = 1 / torch.sqrt((c * c).mean(1, keepdim=True) + 1e-6)
    h = (ref.q(x.detach().cpu().float() - x64.mean(1, keepdim=True).float()) * r).abs()
    gw = (g64 * w64).abs()
    size = r * (gw + gw.mean(1, keepdim=True) + h * (gw * h).mean(1, keepdim=True))
    walk = WALK * (16 + 2 * math.sqrt(n))
    for name, a, want, bound in (("dx", got[0], grads[0], walk * size), ("dw", got[1], grads[1], WALK * (16 + 2 * math.sqrt(rows)) * (g64.abs() * h).sum(0)),
                                 ("db", got[2], grads[2], WALK * (8 + 2 * math.sqrt(rows)) * g64.abs().sum(0))):
        assert a.dtype == dtype
        _within(a, want, (bound + HALF[dtype] * want.abs()) * 1.01 + 1e-38, name)
    assert torch.equal(layer_norm_8bit(x.detach(), w.detach(), b.detach()), y)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,rows", [(384, 5000), (2048, 3000), (40, 20001)])
def test_layer_norm_of_many_rows(dev, dtype, n, rows):
    test_layer_norm(dev, dtype, n, rows)


@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_norm_far_from_zero(dev, dtype):
    """A mean a thousand times the spread, a row of equal numbers, one that is not finite, dimensions and strides."""
    from vtpack_amd.layers import layer_norm_8bit
    x = torch.randn(5, 300, generator=torch.Generator().manual_seed(1)) + 1000
    x[1] = 3.25
    x = x.to(dev, dtype)
    w, b = torch.ones(300, device=dev, dtype=dtype), torch.zeros(300, device=dev, dtype=dtype)
    leaves = [t.requires_grad_() for t in (x.clone(), w, b)]
    dy = _numbers(dev, 5, 300, dtype=dtype)
    want, grads = ref.layer_norm(x, w, b, 1e-6, dy)
    y = layer_norm_8bit(*leaves)
    assert (y.detach().cpu().double() - want).abs().max() <= 2e-3 + 2.0 ** -8 * (dtype == torch.bfloat16) * want.abs().max()
    got = torch.autograd.grad(y, leaves, dy)
    assert float((got[0].cpu().double() - grads[0]).norm()) <= (5e-5 if dtype == torch.float32 else 5e-3) * float(grads[0].norm())
    assert not got[0][1].isnan().any()
    bad = x.clone()
    bad[2, 5], bad[4, 0] = float("nan"), float("inf")
    out = layer_norm_8bit(bad, w, b)
    assert torch.isnan(out[[2, 4]]).all() and torch.equal(out[[0, 1, 3]], y[[0, 1, 3]])
    three = x.reshape(1, 5, 300)[:, ::2]
    assert torch.equal(layer_norm_8bit(three, w, b)[0], y[::2])
    assert torch.equal(layer_norm_8bit(x[:, 3:], w[3:], b[3:]), layer_norm_8bit(x[:, 3:].contiguous(), w[3:].contiguous(), b[3:].contiguous()))


# ------------------------------------------------------------------------------------------------ gradients against differences
def test_gradients_against_differences(dev):
    """At points that blocks hold exactly the gradients are the operators' own: central differences of the function in 64 bits."""
    from vtpack_amd.layers import gelu_8bit, layer_norm_8bit, linear_8bit
    g = torch.Generator().manual_seed(2)
    x = torch.randint(-14, 15, (6, 40), generator=g).double() / 8
    x[:, -1] -= x.sum(1)                               # a mean of zero
    x[:, -1] = x[:, -1].clamp(-14, 14) * 0
    x[:, 0] = 0
    x = torch.cat([x, -x], 1)
    w, b = torch.randint(-7, 8, (9, 80), generator=g).double() / 16, torch.randn(9, generator=g).double().float().double()
    nw, nb = torch.randn(80, generator=g).float().double(), torch.randn(80, generator=g).float().double()
    assert torch.equal(ref.q(x), x) and torch.equal(ref.q(w), w)

    def differences(f, at, t, step=1e-4):
        out = torch.zeros_like(t)
        for i in range(t.numel()):
            d = torch.zeros_like(t).reshape(-1)
            d[i] = step
            d = d.view_as(t)
            out.view(-1)[i] = (f(t + d) - f(t - d)) / (2 * step)
        return out

    cot = {n: torch.randn(6, n, generator=g).to(torch.bfloat16).double() for n in (9, 80)}
    lin = lambda x, w, b: ((x @ w.t() + b) * cot[9]).sum()                                           # noqa: E731
    gel = lambda x: (ref.gelu(x) * cot[80]).sum()                                                    # noqa: E731
    nor = lambda x, w, b: (torch.nn.functional.layer_norm(x, (80,), w, b, 1e-6) * cot[80]).sum()     # noqa: E731
    for op, f, args, n in ((linear_8bit, lin, (x, w, b), 9), (gelu_8bit, gel, (x,), 80), (layer_norm_8bit, nor, (x, nw, nb), 80)):
        leaves = [t.float().to(dev).requires_grad_() for t in args]
        got = torch.autograd.grad(op(*leaves), leaves, cot[n].float().to(dev))
        for k, t in enumerate(args):
            want = differences(lambda v: f(*args[:k], v, *args[k + 1:]), None, t)
            # the difference's own error is a third derivative times 1e-8 / 6, and 1e-16 / 1e-4 of the function
            assert (got[k].cpu().double() - want).abs().max() <= 2e-5 * (1 + want.abs().max()), (op.__name__, k)


# ------------------------------------------------------------------------------------------------ as programs use them
def _pass(dev, dtype, x, w1, b1, w2, b2, nw, nb, dy):
    from vtpack_amd.layers import gelu_8bit, layer_norm_8bit, linear_8bit
    leaves = [t.detach().requires_grad_() for t in (x, w1, b1, w2, b2, nw, nb)]
    h = layer_norm_8bit(leaves[0], leaves[5], leaves[6])
    y = linear_8bit(gelu_8bit(linear_8bit(h, leaves[1], leaves[2])), leaves[3], leaves[4])
    return [y.detach(), *torch.autograd.grad(y, leaves, dy)]


def _mlp(dev, dtype, rows=150, width=192, seed=0):
    x, dy = _numbers(dev, rows, width, dtype=dtype, seed=seed), _numbers(dev, rows, width, dtype=dtype, seed=seed + 9)
    w1, w2 = (_numbers(dev, *s, dtype=dtype, seed=seed + 3, scale=0.04) for s in ((4 * width, width), (width, 4 * width)))
    b1, b2, nw, nb = (_numbers(dev, n, dtype=dtype, seed=seed + 4) for n in (4 * width, width, width, width))
    return x, w1, b1, w2, b2, nw, nb, dy


@pytest.mark.parametrize("dtype", DTYPES)
def test_mlp_is_the_run_of_its_operators(dev, dtype):
    """LayerNorm, Linear, GELU, Linear and back: near a pass that keeps everything, and the same bits every time."""
    operands = _mlp(dev, dtype)
    first = _pass(dev, dtype, *operands)
    for a, b in zip(first, _pass(dev, dtype, *operands)):
        assert torch.equal(a, b)
    x, w1, b1, w2, b2, nw, nb, dy = (t.detach().cpu().double() for t in operands)
    leaves = [t.requires_grad_() for t in (x, w1, b1, w2, b2, nw, nb)]
    F = torch.nn.functional
    y = F.linear(F.gelu(F.linear(F.layer_norm(x, x.shape[-1:], nw, nb, 1e-6), w1, b1)), w2, b2)
    # 8-bit operands are off by 2^-4 of a value at most, some 0.02 of it on the whole, on both sides of two products
    for got, want in zip(first, [y, *torch.autograd.grad(y, leaves, dy)]):
        assert float((got.cpu().double() - want.detach()).norm()) <= 0.12 * float(want.detach().norm())


@pytest.mark.parametrize("dtype", DTYPES)
def test_same_bits_on_another_stream_and_in_a_graph(dev, dtype):
    from vtpack_amd.layers import quantize_blocks
    operands = _mlp(dev, dtype)
    want = _pass(dev, dtype, *operands)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = _pass(dev, dtype, *operands)
        kept = quantize_blocks(operands[0]).dequantize(dtype)
    torch.cuda.current_stream().wait_stream(stream)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    static = [t.clone() for t in operands]
    with torch.cuda.stream(stream):
        _pass(dev, dtype, *static)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _pass(dev, dtype, *static)
        blocks = quantize_blocks(static[0])
        back = blocks.dequantize(dtype)
    for seed in (0, 20, 40, 60):
        fresh = _mlp(dev, dtype, seed=seed)
        for s, f in zip(static, fresh):
            s.copy_(f)
        eager = _pass(dev, dtype, *fresh)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, eager):
            assert torch.equal(a, b)
        assert torch.equal(back, quantize_blocks(fresh[0]).dequantize(dtype))
    assert kept.shape == operands[0].shape


@pytest.mark.parametrize("dtype", DTYPES)
def test_two_passes_beside_each_other(dev, dtype):
    """Forward passes of two inputs before either's gradients, on two streams."""
    a, b = _mlp(dev, dtype, seed=1), _mlp(dev, dtype, rows=77, seed=2)
    want = _pass(dev, dtype, *a), _pass(dev, dtype, *b)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for s, o in zip(streams, (a, b)):
            with torch.cuda.stream(s):
                got.append(_pass(dev, dtype, *o))
    torch.cuda.synchronize()
    for k, g in enumerate(got):
        for u, v in zip(g, want[k % 2]):
            assert torch.equal(u, v)


def test_what_a_pass_keeps(dev):
    """A byte a number, and nothing without gradients; neither x nor weight are held, and changing x afterwards changes nothing."""
    from vtpack_amd.layers import gelu_8bit, layer_norm_8bit, linear_8bit
    rows, width, out = 4096, 1024, 2048
    x, w, b = (t.requires_grad_() for t in _operands(dev, rows, out, width, torch.float32))
    nw, nb = torch.ones(width, device=dev), torch.zeros(width, device=dev)
    dy = torch.ones(rows, out, device=dev)
    for op, kept in ((lambda: linear_8bit(x, w, b), (rows + out) * width), (lambda: gelu_8bit(x), rows * width), (lambda: layer_norm_8bit(x, nw, nb), rows * (width + 4))):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = op()
        held = torch.cuda.memory_allocated() - before - y.numel() * 4
        assert kept <= held <= kept * 1.02 + 4096
        with torch.no_grad():
            z = op()
        assert torch.cuda.memory_allocated() - before - held - 2 * y.numel() * 4 <= 4096
        assert z.grad_fn is None and torch.equal(y, z)
        del y, z
    y = linear_8bit(x, w, b)
    want = torch.autograd.grad(y, (x, w), dy, retain_graph=True)
    with torch.no_grad():
        x.mul_(3.0)
        w.zero_()
    for u, v in zip(torch.autograd.grad(y, (x, w), dy), want):
        assert torch.equal(u, v)
    only = linear_8bit(x.detach(), w, b)
    assert torch.autograd.grad(only, b, dy)[0].shape == b.shape


def test_saved_tensor_hooks(dev):
    """What is kept goes through hooks on saved tensors (here: to host memory and back); what they bring back is looked at."""
    from torch.autograd.graph import save_on_cpu, saved_tensors_hooks
    operands = _mlp(dev, torch.float32)
    want = _pass(dev, torch.float32, *operands)
    with save_on_cpu():
        got = _pass(dev, torch.float32, *operands)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    from vtpack_amd.layers import gelu_8bit, layer_norm_8bit, linear_8bit
    x, w, b = (t.requires_grad_() for t in _operands(dev, 30, 40, 200, torch.float32))
    n = torch.ones(200, device=dev)
    for back in (lambda t: t.cpu(), lambda t: t[:-4], lambda t: t.float(), lambda t: torch.cat([t, t])[1:t.numel() + 1]):
        for op in (lambda: linear_8bit(x, w, b), lambda: gelu_8bit(x), lambda: layer_norm_8bit(x, n, n)):
            with saved_tensors_hooks(lambda t: t, back):
                y = op()
            with pytest.raises(RuntimeError, match="have to be|has to be"):
                y.sum().backward()
            x.grad = w.grad = b.grad = None


@pytest.mark.parametrize("dtype", DTYPES)
def test_worked_out_again(dev, dtype):
    """A checkpointed run keeps no blocks and makes the same again."""
    from torch.utils.checkpoint import checkpoint
    from vtpack_amd.layers import gelu_8bit, layer_norm_8bit, linear_8bit

    def run(x, w1, b1, w2, b2, nw, nb):
        return linear_8bit(gelu_8bit(linear_8bit(layer_norm_8bit(x, nw, nb), w1, b1)), w2, b2)

    *operands, dy = _mlp(dev, dtype)
    leaves = [t.detach().requires_grad_() for t in operands]
    want = torch.autograd.grad(run(*leaves), leaves, dy)
    for reentrant in (False, True):
        again = [t.detach().clone().requires_grad_() for t in operands]
        checkpoint(run, *again, use_reentrant=reentrant).backward(dy)
        for a, b in zip(again, want):
            assert torch.equal(a.grad, b)


def test_threads(dev):
    """Passes of several threads at once, each on its stream."""
    import threading
    operands = [_mlp(dev, torch.float32, rows=40 + 13 * k, seed=k) for k in range(3)]
    want = [_pass(dev, torch.float32, *o) for o in operands]
    torch.cuda.synchronize()
    got, errors = [None] * 3, []

    def work(k):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(5):
                    got[k] = _pass(dev, torch.float32, *operands[k])
            stream.synchronize()
        except Exception as e:                             # for the thread that looks at it
            errors.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for a, b in zip(got, want):
        for u, v in zip(a, b):
            assert torch.equal(u, v)


def test_a_graph_is_used_once_and_weights_are_watched(dev):
    from vtpack_amd.layers import gelu_8bit, layer_norm_8bit, linear_8bit
    x, w, b = (t.requires_grad_() for t in _operands(dev, 30, 40, 64, torch.float32))
    n = torch.ones(64, device=dev, requires_grad=True)
    for op in (lambda: linear_8bit(x, w, b), lambda: gelu_8bit(x), lambda: layer_norm_8bit(x, n, n)):
        y = op()
        torch.autograd.grad(y.sum(), x)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(y.sum(), x)
    y = layer_norm_8bit(x, n, n)
    with torch.no_grad():
        n.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y.sum(), x)


def test_refusals_on_the_gpu(dev):
    from vtpack_amd.layers import Blocks, gelu_8bit, layer_norm_8bit, linear_8bit, quantize_blocks
    x, w, b = _operands(dev, 6, 8, 64, torch.float32)
    kept = quantize_blocks(w)
    n = torch.ones(64, device=dev)
    for bad, args in ((TypeError, (x.double(), w)), (TypeError, (x, w.bfloat16())), (TypeError, (x, w, b.bfloat16())), (ValueError, (x[:, :32], w)),
                      (ValueError, (x, w[0])), (ValueError, (x, w, b[:5])), (RuntimeError, (x, w.cpu())), (ValueError, (x[:, :32], kept)),
                      (ValueError, (x, quantize_blocks(w[0]))), (RuntimeError, (x.cpu(), kept)), (ValueError, (x[:, :0], w[:, :0])), (ValueError, (x, w[:0])),
                      (TypeError, (x, kept, b.bfloat16())), (TypeError, (x.to_sparse(), "w")), (ValueError, (x.to_sparse(), w)), (ValueError, (x[0, 0], w))):
        with pytest.raises(bad):
            linear_8bit(*args)
    with pytest.raises(ValueError, match="act"):
        linear_8bit(x, w, act="relu")
    with pytest.raises(RuntimeError, match="gelu_8bit"):
        linear_8bit(x.clone().requires_grad_(), w, act="gelu")
    with torch.no_grad():
        linear_8bit(x.clone().requires_grad_(), w, act="gelu")
    for bad, args in ((TypeError, (x, n.bfloat16(), n)), (ValueError, (x, n[:5], n)), (ValueError, (x, n, n[None])), (ValueError, (x, n, n, -1.0)),
                      (ValueError, (x, n, n, float("nan"))), (TypeError, (x, None, None)), (ValueError, (torch.ones(2, 8193, device=dev),) * 3)):
        with pytest.raises(bad):
            layer_norm_8bit(*args)
    assert torch.equal(layer_norm_8bit(x, n, n, 0), layer_norm_8bit(x, n, n, 0.0))
    for bad, x_ in ((TypeError, x.half()), (TypeError, 3.0), (ValueError, x[0, 0]), (ValueError, x[:, :0])):
        with pytest.raises(bad):
            gelu_8bit(x_)
        with pytest.raises(bad):
            quantize_blocks(x_)
    with pytest.raises(TypeError):
        kept.dequantize(torch.float16)
    with pytest.raises(TypeError):
        Blocks(x, kept.scales)
    with pytest.raises(ValueError):
        Blocks(kept.values, kept.scales[:, :0])
    leaf = x.clone().requires_grad_()
    for op in (lambda v: linear_8bit(v, w), gelu_8bit, lambda v: layer_norm_8bit(v, n, n)):
        with pytest.raises(RuntimeError, match="gradients of the gradients"):
            torch.autograd.grad(op(leaf).sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(op, (x,), check_trace=False)
        with torch.autograd.forward_ad.dual_level():
            with pytest.raises(RuntimeError, match="forward-mode"):
                op(torch.autograd.forward_ad.make_dual(x, x))


# ------------------------------------------------------------------------------------------------ in the models
def _deit(dev, **kw):
    from vtpack_amd.models.dge.deit_dge import VisionTransformer
    from vtpack_amd.synthetic import set_synthetic_router
    torch.manual_seed(0)
    m = VisionTransformer(img_size=64, patch_size=8, embed_dim=64, depth=2, num_heads=1, mlp_ratio=2, num_classes=7, split_sizes=[4, 2, 1], **kw)
    return set_synthetic_router(m, 2).to(dev).train()


def _pvt(dev):
    from vtpack_amd.models.dge.pvt_dge import PyramidVisionTransformer
    torch.manual_seed(0)
    return PyramidVisionTransformer(img_size=128, patch_size=4, num_classes=9, embed_dims=[64, 64, 64, 64], num_heads=[1, 1, 1, 1], mlp_ratios=[2] * 4,
                                    depths=[1, 1, 1, 1], sr_ratios=[8, 4, 2, 1], split_sizes=[[4, 2, 1]] * 4, qkv_bias=True).to(dev).train()


def _saved_bytes(run):
    """Bytes of the distinct tensors on the GPU that a pass saves for its gradients."""
    from torch.autograd.graph import saved_tensors_hooks
    seen = {}

    def pack(t):
        if t.is_cuda:
            seen[t.untyped_storage().data_ptr()] = t.untyped_storage().nbytes()
        return t
    with saved_tensors_hooks(pack, lambda t: t):
        out = run()
    return out, sum(seen.values())


@pytest.mark.parametrize("make,size", [(_deit, 64), (_pvt, 128)])
def test_training_pass_of_a_model(dev, make, size):
    """The same pass in 8 bits: a loss and gradients beside the full ones', fewer bytes kept, eval mode as it was."""
    from vtpack_amd.synthetic import synthetic_images
    m = make(dev)
    images, target = synthetic_images(4, size, seed=1).to(dev), torch.tensor([1, 0, 3, 2], device=dev)
    runs = []
    for on in (False, True):
        m.set_eight_bit(on)
        torch.manual_seed(5)                              # the gates are sampled
        loss, kept = _saved_bytes(lambda: m(images, target))
        m.zero_grad(set_to_none=True)
        loss.backward()
        runs.append((float(loss.detach()), {n: p.grad.clone() for n, p in m.named_parameters() if p.grad is not None}, kept))
    (loss, grads, kept), (loss8, grads8, kept8) = runs
    assert grads.keys() == grads8.keys() and kept8 < 0.8 * kept
    assert loss8 != loss and abs(loss8 - loss) <= 0.1 * loss
    for n in grads:
        assert torch.isfinite(grads8[n]).all(), n
    whole = [torch.cat([g[n].flatten() for n in grads if "dge.router" not in n]) for g in (grads, grads8)]
    assert float(torch.nn.functional.cosine_similarity(*whole, dim=0)) > 0.9
    m.eval()
    with torch.no_grad():
        a = m(images)
        m.set_eight_bit(False)
        assert torch.equal(a, m(images))


def test_steps_of_a_model_in_eight_bits(dev):
    """Training steps with the harness: weights move, and the same bits twice."""
    from vtpack_amd import harness
    from vtpack_amd.optim import AdamW
    from vtpack_amd.synthetic import synthetic_images
    images, target = synthetic_images(4, 64, seed=1).to(dev), torch.tensor([1, 0, 3, 2], device=dev)
    ends = []
    for _ in range(2):
        m = _deit(dev).set_eight_bit()
        before = {n: p.detach().clone() for n, p in m.named_parameters()}
        opt = AdamW(harness.weight_decay_groups(m, 0.05), lr=1e-3)
        torch.manual_seed(9)
        for _ in range(3):
            out = harness.train_step(m, images, target, opt, dge_enable=True, dge_budget=0.5, balance_scale=0.01, finite=True)
        assert math.isfinite(float(out["loss"]))
        ends.append({n: p.detach() for n, p in m.named_parameters()})
        assert all(not torch.equal(before[n], p) for n, p in m.named_parameters() if p.grad is not None and p.grad.any())
    # (torch's own backward of the patch convolution may differ from run to run)
    for n in ends[0]:
        assert (ends[0][n].float() - ends[1][n].float()).abs().max() <= 3.1e-3, n
