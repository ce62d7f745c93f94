"""The classifier's cross entropy and its gradients against the formula in float64: tiles and slabs around their edges, rows that
are left out, infinite biases, pieces of the classes, strides, graphs, streams.

Bounds.  fp32: every sum is six times its length of products in fp32, sixteen a step of the matrix instruction, and its error
grows as a walk of that many half steps: 2^-24 (8 + 2 sqrt(6 n / 16)) of the 2-norm, n the longest sum.  bf16: the
gradients of the logits are rounded once (neighbours between 1 and 2 are 2^-7 apart: half a step is 2^-8 of a term at most) and so is
the result: element by element 2^-8 |d| |w| + 2^-8 |result|, and what the fp32 sums add."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16]


def _operands(dev, rows, classes, width, dtype, seed=0, bias=True, left_out=0.0):
    g = torch.Generator().manual_seed(seed * 7919 + rows * 31 + classes * 7 + width)
    x = torch.randn(rows, width, generator=g)
    w = torch.randn(classes, width, generator=g) * (1.5 / math.sqrt(width))
    b = torch.randn(classes, generator=g) * 0.5 if bias else None
    t = torch.randint(0, classes, (rows,), generator=g)
    if left_out:
        t[torch.rand(rows, generator=g) < left_out] = -100
    return [None if v is None else v.to(dev, v.dtype if v.dtype == torch.int64 else dtype) for v in (x, w, b, t)]


def _reference(x, w, b, t, smoothing=0.0, ignore=-100, weights=None):
    """-> losses of the rows, d of the logits with the weights of the rows in it, (dx, dw, db), all float64."""
    x, w = x.double(), w.double()
    classes = w.shape[0]
    z = x @ w.t().contiguous() + (0 if b is None else b.double())
    live = (t != ignore) & (t >= 0) & (t < classes)
    rows = torch.arange(x.shape[0], device=x.device)[live]
    lse = torch.logsumexp(z, 1)
    loss = torch.zeros_like(lse)
    loss[live] = lse[live] - (1 - smoothing) * z[rows, t[live]]
    if smoothing:
        loss[live] -= smoothing * z[live].mean(1)
    weights = live.double() / max(1, int(live.sum())) if weights is None else live * weights.double()
    d = torch.exp(z - lse[:, None]) - smoothing / classes
    d[rows, t[live]] -= 1 - smoothing
    d = torch.where(live[:, None], d * weights[:, None], torch.zeros_like(d))
    x = torch.where(live[:, None], x, torch.zeros_like(x))
    return loss, weights, d, (d @ w, d.t().contiguous() @ x, d.sum(0))


def _tolerance(x, w):
    return HALF * (8 + 2 * math.sqrt(6 * max(*x.shape, *w.shape) / 16))


def _near(got, want, tol, floor=0.0):
    assert torch.isfinite(got).all()
    assert float((got.double() - want).norm()) <= tol * float(want.norm()) + floor


def _check(x, w, b, t, smoothing=0.0, reduction="mean", ignore=-100, grad=None):
    from vtpack_amd.layers import linear_cross_entropy
    leaves = [None if v is None else v.detach().requires_grad_() for v in (x, w, b)]
    loss = linear_cross_entropy(*leaves, t, ignore_index=ignore, label_smoothing=smoothing, reduction=reduction)
    scale = grad if grad is not None else torch.ones((), device=x.device) if reduction == "sum" else None
    want, weights, d, grads = _reference(x, w, b, t, smoothing, ignore, scale)
    tol = _tolerance(x, w)
    # of a loss: of the logits it is the difference of
    size = 1 + float((x.double().nan_to_num(0, 0, 0) @ w.double().t()).abs().max()) if x.shape[0] * w.shape[0] < 1 << 22 else 16.0
    if reduction == "none":
        assert (loss.double() - want).abs().max() <= tol * size
    else:
        total = want.sum() if reduction == "sum" else (want * weights).sum()
        assert abs(float(loss.detach()) - float(total)) <= tol * size * (x.shape[0] if reduction == "sum" else 1)
    got = torch.autograd.grad(loss, [v for v in leaves if v is not None], grad)
    for name, g, r in zip("xwb", got, grads):
        assert g.dtype == x.dtype and g.shape == r.shape
        if x.dtype == torch.float32:
            _near(g, r, tol, 1e-30)
        else:
            e = 2.0 ** -8 * r.abs() + tol * float(r.abs().max())
            if name == "x":
                e = e + 2.0 ** -8 * (d.abs() @ w.double().abs()) * 1.01
            elif name == "w":
                e = e + 2.0 ** -8 * (d.abs().t().contiguous() @ x.nan_to_num(0, 0, 0).double().abs()) * 1.01
            else:                                        # the sum of the rounded d: |rounded d - d| <= 2^-8 |d|, summed over the rows
                e = e + 2.0 ** -8 * d.abs().sum(0) * 1.01
            over = float(((g.double() - r).abs() / (e + 1e-30)).max())
            assert over <= 1, name
    return loss, got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,classes,width", [(1, 1, 1), (1, 2, 8), (2, 10, 64), (3, 1000, 192), (127, 129, 65), (128, 128, 128),
                                                (129, 127, 63), (64, 1000, 384), (255, 257, 200), (300, 130, 72), (1021, 1000, 384),
                                                (65, 2049, 320), (17, 3, 1027)])
def test_sizes(dev, dtype, rows, classes, width):
    _check(*_operands(dev, rows, classes, width, dtype))
    _check(*_operands(dev, rows, classes, width, dtype, seed=1, bias=False), smoothing=0.1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_rows_left_out(dev, dtype, reduction):
    """Padding, targets that are no class, features of such rows that are not finite; a weight for every row."""
    x, w, b, t = _operands(dev, 200, 300, 96, dtype, left_out=0.3)
    t[3], t[4], t[150] = 300, -7, 1 << 40
    x[t < 0] = float("nan")
    x[3], x[150] = float("inf"), float("-inf")
    grad = None
    if reduction == "none":
        grad = torch.rand(200, generator=torch.Generator().manual_seed(5)).to(dev) + 0.5
    loss, got = _check(x, w, b, t, smoothing=0.1, reduction=reduction, grad=grad)
    out = (t < 0) | (t >= 300)
    assert not got[0][out].any()
    if reduction == "none":
        assert not loss[out].any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_no_row_counts(dev, dtype):
    from vtpack_amd.layers import linear_cross_entropy
    x, w, b, t = _operands(dev, 20, 30, 64, dtype)
    x[:] = float("nan")
    t[:] = -100
    leaves = [v.requires_grad_() for v in (x, w, b)]
    loss = linear_cross_entropy(*leaves, t)
    assert float(loss.detach()) == 0.0
    for g in torch.autograd.grad(loss, leaves):
        assert not g.any()
    empty = [x.detach()[:0].requires_grad_(), w, b]
    loss = linear_cross_entropy(*empty, t[:0])
    assert float(loss) == 0.0
    for g, v in zip(torch.autograd.grad(loss, empty), empty):
        assert g.shape == v.shape and not g.any()
    assert linear_cross_entropy(*empty, t[:0], reduction="none").shape == (0,)


def test_ignore_index_that_is_a_class(dev):
    x, w, b, t = _operands(dev, 100, 10, 64, torch.float32)
    _check(x, w, b, t, ignore=3)


def test_classes_shut_out_by_the_bias(dev):
    """A bias of -inf takes a class out of the sum; a row whose own class it is loses all, and its gradients stay finite."""
    from vtpack_amd.layers import linear_cross_entropy
    x, w, b, t = _operands(dev, 90, 400, 64, torch.float32)
    b[::3] = float("-inf")
    t = t // 3 * 3 + 1
    t[t >= 400] = 1
    loss, got = _check(x, w, b, t)
    assert not got[1][::3].any()
    b[:] = float("-inf")
    b[7] = 0.0
    assert torch.equal(linear_cross_entropy(x, w, b, torch.full_like(t, 7), reduction="none"), torch.zeros(90, device=dev))
    assert linear_cross_entropy(x, w, b, torch.full_like(t, 8), reduction="none").isposinf().all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_not_a_number(dev, dtype):
    """A NaN or an infinity in a row that counts shows in its loss and leaves the other rows' alone."""
    from vtpack_amd.layers import linear_cross_entropy
    x, w, b, t = _operands(dev, 140, 150, 64, dtype)
    want = linear_cross_entropy(x, w, b, t, reduction="none")
    x[7, 3], x[131, 0] = float("nan"), float("inf")
    got = linear_cross_entropy(x, w, b, t, reduction="none")
    rest = torch.ones(140, dtype=torch.bool, device=dev)
    rest[7] = rest[131] = False
    assert torch.equal(got[rest], want[rest]) and not torch.isfinite(got[~rest]).any()


def test_large_logits(dev):
    """Logits of hundreds: the loss is a difference of neighbours, not of sums."""
    x, w, b, t = _operands(dev, 64, 128, 64, torch.float32)
    _check(x * 30, w * 10, b, t)


@pytest.mark.parametrize("dtype,rows,classes,width", [(torch.bfloat16, 8192, 21841, 128), (torch.float32, 4096, 12000, 64), (torch.bfloat16, 1, 70001, 256),
                                                      (torch.float32, 3, 40000, 100), (torch.bfloat16, 9000, 3, 64),
                                                      (torch.bfloat16, 3, 34001, 1024), (torch.bfloat16, 64, 34001, 1024)])
def test_pieces_and_long_sums(dev, dtype, rows, classes, width):
    """More classes than a piece holds; one row against many classes and the other way around, where sums are cut."""
    _check(*_operands(dev, rows, classes, width, dtype, left_out=0.1 if rows > 10 else 0.0))


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_places(dev, dtype):
    """Rows apart, columns of a wider matrix, storage off the 16-byte boundary, leading dimensions, expanded gradients."""
    from vtpack_amd.layers import linear_cross_entropy
    x, w, b, t = _operands(dev, 60, 70, 64, dtype)
    want = [linear_cross_entropy(x, w, b, t), *_check(x, w, b, t)[1]]
    wide = torch.zeros(60, 200, dtype=dtype, device=dev)
    wide[:, 3:67] = x
    off = torch.zeros(70 * 64 + 1, dtype=dtype, device=dev)
    off[1:] = w.reshape(-1)
    for xs, ws in ((wide[:, 3:67], off[1:].view(70, 64)), (x.t().contiguous().t(), w.t().contiguous().t())):
        xs, ws = xs.detach().requires_grad_(), ws.detach().requires_grad_()
        bs = b.detach().requires_grad_()
        loss = linear_cross_entropy(xs, ws, bs, t)
        got = [loss, *torch.autograd.grad(loss, [xs, ws, bs])]
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    cube = x.view(3, 4, 5, 64).detach().requires_grad_()
    rows = linear_cross_entropy(cube, w, b, t.view(3, 4, 5), reduction="none")
    assert rows.shape == (3, 4, 5)
    rows.sum().backward()
    assert torch.equal(cube.grad.view(60, 64), _check(x, w, b, t, reduction="sum")[1][0])


def test_only_what_is_needed(dev):
    from vtpack_amd.layers import linear_cross_entropy
    x, w, b, t = _operands(dev, 50, 60, 64, torch.float32)
    full = _check(x, w, b, t)[1]
    for i in range(3):
        leaves = [v.detach().requires_grad_(k == i) for k, v in enumerate((x, w, b))]
        linear_cross_entropy(*leaves, t).backward()
        assert torch.equal(leaves[i].grad, full[i])


def test_result_may_be_changed_in_place(dev):
    from vtpack_amd.layers import linear_cross_entropy
    x, w, b, t = _operands(dev, 50, 60, 64, torch.float32)
    want = _check(x, w, b, t)[1][0]
    x = x.detach().requires_grad_()
    loss = linear_cross_entropy(x, w, b, t)
    loss /= 2
    loss.backward()
    assert torch.equal(x.grad, want / 2)


def test_against_differences(dev):
    """The gradient of the loss against its differences along random directions: fp32 losses of about 5, steps of 1e-2."""
    from vtpack_amd.layers import linear_cross_entropy
    x, w, b, t = _operands(dev, 40, 50, 64, torch.float32, left_out=0.2)
    got = _check(x, w, b, t, smoothing=0.2)[1]
    g = torch.Generator().manual_seed(1)
    for i in range(3):
        v = torch.randn((x, w, b)[i].shape, generator=g).to(dev)
        v /= v.norm()
        at = [[p + s * 1e-2 * v if k == i else p for k, p in enumerate((x, w, b))] for s in (1, -1)]
        up, down = (float(_reference(*a, t, 0.2)[0].sum() / int((t >= 0).sum())) for a in at)
        # a difference of step h is off by h^2 / 6 of the third derivative, which is below 1 here
        assert abs((up - down) / 2e-2 - float((got[i] * v).sum())) <= 1e-4 / 6 + 1e-5


@pytest.mark.parametrize("dtype", DTYPES)
def test_same_bits_on_another_stream_and_in_a_graph(dev, dtype):
    from vtpack_amd import ops
    x, w, b, t = _operands(dev, 700, 1500, 192, dtype, left_out=0.1)
    g = torch.ones((), device=dev)

    def run():
        loss, stats, laid_out = ops.cross_entropy(x, w, b, t, -100, 0.1, "mean")
        return [loss, *ops.cross_entropy_backward(x, w, b, t, stats, laid_out, g, -100, 0.1)]

    want = [v.clone() for v in run()]
    assert all(torch.equal(p, q) for p, q in zip(run(), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for k in range(3):
        x.copy_(x.roll(1, 0))
        t.copy_(t.roll(1, 0))
        graph.replay()
        torch.cuda.synchronize()
        again = run()
        assert all(torch.equal(p, q) for p, q in zip(out, again)), k


def test_refusals(dev):
    from vtpack_amd.layers import linear_cross_entropy
    x, w, b, t = _operands(dev, 8, 9, 16, torch.float32)
    for args, kw, error in [((x, w.bfloat16(), b, t), {}, TypeError), ((x.half(), w.half(), b.half(), t), {}, TypeError),
                            ((x, w, b, t.int()), {}, TypeError), ((x, w, b, t.cpu()), {}, RuntimeError), ((x, w[:, :8], b, t), {}, ValueError),
                            ((x, w, b[:3], t), {}, ValueError), ((x, w, b, t[:3]), {}, ValueError), ((x, w, b, t), {"reduction": "max"}, ValueError),
                            ((x, w, b, t), {"label_smoothing": 1.5}, ValueError), ((x, w[:0], b[:0], t), {}, ValueError)]:
        with pytest.raises(error):
            linear_cross_entropy(*args, **kw)
    with pytest.raises(RuntimeError):                    # gradients of the gradients are not to be had
        x = x.requires_grad_()
        dx, = torch.autograd.grad(linear_cross_entropy(x, w, b, t), x, create_graph=True)
        dx.sum().backward()


LARGE, MIDDLE, SMALL, SPLIT = "Shape<2, 4, 4, 2, 64, 2, 1>", "Shape<2, 2, 4, 2, 64, 3, 1>", "Shape<1, 1, 2, 2, 64, 3, 1>", "Shape<2, 2, 4, 2, 32, 2, 3>"


@pytest.mark.parametrize("dtype,rows,classes,width,logits,grads", [
    (torch.bfloat16, 4097, 16385, 1032, LARGE, LARGE), (torch.bfloat16, 8193, 4097, 1024, LARGE, LARGE),
    (torch.bfloat16, 1000, 16640, 260, "Shape<2, 4, 2, 2, 32, 3, 1>", LARGE), (torch.bfloat16, 2049, 16385, 136, "Shape<2, 4, 2, 2, 32, 3, 1>", MIDDLE),
    (torch.bfloat16, 2000, 2000, 1027, "Shape<1, 1, 2, 2, 64, 6, 1>", MIDDLE), (torch.bfloat16, 1025, 8191, 72, "Shape<2, 4, 2, 2, 32, 3, 1>", SMALL),
    (torch.bfloat16, 64, 16384, 64, "Shape<1, 2, 2, 2, 64, 3, 1>", SMALL), (torch.float32, 2049, 16385, 136, SPLIT, SPLIT),
    (torch.float32, 257, 32769, 130, SPLIT, SPLIT), (torch.float32, 64, 16384, 64, "Shape<1, 2, 2, 2, 32, 3, 3>", "Shape<1, 1, 2, 2, 32, 3, 3>"),
    (torch.float32, 1000, 300, 70, "Shape<1, 1, 2, 2, 32, 4, 3>", "Shape<1, 1, 2, 2, 32, 3, 3>")])
def test_shapes_of_tiles(dev, dtype, rows, classes, width, logits, grads):
    """Every shape of the product, one row, class or feature around its tiles and slabs, with sums cut and classes in pieces."""
    from vtpack_amd import _lib, ops
    x, w, b, t = _operands(dev, rows, classes, width, dtype, left_out=0.1)
    loss, stats, laid_out = ops.cross_entropy(x, w, b, t)
    assert any(f"cross_entropy_tiles_kernel<vtdge::{logits}, false>" in _lib.last_kernel(k) for k in range(3))
    one = torch.ones((), device=dev)
    again = ops.cross_entropy_backward(x, w, b, t, stats, None, one)
    used = [_lib.last_kernel(k) for k in range(3)]
    assert any(f"cross_entropy_grad_kernel<vtdge::{grads} >" in n for n in used) and any(f"cross_entropy_d_kernel<vtdge::{logits} >" in n for n in used)
    kept = ops.cross_entropy_backward(x, w, b, t, stats, laid_out, one)
    assert (dtype == torch.float32) == any("cross_entropy_d_kept_kernel" in _lib.last_kernel(k) for k in range(3))
    assert all(torch.equal(p, q) for p, q in zip(again, kept))
    _check(x, w, b, t, smoothing=0.1)


@pytest.mark.parametrize("dtype,width", [(torch.float32, 64), (torch.bfloat16, 72), (torch.bfloat16, 128)])
def test_operands_kept_or_laid_out_again(dev, dtype, width):
    """What the forward call leaves for the gradients is what they would lay out themselves; and they leave it as it is."""
    from vtpack_amd import ops
    x, w, b, t = _operands(dev, 300, 500, width, dtype, left_out=0.2)
    x[t < 0] = float("nan")
    one = torch.ones((), device=dev)
    loss, stats, laid_out = ops.cross_entropy(x, w, b, t)
    assert (laid_out is not None) == (dtype == torch.float32 or width % 64 != 0)
    want = ops.cross_entropy_backward(x, w, b, t, stats, None, one)
    for _ in range(2):
        got = ops.cross_entropy_backward(x, w, b, t, stats, laid_out, one)
        assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("dtype", DTYPES)
def test_backward_twice_and_a_weight_used_twice(dev, dtype):
    from vtpack_amd.layers import linear_cross_entropy
    x, w, b, t = _operands(dev, 130, 200, 96, dtype)
    x2, _, _, t2 = _operands(dev, 77, 200, 96, dtype, seed=3)
    one, two = _check(x, w, b, t)[1][1], _check(x2, w, b, t2)[1][1]
    leaf = w.detach().requires_grad_()
    loss = linear_cross_entropy(x, leaf, b, t)
    again = [torch.autograd.grad(loss, leaf, retain_graph=True)[0] for _ in range(2)]
    assert torch.equal(again[0], one) and torch.equal(again[1], one)
    (loss + linear_cross_entropy(x2, leaf, b, t2)).backward()
    assert torch.equal(leaf.grad, one + two)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_captured_training_pass(dev, dtype):
    """Forward and backward through autograd in one graph, on leaves of its own, replayed over new data beside eager calls."""
    from vtpack_amd.layers import linear_cross_entropy
    x, w, b, t = _operands(dev, 520, 900, 136, dtype, left_out=0.1)
    leaves = [v.clone().requires_grad_() for v in (x, w, b)]
    targets = t.clone()

    def run(leaves, t):
        loss = linear_cross_entropy(*leaves, t, label_smoothing=0.1)
        return [loss.detach(), *torch.autograd.grad(loss, leaves)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(leaves, targets)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(leaves, targets)
    for k in range(4):
        x, t = x.roll(1, 0), t.roll(1, 0)
        with torch.no_grad():
            leaves[0].copy_(x)
            leaves[1].mul_(0.9)
        targets.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        want = run([v.detach().clone().requires_grad_() for v in leaves], t)
        assert all(torch.equal(p, q) for p, q in zip(out, want)), k


def test_two_calls_at_once(dev):
    """Two threads, each on a stream of its own, over calls of several sizes."""
    import threading
    from vtpack_amd.layers import linear_cross_entropy
    sizes = [(300, 500, 96), (1021, 1000, 192), (64, 17000, 64)]
    data = [[_operands(dev, *s, dtype) for s in sizes] for dtype in DTYPES]

    def run(sets):
        out = []
        for x, w, b, t in sets:
            leaves = [v.detach().requires_grad_() for v in (x, w, b)]
            loss = linear_cross_entropy(*leaves, t)
            out += [loss.detach(), *torch.autograd.grad(loss, leaves)]
        return out

    want = [run(sets) for sets in data]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    got[i] = run(data[i])
                torch.cuda.current_stream().synchronize()
        except Exception as e:
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not errors
    for p, q in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(p, q))


def test_saved_operands(dev):
    """Operands changed in place before the backward pass are noticed; a checkpointed loss is worked out again."""
    from torch.utils.checkpoint import checkpoint
    from vtpack_amd.layers import linear_cross_entropy
    x, w, b, t = _operands(dev, 50, 60, 64, torch.float32)
    want = _check(x, w, b, t)[1]
    for change in range(3):
        operands = [v.clone() for v in (x, w, t)]
        leaf = b.detach().requires_grad_()
        loss = linear_cross_entropy(operands[0], operands[1], leaf, operands[2])
        operands[change].zero_()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    leaves = [v.detach().requires_grad_() for v in (x, w, b)]
    checkpoint(linear_cross_entropy, *leaves, t, use_reentrant=False).backward()
    assert all(torch.equal(v.grad, g) for v, g in zip(leaves, want))


def test_no_graph_without_gradients(dev):
    from vtpack_amd.layers import gate_balance, linear_cross_entropy
    x, w, b, t = _operands(dev, 50, 60, 64, torch.float32)
    assert not linear_cross_entropy(x, w, b, t).requires_grad
    with torch.no_grad():
        assert not linear_cross_entropy(x.requires_grad_(), w, b, t).requires_grad
        assert not gate_balance(x)[0].requires_grad
    loss, counts = gate_balance(x)
    assert loss.requires_grad and not counts.requires_grad


def test_a_graph_is_used_once(dev):
    """A second backward pass without retain_graph is refused, and what the first one read is given back."""
    from vtpack_amd.layers import gate_balance, linear_cross_entropy
    x, w, b, t = _operands(dev, 50, 60, 64, torch.float32)
    x.requires_grad_()
    for loss in (linear_cross_entropy(x, w, b, t), gate_balance(x)[0]):
        assert loss.grad_fn.name() in ("LinearCrossEntropyBackward", "GateBalanceBackward")
        loss.backward()
        with pytest.raises(RuntimeError, match="second time"):
            loss.backward()
    both = linear_cross_entropy(x, w, b, t, reduction="none")
    used = torch.cuda.memory_allocated()
    both.sum().backward()
    del both
    x.grad = None
    assert torch.cuda.memory_allocated() < used


def test_forward_mode_is_refused(dev):
    from torch.autograd import forward_ad
    from vtpack_amd.layers import gate_balance, linear_cross_entropy
    x, w, b, t = _operands(dev, 50, 60, 64, torch.float32)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: linear_cross_entropy(dual, w, b, t), lambda: gate_balance(dual)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()


@pytest.mark.parametrize("which", ["x", "weight"])
def test_one_operand_is_laid_out(dev, which):
    """bf16 operands of which one lies as the kernels read it and the other does not; rows left out hold NaN."""
    from vtpack_amd import ops
    from vtpack_amd.layers import linear_cross_entropy
    x, w, b, t = _operands(dev, 300, 500, 128, torch.bfloat16, left_out=0.2)
    x[t < 0] = float("nan")
    want = [linear_cross_entropy(x, w, b, t), *_check(x, w, b, t)[1]]
    place = torch.zeros(((300 if which == "x" else 500) * 128 + 1,), dtype=torch.bfloat16, device=dev)
    place[1:] = (x if which == "x" else w).reshape(-1)
    moved = place[1:].view(-1, 128)
    xs, ws = (moved, w) if which == "x" else (x, moved)
    loss, stats, laid_out = ops.cross_entropy(xs, ws, b, t)
    assert laid_out is None and torch.equal(loss, want[0])
    got = ops.cross_entropy_backward(xs, ws, b, t, stats, None, torch.ones((), device=dev))
    assert all(torch.equal(p, q) for p, q in zip(got, want[1:]))


def test_tracing_is_refused(dev):
    """On every way to a launch: operands that are taken as they are, and those that are brought into form."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from vtpack_amd.layers import gate_balance, linear_cross_entropy
    x, w, b, t = _operands(dev, 50, 60, 64, torch.float32)
    for call in (lambda x: linear_cross_entropy(x, w, b, t), lambda x: linear_cross_entropy(x.t().contiguous().t(), w, b, t), lambda x: gate_balance(x)[0],
                 lambda x: gate_balance(x, indices=t)[0]):
        want = call(x)
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(call, (x,))
        for mode in ("real", "fake"):
            with pytest.raises(RuntimeError, match="cannot be traced"):
                make_fx(call, tracing_mode=mode, _allow_non_fake_inputs=True)(x)
        assert torch.equal(call(x), want)


def test_widths_beyond_32_bits_are_refused(dev):
    """Not taken for their lower 32 bits."""
    from vtpack_amd.layers import linear_cross_entropy
    row = torch.empty((1, (1 << 32) + 64), dtype=torch.bfloat16, device=dev)
    with pytest.raises(RuntimeError, match="rows"):
        linear_cross_entropy(row, row, None, torch.zeros(1, dtype=torch.int64, device=dev))


def test_fp32_up_to_the_largest_number(dev):
    """Finite features and weights next to the largest fp32 number, which bf16 would round to infinity: losses of 1e38, bounded by
    half steps of the logits as all are."""
    from vtpack_amd.layers import linear_cross_entropy
    x, w, b, t = _operands(dev, 40, 150, 64, torch.float32)
    x[3, 0], x[17, 5] = 3.4e38, -3.4028e38
    w[:, 0] *= 0.3
    w[:, 5] *= 0.3
    want, _, d, grads = _reference(x, w, b, t)
    leaves = [v.detach().requires_grad_() for v in (x, w, b)]
    got = linear_cross_entropy(*leaves, t, reduction="none")
    tol = _tolerance(x, w)
    assert ((got.double() - want).abs() <= tol * (16 + want.abs())).all()
    for g, r in zip(torch.autograd.grad(got.sum() / 40, leaves), grads):
        _near(g, r, tol, 1e-30)
    # the largest weights
    x, w, b, t = _operands(dev, 40, 150, 64, torch.float32, seed=1)
    w[7, 3], w[100, 3] = 3.4e38, -3.4e38
    x[:, 3] *= 0.05
    want = _reference(x, w, b, t)[0]
    got = linear_cross_entropy(x, w, b, t, reduction="none")
    assert torch.isfinite(got).all() and ((got.double() - want).abs() <= tol * (16 + want.abs())).all()


@pytest.mark.parametrize("kept", [True, False])
def test_row_weights_up_to_the_largest_number(dev, kept):
    """d of a row whose loss is weighted by 3.4e38, an fp32 operand like any other."""
    from vtpack_amd import ops
    x, w, b, t = _operands(dev, 40, 150, 64, torch.float32)
    x, w, b, t = x[:2], torch.zeros_like(w), torch.zeros_like(b), t[:2]
    b[t[0]] = -200.0                                       # its own class has no share: d is -1 there
    x[:] = x.clamp(-0.5, 0.5)
    grad = torch.tensor([3.4e38, 1.0], device=dev)
    loss, stats, laid_out = ops.cross_entropy(x, w, b, t, reduction="none")
    dx, dw, db = ops.cross_entropy_backward(x, w, b, t, stats, laid_out if kept else None, grad, reduction="none")
    want = _reference(x, w, b, t, weights=grad)[3]
    for g, r in zip((dx, dw, db), want):
        _near(g, r, _tolerance(x, w), 1e-30)


def test_fp32_next_to_the_smallest_numbers(dev):
    """Features below 2^-110 are off by 2^-134 at most, a logit by that times its weights, a loss by twice a logit."""
    from vtpack_amd.layers import linear_cross_entropy
    x, w, b, t = _operands(dev, 40, 150, 64, torch.float32)
    x, w = x * 2.0 ** -118, w * 2.0 ** 118
    want = _reference(x, w, b, t)[0]
    got = linear_cross_entropy(x, w, b, t, reduction="none")
    z = x.double() @ w.double().t()
    bound = 2 * 2.0 ** -134 * float(w.double().abs().sum(1).max()) + _tolerance(x, w) * (1 + float(z.abs().max()))
    assert float((got.double() - want).abs().max()) <= bound


def test_hooks_see_what_is_kept_for_the_gradients(dev):
    """Logits and laid out operands go where saved tensors go: a checkpointed loss keeps none of them, an offloaded one has them on the
    host."""
    from torch.autograd.graph import saved_tensors_hooks
    from torch.utils.checkpoint import checkpoint
    from vtpack_amd.layers import gate_balance, linear_cross_entropy
    x, w, b, t = _operands(dev, 1024, 8192, 64, torch.float32)            # logits of 32 MB
    leaves = [v.detach().requires_grad_() for v in (x, w, b)]
    want = torch.autograd.grad(linear_cross_entropy(*leaves, t), leaves)
    torch.cuda.synchronize()
    for way in ("checkpoint", "host"):
        before = torch.cuda.memory_allocated()
        if way == "checkpoint":
            loss = checkpoint(linear_cross_entropy, *leaves, t, use_reentrant=False)
        else:
            sizes = []
            with saved_tensors_hooks(lambda v: sizes.append(v.nbytes) or v.cpu(), lambda v: v.to(dev)):
                loss = linear_cross_entropy(*leaves, t)
            assert max(sizes) >= 32 << 20
        assert torch.cuda.memory_allocated() - before < 1 << 20
        got = torch.autograd.grad(loss, leaves)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    sizes = []
    with saved_tensors_hooks(lambda v: sizes.append(v.nbytes) or v.cpu(), lambda v: v.to(dev)):
        loss, _ = gate_balance(leaves[0])
    assert len(sizes) == 2
    loss.backward()


@pytest.mark.parametrize("back", ["cpu", "short", "type", "wide"])
def test_hooks_that_bring_back_something_else(dev, back):
    """What unpacking hooks return is looked at before a kernel reads it."""
    from torch.autograd.graph import saved_tensors_hooks
    from vtpack_amd.layers import gate_balance, linear_cross_entropy
    x, w, b, t = _operands(dev, 50, 60, 64, torch.float32)
    leaves = [v.detach().requires_grad_() for v in (x, w, b)]
    change = {"cpu": lambda v: v.cpu(), "short": lambda v: v[:len(v) // 2], "type": lambda v: v.half() if v.is_floating_point() else v.int(),
              "wide": lambda v: torch.stack([v, v], -1)[..., 0]}[back]
    for which in range(6):
        seen = []

        def unpack(v):
            seen.append(1)
            return change(v) if len(seen) == which + 1 else v

        with saved_tensors_hooks(lambda v: v, unpack):
            loss = linear_cross_entropy(*leaves, t)
        with pytest.raises(RuntimeError, match="^linear_cross_entropy: "):
            torch.autograd.grad(loss, leaves)
        assert len(seen) == 6
    with saved_tensors_hooks(lambda v: v, change):
        loss, _ = gate_balance(leaves[0], mask=t > 3)
    with pytest.raises(RuntimeError, match="^gate_balance: "):
        loss.backward()


@pytest.mark.parametrize("rows,classes,width,kept", [(8192, 8192, 64, True), (8192, 9001, 72, False), (16411, 4000, 40, True), (60000, 2100, 64, False)])
def test_fp32_gradients_over_pieces(dev, rows, classes, width, kept):
    """Classes in more than one piece, the last of them shorter, with d from kept logits and worked out again."""
    from vtpack_amd import _lib, ops
    x, w, b, t = _operands(dev, rows, classes, width, torch.float32, left_out=0.1)
    one = torch.ones((), device=dev)
    loss, stats, laid_out = ops.cross_entropy(x, w, b, t)
    again = ops.cross_entropy_backward(x, w, b, t, stats, None, one)
    pieces = [_lib.last_kernel(k) for k in range(8)]
    assert sum("cross_entropy_grad_kernel" in n for n in pieces) >= 2 and sum("cross_entropy_d_kernel" in n for n in pieces) >= 2
    if laid_out is not None:
        got = ops.cross_entropy_backward(x, w, b, t, stats, laid_out, one)
        used = [_lib.last_kernel(k) for k in range(6)]
        assert (sum("cross_entropy_d_kept_kernel" in n for n in used) >= 2) == kept
        assert all(torch.equal(p, q) for p, q in zip(again, got))
    _check(x, w, b, t, smoothing=0.1)
