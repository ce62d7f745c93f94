"""The balance loss of router gates, its counts and its gradient, against the formula in float64.

Bounds: probabilities are a few fp32 roundings off (exp of a difference d is off by |d| half steps besides), their sums run in fp32 over the
tokens of 16 lanes and in double from there: 2^-24 (16 + largest difference) of the 2-norm; bf16 gradients half a step more, 2^-8 of each."""
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16]


def _gate(dev, tokens, E, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + 1000 * E + tokens)
    return (torch.randn(tokens, E, generator=g) * 1.5 + torch.randn(E, generator=g)).to(dev, dtype)


def _reference(gate, top_k, mask=None, indices=None):
    """In float64 on the CPU -> loss, counts, gradient."""
    z = gate.detach().cpu().double()
    T, E = z.shape
    live = torch.ones(T, dtype=torch.bool) if mask is None else mask.cpu().clone()
    live &= ~(z == float("-inf")).all(1)
    if indices is None:
        key = torch.where(z.isnan(), torch.full_like(z, 1e300), z)          # a stable sort leaves equals in their order
        indices = torch.sort(-key, dim=1, stable=True).indices[:, :top_k]
    else:
        indices = indices.cpu()
    chosen = indices[live].reshape(-1)
    counts = torch.bincount(chosen[(chosen >= 0) & (chosen < E)], minlength=E)
    n = max(1, int(live.sum()))
    p = torch.softmax(z, 1)
    f = counts.double() / (n * indices.shape[1])
    loss = E * float((f * p[live].sum(0) / n).sum())
    grad = torch.zeros_like(z)
    grad[live] = (E / n) * p[live] * (f - (p[live] @ f)[:, None])
    return loss, counts, grad


def _check(gate, top_k=1, mask=None, indices=None):
    from vtpack_amd.layers import gate_balance
    gate = gate.detach().requires_grad_()
    loss, counts = gate_balance(gate, indices, top_k, mask)
    want, n, grad = _reference(gate.reshape(-1, gate.shape[-1]), top_k, None if mask is None else mask.reshape(-1),
                               None if indices is None else indices.reshape(gate.numel() // gate.shape[-1], -1))
    assert counts.dtype == torch.int64 and torch.equal(counts.cpu(), n)
    z = gate.detach().double()
    z = z[torch.isfinite(z) & (z > -1e4)]                # what is shut out by the lowest value has no probability
    tol = HALF * (16 + (float(z.max() - z.min()) if z.numel() else 0))
    assert abs(float(loss) - want) <= tol * abs(want)
    got, = torch.autograd.grad(loss, gate, torch.tensor(2.0, device=gate.device))
    assert got.dtype == gate.dtype and got.shape == gate.shape
    err = (got.reshape(grad.shape).cpu().double() - 2 * grad).norm()
    # (f_j - sum f p) cancels where the choices are even: the bound is of its terms
    size = 2 * float((_terms(gate, n, top_k if indices is None else indices.shape[-1], grad)).norm())
    assert float(err) <= tol * size + (2.0 ** -8 * 2 * float(grad.norm()) if gate.dtype == torch.bfloat16 else 0) + 1e-30
    return loss, counts, got


def _terms(gate, counts, k, grad):
    z = gate.detach().reshape(grad.shape).cpu().double()
    p = torch.softmax(z, 1).nan_to_num(0)
    total = max(1, int(counts.sum()))
    f = counts.double() / total
    n = max(1, total // k)
    return (z.shape[1] / n) * p * (f + (p @ f)[:, None])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("E", [1, 2, 3, 15, 16, 17, 32, 33, 64, 65, 128, 130, 160, 192, 193, 256, 257, 511, 512])
def test_experts(dev, dtype, E):
    for tokens, k in ((1, 1), (37, min(E, 2)), (300, min(E, 8))):
        _check(_gate(dev, tokens, E, dtype), k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens", [15, 16, 17, 255, 256, 257, 8191, 8192, 8193, 20011])
def test_tokens(dev, dtype, tokens):
    g = torch.Generator().manual_seed(tokens)
    mask = (torch.rand(tokens, generator=g) < 0.6).to(dev)
    _check(_gate(dev, tokens, 3, dtype), 1)
    _check(_gate(dev, tokens, 40, dtype), 5, mask)


@pytest.mark.parametrize("dtype", DTYPES)
def test_equal_logits_go_to_the_lowest(dev, dtype):
    gate = torch.zeros(400, 20, device=dev, dtype=dtype)
    gate[::2, 0] = -0.0
    loss, counts, _ = _check(gate, 3)
    assert counts.tolist() == [400, 400, 400] + [0] * 17
    _check(torch.randint(-2, 3, (500, 33), generator=torch.Generator().manual_seed(0)).to(dev, dtype), 7)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("E,k", [(3, 1), (40, 3), (160, 6)])
def test_not_a_number_is_the_largest(dev, dtype, E, k):
    """NaN of every kind are one value above infinity: the lowest experts with one are chosen first."""
    from vtpack_amd.layers import gate_balance
    gate = _gate(dev, 64, E, dtype)
    bits = gate.view(torch.int16 if dtype == torch.bfloat16 else torch.int32)
    some, all_ones = (0x7fc0, -1) if dtype == torch.bfloat16 else (0x7fc00000, -1)
    g = torch.Generator().manual_seed(4)
    for kind in (some, all_ones, 0x7fff if dtype == torch.bfloat16 else 0x7fffffff):
        for t, e in zip(torch.randint(0, 64, (30,), generator=g).tolist(), torch.randint(0, E, (30,), generator=g).tolist()):
            bits[t, e] = kind
    bits[0, 0], bits[1, 0], bits[2, E - 1] = all_ones, some, all_ones
    gate[3, 1] = float("inf")
    key = torch.where(gate.isnan(), torch.full_like(gate, float("inf")).double() , gate.double().clamp(max=1e300)).cpu()
    chosen = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :k]
    want = torch.bincount(chosen.reshape(-1), minlength=E)
    assert torch.equal(gate_balance(gate, top_k=k)[1].cpu(), want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_masks(dev, dtype):
    """Experts masked by -inf or by the type's lowest value, tokens whose experts are all masked, what is masked not finite, and
    nothing left at all."""
    from vtpack_amd.layers import gate_balance
    gate = _gate(dev, 300, 24, dtype)
    gate[:, 5] = float("-inf")
    gate[::3, 7] = torch.finfo(dtype).min
    gate[10] = float("-inf")
    mask = torch.ones(300, dtype=torch.bool, device=dev)
    mask[20:50] = False
    gate[20:30] = float("nan")
    gate[30:40] = float("inf")
    got = _check(gate, 2, mask)[2]
    assert not got[20:50].any() and not got[10].any() and not got[:, 5].any()
    gate = gate.detach().requires_grad_()
    loss, counts = gate_balance(gate, mask=torch.zeros_like(mask))
    assert float(loss) == 0 and not counts.any() and not torch.autograd.grad(loss, gate)[0].any()
    loss, counts = gate_balance(gate[:0])
    assert float(loss) == 0 and counts.tolist() == [0] * 24
    loss.backward()
    # a NaN that counts shows
    loss, counts = gate_balance(gate.detach()[15:35])
    assert torch.isnan(loss)


@pytest.mark.parametrize("dtype", DTYPES)
def test_choices_made_elsewhere(dev, dtype):
    gate = _gate(dev, 600, 9, dtype).view(20, 5, 6, 9)
    g = torch.Generator().manual_seed(3)
    one = torch.randint(0, 9, (20, 5, 6), generator=g).to(dev)
    loss, counts, _ = _check(gate, indices=one.unsqueeze(-1))
    from vtpack_amd.layers import gate_balance
    again = gate_balance(gate, indices=one)
    assert torch.equal(again[0], loss) and torch.equal(again[1], counts)
    several = torch.randint(-1, 10, (20, 5, 6, 19), generator=g).to(dev)      # those that are no expert are not counted
    mask = (torch.rand(20, 5, 6, generator=g) < 0.7).to(dev)
    loss, counts = gate_balance(gate, several, mask=mask)
    want, n, _ = _reference(gate.reshape(600, 9), 0, mask.reshape(-1), several.reshape(600, 19))
    assert torch.equal(counts.cpu(), n) and abs(float(loss) - want) <= HALF * 40 * want


def test_strides_streams_and_graphs(dev):
    from vtpack_amd import ops
    from vtpack_amd.layers import gate_balance
    wide = _gate(dev, 5000, 60, torch.float32)
    want = _check(wide[:, 7:27].contiguous(), 2)
    got = _check(wide[:, 7:27], 2)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    gate = wide[:, 7:27].contiguous()
    one = torch.ones((), device=dev)

    def run():
        loss, counts, share = ops.gate_balance(gate, None, None, 2)
        return loss, counts, ops.gate_balance_backward(gate, None, share, one)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run()
    side.synchronize()
    assert torch.equal(other[0], want[0]) and torch.equal(other[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for _ in range(3):
        gate.copy_(gate.roll(3, 1) * 1.1)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, run()))
    loss, _ = gate_balance(gate.requires_grad_())
    loss *= 3.0                                          # results may be changed in place
    loss.backward()
    assert gate.grad.abs().sum() > 0


def test_refusals(dev):
    from vtpack_amd.layers import gate_balance
    gate = _gate(dev, 10, 6, torch.float32)
    idx = torch.zeros(10, dtype=torch.int64, device=dev)
    for args, kw, error in [((gate.half(),), {}, TypeError), ((gate,), {"top_k": 0}, ValueError), ((gate,), {"top_k": 7}, ValueError),
                            ((gate.new_zeros(4, 513),), {}, ValueError), ((gate, idx.int()), {}, TypeError), ((gate, idx[:4]), {}, ValueError),
                            ((gate,), {"mask": idx}, TypeError), ((gate,), {"mask": idx.bool()[:3]}, ValueError), ((gate, idx.cpu()), {}, RuntimeError),
                            ((gate.new_zeros(4, 0),), {}, ValueError)]:
        with pytest.raises(error):
            gate_balance(*args, **kw)
