"""The AdamW step against the formula in float64: sizes around a block and a chunk, both moment formats, strides, missing
gradients, graphs, state dicts.

Bounds: a weight takes its own rounding, that of lr wd p and some ten of its update, each half a step: 2^-24 (3 |p| + 16 |update|),
bf16 a rounding of the weight more: its
neighbours between 1 and 2 are 2^-7 apart, so that one is off by 2^-8 of the value at most.  The fp32 moments take three roundings of terms that may cancel.  The eight-bit ones are made
by operations that are each rounded once, as the reference repeats: the same codes and scales."""
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16]
SIZES = [1, 3, 4, 255, 256, 257, 1000, 4095, 4096, 4097, 12289]
LR, BETAS, EPS, DECAY = 1e-3, (0.9, 0.999), 1e-8, 0.05


def _tensors(dev, shapes, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g) * torch.exp(torch.randn(s, generator=g)) * scale).to(dev, dtype) for s in shapes]


def _f32(t):
    return t.float().double()


def _hash(n, step):
    low = 0xffffffff
    h = (torch.arange(n) * 0x6a09e667 + ((step * 0xbb67ae85) & low)) & low
    h = ((h ^ (h >> 16)) * 0x3c6ef373) & low
    h = ((h ^ (h >> 15)) * 0xa54ff53b) & low
    return h ^ (h >> 16)


def _codes(flat, step, first):
    """-> values of the codes (without the scale), scales: float64 [n], [ceil(n / 256)]."""
    mantissa, small, top = (3, 2.0 ** -6, 448.0) if first else (2, 2.0 ** -14, 57344.0)
    n = flat.numel()
    b = torch.cat([flat, flat.new_zeros(-n % 256)]).view(-1, 256)
    most = b.abs().amax(1, keepdim=True)
    some = most >= 2.0 ** -100
    scale = torch.where(some, _f32(most * _f32(torch.tensor(1 / top, dtype=torch.float64))), torch.zeros_like(most))
    x = torch.where(some, _f32(b.abs() * _f32(top / most.clamp(min=2.0 ** -100))), torch.zeros_like(b)).clamp(max=top)
    h = _hash(b.numel(), step).view_as(b)
    share = ((h & 0xffff) if first else (h >> 16)).double() / 65536
    unit = torch.exp2(torch.floor(torch.log2(x.clamp(min=small)) + 1e-12) - mantissa)
    q = torch.floor(torch.where(x < small, _f32(x + small) - small, x) / unit + share) * unit
    if not first:
        q = torch.where((x > 0) & (q == 0), torch.full_like(q, 2.0 ** -16), q)
    return (q * b.sign()).view(-1)[:n], scale.view(-1)


class _Reference:
    """One weight, in float64 on the CPU, flat in the order of memory."""

    def __init__(self, p, bits, steps=0):
        self.bits, self.t, n = bits, steps, p.numel()
        self.p = p.detach().cpu().double().reshape(-1)
        self.m, self.v = torch.zeros(n, dtype=torch.float64), torch.zeros(n, dtype=torch.float64)
        self.ms = self.vs = torch.zeros(-(-n // 256), dtype=torch.float64)

    def step(self, g, lr=LR):
        self.t += 1
        g = g.detach().cpu().double().reshape(-1)
        b1, b2 = BETAS
        if self.bits == 8:
            n = g.numel()
            m, v = (_f32(c * s.repeat_interleave(256)[:n]) for c, s in ((self.m, self.ms), (self.v, self.vs)))
            f = [float(torch.tensor(x, dtype=torch.float32)) for x in (b1, 1 - b1, b2, 1 - b2)]
            m = _f32(_f32(m * f[0]) + _f32(g * f[1]))
            v = _f32(_f32(v * f[2]) + _f32(_f32(g * f[3]) * g))
        else:
            m, v = b1 * self.m + (1 - b1) * g, b2 * self.v + (1 - b2) * g * g
        self.update = lr / (1 - b1 ** self.t) * m / ((v / (1 - b2 ** self.t)).sqrt() + EPS)
        self.p = self.p * (1 - lr * DECAY) - self.update
        if self.bits == 8:
            (self.m, self.ms), (self.v, self.vs) = _codes(m, self.t, True), _codes(v, self.t, False)
        else:
            self.m, self.v = m, v

    def check(self, p, state, steps=1):
        got = p.detach().cpu().double().reshape(-1)
        e = steps * HALF * (3 * self.p.abs() + 16 * self.update.abs() + 16 * LR)
        if p.dtype == torch.bfloat16:
            e = e + 2.0 ** -8 * self.p.abs()
        over = float(((got - self.p).abs() / e).max())
        assert over <= 1
        m, v = (state[k].detach().cpu().double().reshape(-1) if state[k].dtype == torch.float32 else state[k].detach().float().cpu().double().reshape(-1)
                for k in ("exp_avg", "exp_avg_sq"))
        if self.bits == 8:
            assert torch.equal(m, self.m) and torch.equal(v, self.v)
            assert torch.equal(state["exp_avg_scale"].cpu().double(), self.ms) and torch.equal(state["exp_avg_sq_scale"].cpu().double(), self.vs)
        else:
            # three roundings of each step's terms, none larger than the gradients seen
            top = steps * 4 * HALF
            assert float((m - self.m).norm()) <= top * max(float(self.m.norm()), 1e-30) * 4
            assert float((v - self.v).norm()) <= top * max(float(self.v.norm()), 1e-30)
        self.p = got                                  # weights are compared step by step
        if self.bits == 32:
            self.m, self.v = m, v


def _optimizer(params, bits, **kw):
    from vtpack_amd.optim import AdamW
    return AdamW(params, lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, state_bits=bits, **kw)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", DTYPES)
def test_sizes(dev, dtype, bits):
    shapes = [(n,) for n in SIZES] + [(0,), (3, 0), (7, 11, 13), ()]
    params = [torch.nn.Parameter(t) for t in _tensors(dev, shapes, dtype, 1)]
    refs = [_Reference(p, bits) for p in params]
    opt = _optimizer(params, bits)
    for k in range(4):
        for p, g in zip(params, _tensors(dev, shapes, dtype, 10 + k, 1e-3)):
            p.grad = g
        opt.step()
        for p, r in zip(params, refs):
            if p.numel():
                r.step(p.grad)
                r.check(p, opt.state[p])
    assert opt.param_groups[0]["step"] == 4


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors(dev, bits):
    """More than one launch's table holds, in two types."""
    from vtpack_amd import _lib
    shapes = [(1 + 37 * i % 500,) for i in range(230)]
    params = [torch.nn.Parameter(t) for t in _tensors(dev, shapes, torch.float32, 2) + _tensors(dev, shapes, torch.bfloat16, 3)]
    refs = [_Reference(p, bits) for p in params]
    opt = _optimizer(params, bits)
    for p, g in zip(params, _tensors(dev, shapes, torch.float32, 4, 1e-3) + _tensors(dev, shapes, torch.bfloat16, 5, 1e-3)):
        p.grad = g
    opt.step()
    assert f"adamw_kernel<unsigned short, {bits}, false>" in _lib.last_kernel()
    for p, r in zip(params, refs):
        r.step(p.grad)
        r.check(p, opt.state[p])


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", DTYPES)
def test_more_than_the_caches_hold(dev, dtype, bits):
    """The steps of weights that go past the caches: a large one, and small ones of the same call, against a call of their own."""
    from vtpack_amd import _lib
    sizes = [(1 << 25) + 1029, 100003, 77]
    values, grads = _tensors(dev, [(n,) for n in sizes], dtype, 31), _tensors(dev, [(n,) for n in sizes], dtype, 32, 1e-3)
    ends = [torch.nn.Parameter(t[:5000].clone()) for t in values[:1]] + [torch.nn.Parameter(t.clone()) for t in values[1:]]
    large = [torch.nn.Parameter(t) for t in values]
    opts = [_optimizer(ps, bits) for ps in (large, ends)]
    for k in range(2):
        for ps in (large, ends):
            for p, g in zip(ps, grads):
                p.grad = g[:p.numel()] * (1 + k)
        for opt, name in zip(opts, ("true", "false")):
            opt.step()
            assert _lib.last_kernel().endswith(f", {bits}, {name}>")
        for p, q in zip(large, ends):
            # the same elements in the same places: whole blocks are the same, and so are whole tensors
            n = q.numel() if q.numel() == p.numel() else q.numel() // 256 * 256
            assert torch.equal(p[:n], q[:n])
            assert all(torch.equal(opts[0].state[p][key][:n].view(torch.uint8), opts[1].state[q][key][:n].view(torch.uint8)) for key in ("exp_avg", "exp_avg_sq"))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_places(dev, dtype, bits):
    """Weights off every vector's boundary, channels-last and transposed ones, gradients of other strides, neighbours left alone."""
    flat = _tensors(dev, [(6000,)], dtype, 6)[0]
    kept = flat.clone()
    params = [torch.nn.Parameter(flat[1:1002]), torch.nn.Parameter(flat[1003:1003 + 700]), torch.nn.Parameter(flat[2001:2001 + 35 * 40].view(35, 40).t()),
              torch.nn.Parameter(_tensors(dev, [(16, 9, 5, 3)], dtype, 7)[0].contiguous(memory_format=torch.channels_last))]
    order = [lambda t: t, lambda t: t, lambda t: t.t(), lambda t: t.permute(0, 2, 3, 1)]          # to the order of memory
    refs = [_Reference(f(p.detach()), bits) for f, p in zip(order, params)]
    opt = _optimizer(params, bits)
    for k in range(3):
        grads = [g.clone() for g in _tensors(dev, [p.shape for p in params], dtype, 20 + k, 1e-3)]
        grads[0] = torch.stack([grads[0], grads[0]], 1)[:, 1]
        for p, g in zip(params, grads):
            p.grad = g
        opt.step()
        for f, p, r in zip(order, params, refs):
            s = {key: f(t) if t.dim() == p.dim() and not key.endswith("scale") else t for key, t in opt.state[p].items() if torch.is_tensor(t)}
            r.step(f(p.grad))
            r.check(f(p.detach()), s)
    untouched = torch.ones(6000, dtype=torch.bool, device=dev)
    for a, n in ((1, 1001), (1003, 700), (2001, 1400)):
        untouched[a:a + n] = False
    assert torch.equal(flat[untouched], kept[untouched])


@pytest.mark.parametrize("bits", [32, 8])
def test_missing_gradients(dev, bits):
    """A weight's count of steps leaves out those without a gradient for it."""
    shapes = [(300,), (500,), (700,)]
    params = [torch.nn.Parameter(t) for t in _tensors(dev, shapes, torch.float32, 8)]
    refs = [_Reference(p, bits) for p in params]
    opt = _optimizer(params, bits)
    here = [(1, 1, 0), (1, 0, 0), (1, 1, 1), (0, 0, 0), (0, 1, 1), (1, 1, 1)]
    for k, row in enumerate(here):
        grads = _tensors(dev, shapes, torch.float32, 30 + k, 1e-3)
        for p, g, there in zip(params, grads, row):
            p.grad = g if there else None
        before = [p.detach().clone() for p in params]
        opt.step()
        for p, r, there, b in zip(params, refs, row, before):
            if there:
                r.step(p.grad)
                r.check(p, opt.state[p])
            else:
                assert torch.equal(p, b)


@pytest.mark.parametrize("bits", [32, 8])
def test_same_bits_again_and_in_a_graph(dev, bits):
    """Replays against eager steps, with lr read at the replay and work of the program's between."""
    shapes = [(777,), (64, 33), (5000,)]

    def make(capturable):
        params = [torch.nn.Parameter(t) for t in _tensors(dev, shapes, torch.float32, 9)]
        opt = _optimizer(params, bits, capturable=capturable)
        for p in params:
            p.grad = torch.empty_like(p)
        return params, opt

    def fill(params, k, scale=1e-3):
        for p, g in zip(params, _tensors(dev, shapes, torch.float32, 40 + k, scale)):
            p.grad.copy_(g)

    eager, opt = make(False)
    device, dopt = make(True)
    lr = torch.tensor([LR], device=dev)
    dopt.param_groups[0]["lr"] = lr
    opt.param_groups[0]["lr"] = float(lr)                 # what fp32 holds of it
    fill(eager, 0)
    fill(device, 0)
    opt.step()
    dopt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dopt.step()
    for k in range(1, 5):
        rate = LR / k
        lr.fill_(rate)
        opt.param_groups[0]["lr"] = float(lr)
        fill(eager, k)
        fill(device, k)
        opt.step()
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(eager, device):
            assert torch.equal(p, q)
            for key, t in opt.state[p].items():
                if torch.is_tensor(t):
                    assert torch.equal(t.view(torch.uint8), dopt.state[q][key].view(torch.uint8))
    assert int(dopt.param_groups[0]["step"]) == opt.param_groups[0]["step"] == 5


@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict(dev, bits):
    shapes = [(777,), (64, 33)]
    params = [torch.nn.Parameter(t) for t in _tensors(dev, shapes, torch.bfloat16, 9)]
    opt = _optimizer(params, bits)
    for k in range(6):
        if k == 3:
            saved = {key: v for key, v in opt.state_dict().items()}
            other = [torch.nn.Parameter(p.detach().clone()) for p in params]
            again = _optimizer(other, bits)
            again.load_state_dict(saved)
        for p, g in zip(params, _tensors(dev, shapes, torch.bfloat16, 50 + k, 1e-3)):
            p.grad = g
        opt.step()
        if k >= 3:
            for p, q in zip(params, other):
                q.grad = p.grad
            again.step()
            for p, q in zip(params, other):
                assert torch.equal(p, q)
                assert all(torch.equal(t.view(torch.uint8), again.state[q][key].view(torch.uint8)) for key, t in opt.state[p].items() if torch.is_tensor(t))


def test_eight_bits_follow_slow_changes(dev):
    """The second moment of a constant gradient decays to its square by 0.1 percent a step, a sixtieth of a code's step at least: its
    mean over many elements follows (each code is off by less than a fourth of itself, the mean of 65536 by 2^-8 of that)."""
    p = torch.nn.Parameter(torch.zeros(1 << 16, device=dev))
    opt = _optimizer([p], 8)
    ref_v = ref_m = 0.0
    for k in range(400):
        g = 1.0 if k < 20 else 0.1
        p.grad = torch.full_like(p, g) * (1 + 0.2 * torch.linspace(0, 1, p.numel(), device=dev))
        opt.step()
        ref_m, ref_v = 0.9 * ref_m + 0.1 * g, 0.999 * ref_v + 0.001 * g * g
    s, f = opt.state[p], 1 + 0.2 * torch.linspace(0, 1, p.numel(), device=dev)
    for key, want, power in (("exp_avg", ref_m, 1), ("exp_avg_sq", ref_v, 2)):
        value = s[key].float() * s[key + "_scale"].repeat_interleave(256) / f ** power
        assert abs(float(value.mean()) / want - 1) <= 0.25 * 2.0 ** -8 * 20       # the walk of the last steps, 1 / (1 - 0.999) at most
        assert float((s[key].float() == 0).float().mean()) < 0.01


@pytest.mark.parametrize("bits", [32, 8])
def test_not_a_number(dev, bits):
    """A gradient that is not finite shows in its weight (and its block's moments), and nowhere else."""
    p = torch.nn.Parameter(_tensors(dev, [(1000,)], torch.float32, 1)[0])
    q = torch.nn.Parameter(p.detach().clone())
    grads = _tensors(dev, [(1000,)], torch.float32, 2, 1e-3)[0]
    opt, other = _optimizer([p], bits), _optimizer([q], bits)
    p.grad, q.grad = grads.clone(), grads.clone()
    p.grad[300], p.grad[310] = float("nan"), float("inf")
    opt.step()
    other.step()
    touched = torch.zeros(1000, dtype=torch.bool, device=dev)
    touched[300] = touched[310] = True
    assert not torch.isfinite(p[touched]).any() and torch.equal(p[~touched], q[~touched])
    if bits == 8:
        touched[256:512] = True
        for key in ("exp_avg", "exp_avg_sq"):
            scale = opt.state[p][key + "_scale"]
            assert not torch.isfinite(scale[1]) and torch.equal(scale[[0, 2, 3]], other.state[q][key + "_scale"][[0, 2, 3]])


def test_weights_in_another_place(dev):
    """Storage that moved between steps, moments a program puts in place, the weights' version seen by what derives from them."""
    shapes = [(1000,), (300,)]
    params = [torch.nn.Parameter(t) for t in _tensors(dev, shapes, torch.float32, 11)]
    refs = [_Reference(p, 32) for p in params]
    opt = _optimizer(params, 32)
    for k in range(4):
        for p, g in zip(params, _tensors(dev, shapes, torch.float32, 60 + k, 1e-3)):
            p.grad = g
        if k == 2:
            params[0].data = params[0].data.clone()
        if k == 3:
            opt.state[params[1]]["exp_avg"] = opt.state[params[1]]["exp_avg"].clone()
        version = params[0]._version
        opt.step()
        assert params[0]._version > version
        for p, r in zip(params, refs):
            r.step(p.grad)
            r.check(p, opt.state[p])


def test_on_another_stream(dev):
    outs = []
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
        p = torch.nn.Parameter(_tensors(dev, [(100000,)], torch.float32, 12)[0])
        p.grad = _tensors(dev, [(100000,)], torch.float32, 13)[0]
        opt = _optimizer([p], 8)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            for _ in range(3):
                opt.step()
        torch.cuda.synchronize()
        outs.append(p)
    assert torch.equal(*outs)


def test_refusals(dev):
    from vtpack_amd.optim import AdamW

    def step(p, g, **kw):
        p = torch.nn.Parameter(p)
        p.grad = g
        AdamW([p], **kw).step()

    x = torch.randn(8, 8, device=dev)
    for p, g, error in [(x.half(), x.half(), TypeError), (x[:, :4], x[:, :4], ValueError), (x.double(), x.double(), TypeError),
                        (x, x.to_sparse(), ValueError)]:
        with pytest.raises(error):
            step(p, g)
    p = torch.nn.Parameter(x.clone())
    p.grad = x.clone()
    opt = AdamW([p], state_bits=8)
    opt.step()
    opt.param_groups[0]["state_bits"] = 32
    with pytest.raises(ValueError, match="exp_avg"):
        opt.step()
    opt = AdamW([p])
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="capturable"):
        with torch.cuda.graph(graph):
            opt.step()
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="before the capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            AdamW([p], capturable=True).step()
    torch.cuda.synchronize()
    opt = AdamW([p], lr=torch.tensor(1e-3, device=dev), capturable=True)
    opt.step()
    opt.param_groups[0]["lr"] = torch.tensor(1e-3)
    with pytest.raises(ValueError):
        opt.step()


@pytest.mark.parametrize("bits", [32, 8])
def test_steps_that_find_everything_in_place(dev, bits, monkeypatch):
    """Two groups over several steps, one native call each; what has moved in between is found."""
    from vtpack_amd import optim
    looked = []
    take = optim._Batch.take_gradients
    monkeypatch.setattr(optim._Batch, "take_gradients", lambda self, grads: looked.append(1) or take(self, grads))
    shapes = [(700,), (3, 50), (1025,), (8,)]
    params = [torch.nn.Parameter(t) for t in _tensors(dev, shapes, torch.float32, 21)]
    refs = [_Reference(p, bits) for p in params]
    opt = _optimizer([{"params": params[:2]}, {"params": params[2:]}], bits)
    expect = {7: 1}                                        # groups whose gradients are laid out anew in Python
    for k in range(9):
        for p, g in zip(params, _tensors(dev, shapes, torch.float32, 80 + k, 1e-3)):
            p.grad = g
        if k == 3:                                         # a moment whose storage is another
            m = opt.state[params[0]]["exp_avg"]
            m.data = m.data.clone()
        if k == 4:                                         # all states replaced by copies
            opt.load_state_dict(opt.state_dict())
        if k == 6:                                         # a weight with storage of its own, at another place
            params[3].data = params[3].data.clone()
        if k == 7:                                         # a gradient of other strides
            params[1].grad = params[1].grad.t().contiguous().t()
        for g in opt.param_groups:
            g["lr"] = LR * (1 + k % 2)
        before, versions = len(looked), [p._version for p in params]
        opt.step()
        assert len(looked) - before == expect.get(k, 0), k
        assert all(p._version > v for p, v in zip(params, versions))
        for p, r in zip(params, refs):
            r.step(p.grad, LR * (1 + k % 2))
            r.check(p, opt.state[p])
    assert all(g["step"] == 9 for g in opt.param_groups)
    params[0].grad.data = params[0].grad.data[:10]         # a gradient that no longer fits
    with pytest.raises(ValueError):
        opt.step()


def test_weights_over_each_other_are_refused(dev):
    from vtpack_amd.optim import AdamW
    flat = torch.randn(1000, device=dev)
    for a, b in ((flat, flat), (flat[:600], flat[599:])):
        params = [torch.nn.Parameter(a), torch.nn.Parameter(b)]
        for p in params:
            p.grad = torch.ones_like(p)
        with pytest.raises(ValueError, match="over each other"):
            AdamW(params).step()
    p = torch.nn.Parameter(flat)
    p.grad = torch.ones_like(p)
    with pytest.warns(UserWarning, match="duplicate"):
        opt = AdamW([p, p])
    with pytest.raises(ValueError, match="over each other"):
        opt.step()
    halves = [torch.nn.Parameter(flat[:500]), torch.nn.Parameter(flat[500:])]       # side by side
    for p in halves:
        p.grad = torch.ones_like(p)
    AdamW(halves).step()


def test_steps_leave_no_memory_behind(dev):
    import gc
    from vtpack_amd.layers import gate_balance, linear_cross_entropy
    x, w = (torch.randn(n, 64, device=dev, requires_grad=True) for n in (100, 50))
    t = torch.randint(0, 50, (100,), device=dev)
    opt = _optimizer([x, w], 8)
    used = []
    for k in range(6):
        for _ in range(50):
            opt.zero_grad()
            (linear_cross_entropy(x, w, None, t) + gate_balance(x, mask=t > 3)[0]).backward()
            opt.step()
        if k == 3:
            opt.load_state_dict(opt.state_dict())          # tables are made anew
        opt.zero_grad()
        gc.collect()
        used.append(torch.cuda.memory_allocated())
    assert used[-1] <= used[0]


@pytest.mark.parametrize("bits", [32, 8])
def test_groups_that_are_looked_over_once(dev, bits, monkeypatch):
    """A frozen weight among others, weights of other strides: what was found out about them is kept from step to step."""
    from vtpack_amd import _lib, optim
    shapes = [(300,), (40, 30), (77,)]
    frozen = [torch.nn.Parameter(t) for t in _tensors(dev, shapes, torch.float32, 41)]
    strided = [torch.nn.Parameter(_tensors(dev, [(30, 20)], torch.float32, 42)[0].t()), torch.nn.Parameter(_tensors(dev, [(50,)], torch.float32, 43)[0])]
    refs = [_Reference(p if p.is_contiguous() else p.detach().t(), bits) for p in frozen + strided]
    opt = _optimizer([{"params": frozen}, {"params": strided}], bits)
    split, native = [], []
    real, made = optim.AdamW._split, _lib.training().adamw_batch

    class Native:
        def __getattr__(self, name):
            return getattr(real_native, name)

        def adamw_batch(self, *args):
            native.append(1)
            return made(*args)

    real_native, wrapped = _lib.training(), Native()
    monkeypatch.setattr(_lib, "training", lambda: wrapped)
    monkeypatch.setattr(optim.AdamW, "_split", lambda self, *args: split.append(1) or real(self, *args))
    for k in range(4):
        for i, (p, g) in enumerate(zip(frozen + strided, _tensors(dev, [p.shape for p in frozen + strided], torch.float32, 90 + k, 1e-3))):
            p.grad = None if i == 1 else g.t().contiguous().t() if i == 3 else g
        opt.step()
        for p, r in zip(frozen + strided, refs):
            if p.grad is not None:
                flip = (lambda t: t) if p.is_contiguous() else (lambda t: t.t() if t.dim() == 2 else t)
                r.step(flip(p.grad))
                r.check(flip(p.detach()), {key: flip(t) for key, t in opt.state[p].items() if torch.is_tensor(t)})
    assert len(native) == 2 and len(split) == 1


@pytest.mark.parametrize("bits", [32, 8])
def test_another_tensor_at_the_same_address(dev, bits):
    """Weights and moments whose storage is given up and taken again, as others of other sizes and types: found or refused."""
    flat = torch.randn(2048, device=dev)
    p, q = torch.nn.Parameter(flat[:1024]), torch.nn.Parameter(torch.randn(1024, device=dev).view(32, 32).t())
    opt = _optimizer([{"params": [p]}, {"params": [q]}], bits)
    for x in (p, q):
        x.grad = torch.full_like(x, 1e-3)
    opt.step()
    opt.step()
    for x in (p, q):                                       # half of the weight, its states as they were
        kept, moment = x.data, opt.state[x]["exp_avg"].data
        x.data = x.data[:x.shape[0] // 2]
        x.grad = torch.full_like(x, 1e-3)
        whole = kept.clone()
        with pytest.raises(ValueError):
            opt.step()
        assert torch.equal(kept, whole)
        x.data = kept
        x.grad = torch.full_like(x, 1e-3)
        if bits == 32:                                     # the moment's memory under another type
            opt.state[x]["exp_avg"].data = moment.view(torch.int32)
            with pytest.raises(ValueError):
                opt.step()
            opt.state[x]["exp_avg"].data = moment
    opt.step()


@pytest.mark.parametrize("bits", [32, 8])
def test_a_step_that_is_refused_changes_nothing(dev, bits):
    """Neither the counts of the weights that have no gradient, nor the weights of a group that come before the one that does not fit."""
    params = [torch.nn.Parameter(_tensors(dev, [(300,)], d, i)[0]) for i, d in enumerate((torch.float32, torch.float32, torch.bfloat16))]
    refs = [_Reference(p, bits) for p in params]
    opt = _optimizer(params, bits)
    for k in range(3):
        for bad in (True, False) if k else (False,):
            for i, p in enumerate(params):
                p.grad = _tensors(dev, [(300,)], p.dtype, 70 + 3 * k + i, 1e-3)[0]
            if not bad:
                opt.step()
                for p, r in zip(params, refs):
                    r.step(p.grad)
                    r.check(p, opt.state[p])
                continue
            before = [p.detach().clone() for p in params]
            if k == 1:
                params[0].grad = None
            params[2].grad.data = params[2].grad.data[:299]
            with pytest.raises(ValueError):
                opt.step()
            assert all(torch.equal(p, q) for p, q in zip(params, before)) and opt.param_groups[0]["step"] == k


@pytest.mark.parametrize("bits", [32, 8])
def test_a_layer_frozen_after_some_steps(dev, bits, monkeypatch):
    """What is looked over once for the weights that go on is kept from step to step, and made anew when the others come back."""
    from vtpack_amd import _lib
    shapes = [(300,), (40, 30), (77,), (1025,)]
    params = [torch.nn.Parameter(t) for t in _tensors(dev, shapes, torch.float32, 51)]
    refs = [_Reference(p, bits) for p in params]
    opt = _optimizer(params, bits)
    real, made = _lib.training(), []

    class Native:
        def __getattr__(self, name):
            return getattr(real, name)

        def adamw_batch(self, *args):
            made.append(1)
            return real.adamw_batch(*args)

    wrapped = Native()
    monkeypatch.setattr(_lib, "training", lambda: wrapped)
    here = [(1, 1, 1, 1)] * 2 + [(1, 0, 0, 1)] * 4 + [(1, 1, 1, 1)] * 2 + [(1, 0, 0, 1)] * 2
    for k, row in enumerate(here):
        for p, g, there in zip(params, _tensors(dev, shapes, torch.float32, 140 + k, 1e-3), row):
            p.grad = g if there else None
        opt.step()
        for p, r in zip(params, refs):
            if p.grad is not None:
                r.step(p.grad)
                r.check(p, opt.state[p])
        if k == 5:
            assert len(made) == 2                          # of all weights, and of those that went on


@pytest.mark.parametrize("bits", [32, 8])
def test_states_in_another_order(dev, bits, monkeypatch):
    """A state dict whose weights come in another order: a step is one native call all the same."""
    from vtpack_amd import optim
    looked = []
    launch = optim.AdamW._launch
    monkeypatch.setattr(optim.AdamW, "_launch", lambda self, *args: looked.append(1) or launch(self, *args))
    shapes = [(300,), (40, 30), (77,), (5,)]
    params = [torch.nn.Parameter(t) for t in _tensors(dev, shapes, torch.float32, 61)]
    refs = [_Reference(p, bits) for p in params]
    opt = _optimizer([{"params": params[:3]}, {"params": params[3:]}], bits)
    for k in range(5):
        for p, g, r in zip(params, _tensors(dev, shapes, torch.float32, 160 + k, 1e-3), refs):
            p.grad = g
            r.step(g)
        if k == 2:
            saved = opt.state_dict()
            saved["state"] = dict(reversed(list(saved["state"].items())))
            opt.load_state_dict(saved)
        opt.step()
        for p, r in zip(params, refs):
            r.check(p, opt.state[p])
    assert not looked


def test_an_optimizer_that_its_weights_refer_to_is_collected(dev):
    """A step inside a weight's own hook; and weights that move away leave no memory behind."""
    import gc
    import weakref
    gc.collect()
    used = torch.cuda.memory_allocated()
    p = torch.nn.Parameter(torch.randn(1 << 20, device=dev))
    opt = _optimizer([p], 32)
    p.optimizer = opt
    p.register_post_accumulate_grad_hook(lambda q: q.optimizer.step())
    for _ in range(2):
        (p * 2).sum().backward()
    assert opt.param_groups[0]["step"] == 2
    dead = weakref.ref(opt)
    del p, opt
    gc.collect()
    assert dead() is None and torch.cuda.memory_allocated() <= used


@pytest.mark.parametrize("strided", [False, True])
def test_weights_that_move_away_leave_no_memory(dev, strided):
    w = torch.randn(1 << 10, 1 << 10, device=dev)
    p = torch.nn.Parameter(w.t() if strided else w)
    opt = _optimizer([p], 32)
    for _ in range(2):
        p.grad = torch.full_like(p, 1e-3)
        opt.step()
    del w
    p.grad = None
    used = torch.cuda.memory_allocated()
    p.data = p.data.cpu()
    assert used - torch.cuda.memory_allocated() >= 4 << 20
