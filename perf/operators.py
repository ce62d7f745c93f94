"""The operators of a training step behind the encoder: the classifier's cross entropy with its gradients, the balance loss of
the routers' gates with its gradient, and the AdamW step over all weights.

  cross_entropy  logits x W^T + b of rows of features, softmax cross entropy with label smoothing and left-out rows; the mean
                 loss with the gradients of x, W and b, or (`train` false) every row's own loss, as a validation pass logs it;
  balance        E sum_e f_e P_e of gate logits: f_e the fraction of the choices that fell on e, P_e its mean probability;
                 the counts, and with `train` the gradient of the logits;
  adamw          one step over a list of tensors, both moments kept in 32 bits or in 8 bits with a scale for 256 of them.

Eight-bit moments: the first as e4m3 with the scale max|m| / 448, the second as e5m2 with max v / 57344, over 256 consecutive
elements of a tensor.  A value is rounded down or up at random, so that slow changes are not lost: 16 bits of a hash of the
element's place and the step's number are added below the last bit that stays.  A second moment that is not zero stays so.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
IGNORE = -100
BLOCK = 256                      # elements of a tensor that share a scale
BETAS, EPS = (0.9, 0.999), 1e-8
# of an 8-bit type: bits of the mantissa, smallest normal and largest number, whether it takes the low half of the random bits
FIRST, SECOND = (3, 2.0 ** -6, 448.0, True), (2, 2.0 ** -14, 57344.0, False)


# ------------------------------------------------------------------------------------------------ cases
def _ce(name, dtype, rows, width, classes, bias=True, smoothing=0.0, left_out=0.0, train=True):
    return {"name": name, "op": "cross_entropy", "dtype": dtype, "rows": rows, "width": width, "classes": classes, "bias": bias,
            "smoothing": smoothing, "left_out": left_out, "train": train}


def _balance(name, dtype, tokens, experts, top_k=1, padded=0.0, train=True):
    return {"name": name, "op": "balance", "dtype": dtype, "tokens": tokens, "experts": experts, "top_k": top_k, "padded": padded,
            "train": train}


def _adamw(name, dtype, bits, width, depth, classes, lr=5e-4, decay=0.05):
    return {"name": name, "op": "adamw", "dtype": dtype, "bits": bits, "width": width, "depth": depth, "classes": classes, "lr": lr,
            "decay": decay}


def listed():
    return [
        # DeiT-S trained in bf16: the class tokens of a batch of 256 pictures, 1000 classes, the usual smoothing
        _ce("ce_small_bf16_b256", "bf16", 256, 384, 1000, smoothing=0.1),
        # the published data type: DeiT-Ti in fp32, a batch of odd size
        _ce("ce_tiny_f32_b1021", "f32", 1021, 192, 1000, smoothing=0.1),
        # pre-training on a large label set, the widest model; a last batch in part padded
        _ce("ce_base_bf16_21841", "bf16", 2999, 768, 21841, left_out=0.05),
        # the same head in fp32
        _ce("ce_small_f32_21841", "f32", 2048, 384, 21841),
        # a vocabulary over many positions at once, no bias: the largest
        _ce("ce_wide_bf16_65536", "bf16", 8192, 1024, 65536, bias=False),
        # one row against a large vocabulary, the loss alone: scoring a single answer
        _ce("ce_one_row_bf16_65536", "bf16", 1, 1024, 65536, bias=False, train=False),
        # gates of one encoder layer: 8 pictures of 16 regions, three granularities
        _balance("balance_layer_f32_128", "f32", 128, 3),
        # the gates of 512 px pictures, a whole layer of a large batch
        _balance("balance_layer_bf16_65536", "bf16", 65536, 3),
        # a router of many experts, several for each token, a padded batch
        _balance("balance_experts_bf16_131071", "bf16", 131071, 160, top_k=6, padded=0.1),
        # all weights of DeiT-Ti: 5.7 M in about 200 tensors
        _adamw("adamw_tiny_f32", "f32", 32, 192, 12, 1000),
        # all weights of DeiT-S, moments in 8 bits
        _adamw("adamw_small_f32_8bit", "f32", 8, 384, 12, 1000),
        # 100 M weights in bf16, moments in 32 bits
        _adamw("adamw_wide_bf16", "bf16", 32, 1024, 8, 1000),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, spread over the logarithm, hardly ever round."""
    return min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))


def draw(rng):
    op = rng.choice(["cross_entropy", "cross_entropy", "balance", "adamw"])
    dtype = rng.choice(["bf16", "f32"])
    if op == "cross_entropy":
        most = 8192 * 1024 * 65536 // (1 if dtype == "bf16" else 8)
        classes, width = _spread(rng, 2, 65536), _spread(rng, 32, 1024)
        if rng.random() < 0.5:
            width = -(-width // 64) * 64
        rows = _spread(rng, 1, max(1, min(8192, most // (classes * width))))
        case = _ce("", dtype, rows, width, classes, bias=rng.random() < 0.7, smoothing=rng.choice([0.0, 0.1]),
                   left_out=rng.choice([0.0, 0.0, 0.2]), train=rng.random() < 0.8)
    elif op == "balance":
        experts = _spread(rng, 2, 512)
        tokens = _spread(rng, 1, 131072 * 160 // experts if experts > 160 else 131072)
        case = _balance("", dtype, tokens, experts, top_k=rng.randint(1, min(8, experts)), padded=rng.choice([0.0, 0.3]),
                        train=rng.random() < 0.8)
    else:
        case = _adamw("", dtype, rng.choice([32, 8]), _spread(rng, 32, 1024), rng.randint(1, 8), _spread(rng, 2, 2000),
                      lr=rng.choice([1e-3, 5e-4]), decay=rng.choice([0.0, 0.05]))
    del case["name"]
    return case


def _shapes(case):
    """The weights of a vision transformer of that width, depth and number of classes, biases and norms among them."""
    c = case["width"]
    layer = [(c,), (c,), (c, c), (c,), (2 * c, c), (2 * c,), (c, c), (c,), (c,), (c,), (4 * c, c), (4 * c,), (c, 4 * c), (c,), (3, c), (3,)]
    return [(1, 1, c), (1, 257, c), (c, 3, 16, 16), (c,)] + layer * case["depth"] + [(c,), (c,), (case["classes"], c), (case["classes"],)]


# ------------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ce_inputs(case, seed):
    g, dtype = _generator(seed), DTYPES[case["dtype"]]
    rows, width, classes = case["rows"], case["width"], case["classes"]
    x = torch.randn(rows, width, device="cuda", generator=g)
    w = torch.randn(classes, width, device="cuda", generator=g) * (1.5 * width ** -0.5)
    b = torch.randn(classes, device="cuda", generator=g) * 0.5
    target = torch.randint(0, classes, (rows,), device="cuda", generator=g)
    # a model in training: the right class stands out by now
    x = x + 0.05 * width ** 0.5 * w[target]
    if case["left_out"] > 0 and rows > 1:
        out = torch.rand(rows, device="cuda", generator=g) < case["left_out"]
        out[0] = False
        target = torch.where(out, IGNORE, target)
    return x.to(dtype), w.to(dtype), b.to(dtype) if case["bias"] else None, target


def _balance_inputs(case, seed):
    g = _generator(seed)
    gate = torch.randn(case["tokens"], case["experts"], device="cuda", generator=g)
    gate = (gate + 0.5 * torch.randn(case["experts"], device="cuda", generator=g)).to(DTYPES[case["dtype"]])
    mask = None
    if case["padded"] > 0 and case["tokens"] > 1:
        mask = torch.rand(case["tokens"], device="cuda", generator=g) >= case["padded"]
        mask[0] = True
    return gate, mask


def _adamw_inputs(case, seed):
    """-> weights, gradients, first and second moments (fp32 values), [blocks, BLOCK]: the tensors one behind the other in one
    allocation, each from a block's start on, zeros behind its end."""
    g = _generator(seed)
    sizes = [math.prod(s) for s in _shapes(case)]
    shape = (sum(-(-n // BLOCK) for n in sizes), BLOCK)
    p, grad, m, v, spread = (torch.randn(shape, device="cuda", generator=g) for _ in range(5))
    grad = grad * 1e-4 * torch.exp(0.5 * spread)
    m = 0.3 * grad + 5e-5 * m
    v = (1e-4 * v) ** 2 + 0.01 * grad * grad
    used = (_places(sizes, "cuda") < _of_blocks(sizes, torch.tensor(sizes, device="cuda")).unsqueeze(1)).float()
    return tuple(t * used for t in (0.02 * p, grad, m, v))


def _views(case, flat, scales=False):
    """The tensors of `flat` (`scales`: one value for each block)."""
    shapes = _shapes(case)
    blocks = [-(-math.prod(s) // BLOCK) for s in shapes]
    if scales:
        return list(flat.split(blocks))
    return [t.view(-1)[:math.prod(s)].view(s) for t, s in zip(flat.split(blocks), shapes)]


def prepare(case, seed):
    if case["op"] == "cross_entropy":
        x, w, b, target = _ce_inputs(case, seed)
        leaves = [t.requires_grad_(case["train"]) for t in (x, w, b) if t is not None]
        return {"case": case, "x": x, "weight": w, "bias": b, "target": target, "leaves": leaves}
    if case["op"] == "balance":
        gate, mask = _balance_inputs(case, seed)
        return {"case": case, "gate": gate.requires_grad_(case["train"]), "mask": mask}
    p, grad, m, v = _adamw_inputs(case, seed)
    dtype = DTYPES[case["dtype"]]
    state = {"case": case, "step": 99, "params": p.to(dtype), "grads": grad.to(dtype), "m": m, "v": v}
    if case["bits"] == 8:
        sizes = [math.prod(s) for s in _shapes(case)]
        state["m"], state["m_scale"] = _encode(m, sizes, 98, torch.float8_e4m3fn)
        state["v"], state["v_scale"] = _encode(v, sizes, 98, torch.float8_e5m2)
    if own:
        from vtpack_amd.optim import AdamW
        leaves = [torch.nn.Parameter(t) for t in _views(case, state["params"])]
        optimizer = AdamW(leaves, lr=case["lr"], betas=BETAS, eps=EPS, weight_decay=case["decay"], state_bits=case["bits"])
        optimizer.param_groups[0]["step"] = state["step"]
        for names in (("grads", None), ("m", "exp_avg"), ("v", "exp_avg_sq"), ("m_scale", "exp_avg_scale"), ("v_scale", "exp_avg_sq_scale")):
            if names[0] in state:
                for leaf, t in zip(leaves, _views(case, state[names[0]], names[0].endswith("scale"))):
                    if names[1] is None:
                        leaf.grad = t
                    else:
                        optimizer.state[leaf][names[1]] = t
        state["optimizer"] = optimizer
    return state


# ------------------------------------------------------------------------------------------------ plain forms
def _ce_plain(case, x, w, b, target):
    x32, w32, eps, classes = x.detach().float(), w.detach().float(), case["smoothing"], case["classes"]
    logits = x32 @ w32.t()
    if b is not None:
        logits = logits + b.detach().float()
    live = (target != IGNORE).float()
    at = target.clamp(min=0).unsqueeze(1)
    top = logits.max(1, keepdim=True).values
    e = torch.exp(logits - top)
    total = e.sum(1, keepdim=True)
    lse = top + torch.log(total)
    loss = (lse - (1 - eps) * logits.gather(1, at)).squeeze(1) - eps * logits.mean(1)
    loss = torch.where(live > 0, loss, torch.zeros_like(loss))
    if not case["train"]:
        return loss
    count = live.sum().clamp(min=1)
    g = (live / count).unsqueeze(1)
    d = e * (g / total)
    if eps > 0:
        d = d - g * (eps / classes)
    d.scatter_add_(1, at, -(1 - eps) * g)
    out = [loss.sum() / count, (d @ w32).to(x.dtype), (d.t() @ x32).to(w.dtype)]
    return out + [d.sum(0).to(b.dtype)] if b is not None else out


def _balance_plain(case, gate, mask):
    z, experts, k = gate.detach().float(), case["experts"], case["top_k"]
    e = torch.exp(z - z.max(1, keepdim=True).values)
    p = e / e.sum(1, keepdim=True)
    # ties go to the lowest index: argmax gives the first, a stable sort keeps them in order
    chosen = z.argmax(1, keepdim=True) if k == 1 else torch.sort(z, dim=1, descending=True, stable=True).indices[:, :k]
    live = torch.ones(z.shape[0], device=z.device) if mask is None else mask.float()
    tokens = live.sum().clamp(min=1)
    counts = torch.zeros_like(z).scatter_(1, chosen, live.unsqueeze(1).expand(-1, k)).sum(0)
    f = counts.double() / (tokens * k)
    mean = (p * live.unsqueeze(1)).sum(0, dtype=torch.float64) / tokens
    loss = (experts * (f * mean).sum()).float()
    if not case["train"]:
        return [loss, counts.long()]
    f32 = f.float()
    grad = (experts / tokens) * live.unsqueeze(1) * p * (f32 - (p * f32).sum(1, keepdim=True))
    return [loss, counts.long(), grad.to(gate.dtype)]


def _of_blocks(sizes, values):
    """values[i] for every block of tensor i."""
    return torch.repeat_interleave(values, torch.tensor([-(-n // BLOCK) for n in sizes], device=values.device))


def _places(sizes, device):
    """The place of every element in its own tensor, [blocks, BLOCK]."""
    blocks = torch.tensor([-(-n // BLOCK) for n in sizes], device=device)
    first = _of_blocks(sizes, torch.cumsum(blocks, 0) - blocks)
    return ((torch.arange(first.numel(), device=device) - first) * BLOCK).unsqueeze(1) + torch.arange(BLOCK, device=device)


def _dither(at, step):
    """32 bits for every element from its place and the step's number: multiplications by odd numbers (the first 32 bits behind the
    point of the square roots of 2, 3, 5 and 7, the last bit set) with shifts between them."""
    low = 0xffffffff
    h = (at * 0x6a09e667 + ((step * 0xbb67ae85) & low)) & low
    h = ((h ^ (h >> 16)) * 0x3c6ef373) & low
    h = ((h ^ (h >> 15)) * 0xa54ff53b) & low
    return h ^ (h >> 16)


def _encode(values, sizes, step, dtype):
    """[blocks, BLOCK] fp32 -> 8-bit values of `dtype` and a scale for each block."""
    first = dtype == torch.float8_e4m3fn
    top, small, drop = (448.0, 2.0 ** -6, 20) if first else (57344.0, 2.0 ** -14, 21)
    size = values.abs()
    most = size.max(1, keepdim=True).values
    zero = most < 2.0 ** -100
    scale = torch.where(zero, torch.zeros_like(most), most * (1.0 / top))
    inverse = torch.where(zero, torch.zeros_like(most), torch.full_like(most, top) / most)
    x = torch.clamp(size * inverse, max=top)
    lift = torch.where(x < small, torch.full_like(x, small), torch.zeros_like(x))
    bits = (x + lift).view(torch.int32)
    h = _dither(_places(sizes, x.device), step)
    noise = ((h & 0xffff) if first else (h >> 16)) << (drop - 16)
    kept = ((bits + noise.int()) >> drop) << drop
    q = kept.view(torch.float32) - lift
    if not first:
        q = torch.where((x > 0) & (q == 0), torch.full_like(q, 2.0 ** -16), q)
    return torch.copysign(q, values).to(dtype), scale.squeeze(1)


def _adamw_plain(state):
    case, (b1, b2) = state["case"], BETAS
    state["step"] += 1
    step = state["step"]
    p, g, m, v = (state[k].float() for k in ("params", "grads", "m", "v"))
    if case["bits"] == 8:
        m = m * state["m_scale"].unsqueeze(1)
        v = v * state["v_scale"].unsqueeze(1)
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * (1 - b2)) * g
    p = p * (1 - case["lr"] * case["decay"])
    p = p - (case["lr"] / (1 - b1 ** step)) * (m / (torch.sqrt(v) * (1 / math.sqrt(1 - b2 ** step)) + EPS))
    state["params"] = p.to(state["params"].dtype)
    if case["bits"] == 8:
        sizes = [math.prod(s) for s in _shapes(case)]
        state["m"], state["m_scale"] = _encode(m, sizes, step, torch.float8_e4m3fn)
        state["v"], state["v_scale"] = _encode(v, sizes, step, torch.float8_e5m2)
    else:
        state["m"], state["v"] = m, v
    return _adamw_outputs(state)


def _adamw_outputs(state):
    return {k: state[k] for k in ("params", "m", "v", "m_scale", "v_scale") if k in state}


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    if case["op"] == "cross_entropy":
        if not own:
            return _ce_plain(case, state["x"], state["weight"], state["bias"], state["target"])
        from vtpack_amd.layers import linear_cross_entropy
        loss = linear_cross_entropy(state["x"], state["weight"], state["bias"], state["target"], ignore_index=IGNORE,
                                    label_smoothing=case["smoothing"], reduction="mean" if case["train"] else "none")
        return [loss, *torch.autograd.grad(loss, state["leaves"])] if case["train"] else loss
    if case["op"] == "balance":
        if not own:
            return _balance_plain(case, state["gate"], state["mask"])
        from vtpack_amd.layers import gate_balance
        loss, counts = gate_balance(state["gate"], top_k=case["top_k"], mask=state["mask"])
        return [loss, counts, *torch.autograd.grad(loss, [state["gate"]])] if case["train"] else [loss, counts]
    if not own:
        return _adamw_plain(state)
    state["optimizer"].step()
    return _adamw_outputs(state)


# ------------------------------------------------------------------------------------------------ work
def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "cross_entropy":
        r, h, v = case["rows"], case["width"], case["classes"]
        operands = (r * h + v * h + (v if case["bias"] else 0)) * size
        if not case["train"]:
            return {"bytes": operands + 8 * r + 4 * r, "flops": 2 * r * h * v}
        # the logits, then from their gradients those of x and of W
        return {"bytes": 2 * operands + 8 * r + 4, "flops": 6 * r * h * v}
    if case["op"] == "balance":
        n = case["tokens"] * case["experts"]
        mask = case["tokens"] if case["padded"] > 0 else 0
        return {"bytes": n * size * (2 if case["train"] else 1) + mask + 8 * case["experts"] + 4, "flops": n * (8 if case["train"] else 5)}
    n = sum(math.prod(s) for s in _shapes(case))
    states = 4 * 4 * n if case["bits"] == 32 else (4 + 16 / BLOCK) * n
    return {"bytes": int(3 * size * n + states), "flops": 14 * n}


# ------------------------------------------------------------------------------------------------ in 64 bits
def _ce_exact(case, seed):
    x, w, b, target = _ce_inputs(case, seed)
    x, w = x.double(), w.double()
    logits = torch.mm(x, w.t().contiguous())
    if b is not None:
        logits += b.double()
    rows = torch.arange(case["rows"], device=x.device)
    live = target >= 0
    lse = torch.logsumexp(logits, 1)
    wanted = torch.zeros_like(logits) + case["smoothing"] / case["classes"]
    wanted[rows[live], target[live]] += 1 - case["smoothing"]
    loss = (lse - (wanted * logits).sum(1)) * live
    if not case["train"]:
        return loss
    count = max(1, int(live.sum()))
    d = (torch.exp(logits - lse[:, None]) - wanted) * (live[:, None] / count)
    out = [loss.sum() / count, torch.mm(d, w), torch.mm(d.t().contiguous(), x)]
    return out if b is None else out + [d.sum(0)]


def _balance_exact(case, seed):
    gate, mask = _balance_inputs(case, seed)
    if mask is None:
        mask = torch.ones(case["tokens"], dtype=torch.bool, device="cuda")
    k, experts = case["top_k"], case["experts"]
    z = gate[mask].double()
    p = torch.softmax(z, 1)
    # the k largest, lower indices first: (logit, -index) as one key
    order = torch.from_numpy(np.lexsort((np.broadcast_to(np.arange(experts), z.shape), -z.cpu().numpy()), axis=1)[:, :k].copy())
    counts = torch.bincount(order.reshape(-1), minlength=experts).cuda()
    f = counts.double() / (z.shape[0] * k)
    loss = experts * torch.dot(f, p.mean(0))
    if not case["train"]:
        return [loss, counts]
    grad = torch.zeros(gate.shape, dtype=torch.float64, device="cuda")
    grad[mask] = p * (f - (p @ f)[:, None]) * (experts / z.shape[0])
    return [loss, counts, grad]


def _f32(t):
    """A value as a 32-bit number holds it, in 64 bits."""
    return t.float().double()


def _coded(blocks, place, step, mantissa, smallest, top, low_bits):
    """8-bit values and scales of a moment by counting: multiples of the step between neighbours, in 64 bits."""
    most = blocks.abs().amax(1, keepdim=True)
    some = most >= 2.0 ** -100
    scale = _f32(most * float(np.float32(1.0 / top))) * some
    x = _f32(blocks.abs() * torch.where(some, _f32(top / most.clamp(min=2.0 ** -100)), torch.zeros_like(most))).clamp(max=top)
    h = _dither(place, step)
    share = ((h % 65536) if low_bits else torch.div(h, 65536, rounding_mode="floor")).double() / 65536
    octave = x.clamp(min=smallest) / (2 * torch.frexp(x.clamp(min=smallest)).mantissa)
    unit = octave * 2.0 ** -mantissa
    q = torch.floor(torch.where(x < smallest, _f32(x + smallest) - smallest, x) / unit + share) * unit
    if not low_bits:
        q = torch.where((x > 0) & (q == 0), torch.full_like(q, 2.0 ** -16), q)
    return q * blocks.sign(), scale.squeeze(1)


def _adamw_exact(case, seed):
    p, g, m, v = _adamw_inputs(case, seed)
    dtype, step, (b1, b2) = DTYPES[case["dtype"]], 100, BETAS
    p, g = p.to(dtype).double(), g.to(dtype).double()
    sizes = [math.prod(s) for s in _shapes(case)]
    place = _places(sizes, "cuda")
    if case["bits"] == 8:
        coarse = [_coded(t.double(), place, 98, *how) for t, how in ((m, FIRST), (v, SECOND))]
        m, v = (_f32(t * s.unsqueeze(1)) for t, s in coarse)
        # what the codes are made from is rounded to 32 bits step by step, the factors too; the rest is not
        c1, c2, d1, d2 = (float(np.float32(t)) for t in (b1, b2, 1 - b1, 1 - b2))
        m = _f32(_f32(m * c1) + _f32(g * d1))
        v = _f32(_f32(v * c2) + _f32(_f32(g * d2) * g))
    else:
        m = m.double() * b1 + g * (1 - b1)
        v = v.double() * b2 + g * g * (1 - b2)
    out = {"params": p * (1 - case["lr"] * case["decay"]) - case["lr"] * (m / (1 - b1 ** step)) / (torch.sqrt(v / (1 - b2 ** step)) + EPS)}
    if case["bits"] == 8:
        m, out["m_scale"] = _coded(m, place, step, *FIRST)
        v, out["v_scale"] = _coded(v, place, step, *SECOND)
    return {**out, "m": m, "v": v}


def exact(case, seed):
    return {"cross_entropy": _ce_exact, "balance": _balance_exact, "adamw": _adamw_exact}[case["op"]](case, seed)
