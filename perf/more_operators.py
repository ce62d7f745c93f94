"""The operators on blocks of 8-bit numbers: the checkpoint of an activation, the Linear that multiplies them, and the Linear, GELU
and LayerNorm of a training step that keep their input in them.

A block is 128 consecutive numbers of a row (the last of a row may be shorter): e4m3 values and a power of two 2^e, e the smallest whole
number with max |x| 2^-e <= 448, and -110 at least.

  checkpoint    an activation brought into blocks and back;
  linear        act(Q(x) Q(W)^T + b), W kept in blocks;
  linear_train  the same without act, W in full, with the gradients g Q(W), g^T Q(x) and the column sums of g, the gradient that comes in
                rounded to bf16;
  gelu          x Phi(x) with dx from Q(x);
  layer_norm    with its gradients from Q(x - mean); the mean is the fp32 number next to the row's.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
BLOCK = 128
LEAST = -110                     # exponent of a scale
EPS = 1e-6


# ------------------------------------------------------------------------------------------------ cases
def _linear(name, dtype, rows, width, out, act="none", bias=True):
    return {"name": name, "op": "linear", "dtype": dtype, "rows": rows, "width": width, "out": out, "act": act, "bias": bias}


def _train(name, dtype, rows, width, out, bias=True):
    return {"name": name, "op": "linear_train", "dtype": dtype, "rows": rows, "width": width, "out": out, "bias": bias}


def _plane(op, name, dtype, rows, width):
    return {"name": name, "op": op, "dtype": dtype, "rows": rows, "width": width}


def listed():
    return [
        # an activation of 256 pictures of 256 tokens, kept for the backward pass
        _plane("checkpoint", "checkpoint_bf16_65536x1024", "bf16", 65536, 1024),
        # fp32 rows that end inside a block
        _plane("checkpoint", "checkpoint_f32_2056x1500", "f32", 2056, 1500),
        # one token against a wide weight: serving, where the weight's bytes count
        _linear("linear_one_row_bf16_4096x16384", "bf16", 1, 4096, 16384, act="gelu"),
        # the first product of DeiT-Ti's MLP in the published type, an odd number of packed queries
        _linear("linear_tiny_f32_1021x192x768", "f32", 1021, 192, 768, act="gelu"),
        # the first product of a wide model's MLP, a large batch: the largest
        _linear("linear_wide_bf16_65536x1024x4096", "bf16", 65536, 1024, 4096, act="gelu"),
        # DeiT-S in fp32, 16 pictures with their class tokens: the attention's projection in training
        _train("train_small_f32_4112x384x384", "f32", 4112, 384, 384),
        # nothing a multiple of anything
        _train("train_odd_bf16_2999x777x1301", "bf16", 2999, 777, 1301, bias=False),
        # a wide model's MLP in training
        _train("train_wide_bf16_32768x1024x4096", "bf16", 32768, 1024, 4096),
        # DeiT-S in fp32: the MLP's hidden layer
        _plane("gelu", "gelu_small_f32_4112x1536", "f32", 4112, 1536),
        # a wide model's hidden layer, a large batch
        _plane("gelu", "gelu_wide_bf16_65536x4096", "bf16", 65536, 4096),
        # DeiT-S in fp32: the norms of 16 pictures
        _plane("layer_norm", "norm_small_f32_4112x384", "f32", 4112, 384),
        # a wide model's, a large batch
        _plane("layer_norm", "norm_wide_bf16_65536x1024", "bf16", 65536, 1024),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, spread over the logarithm, hardly ever round."""
    return min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))


def _width(rng, low, high):
    n = _spread(rng, low, high)
    return -(-n // 64) * 64 if rng.random() < 0.5 else n


def draw(rng):
    op = rng.choice(["linear", "linear", "linear_train", "linear_train", "gelu", "layer_norm", "checkpoint"])
    dtype = rng.choice(["bf16", "f32"])
    if op in ("linear", "linear_train"):
        width, out = _width(rng, 32, 4096), _width(rng, 32, 16384 if op == "linear" else 4096)
        most = (65536 if op == "linear" else 32768) * 1024 * 4096 // 2
        rows = _spread(rng, 1, max(1, min(65536, most // (width * out))))
        bias = rng.random() < 0.7
        case = _linear("", dtype, rows, width, out, rng.choice(["none", "gelu"]), bias) if op == "linear" else _train("", dtype, rows, width, out, bias)
    else:
        width = _width(rng, 32, 4096)
        case = _plane(op, "", dtype, _spread(rng, 1, min(65536, 65536 * 1024 // width)), width)
    del case["name"]
    return case


# ------------------------------------------------------------------------------------------------ inputs
def _randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _inputs(case, seed):
    """-> the operands in 32 bits and the gradient that comes in (None where there is none)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, width = case["rows"], case["width"]
    # activations: some channels are far larger than others, and not around zero
    x = _randn(g, rows, width) * torch.exp(0.6 * _randn(g, width)) + 0.3 * _randn(g, width)
    if case["op"] == "checkpoint":
        return [x], None
    if case["op"] == "gelu":
        return [x], 1e-3 * _randn(g, rows, width)
    if case["op"] == "layer_norm":
        return [x, 1 + 0.2 * _randn(g, width), 0.2 * _randn(g, width)], 1e-3 * _randn(g, rows, width)
    w = _randn(g, case["out"], width) * (0.7 * width ** -0.5)
    b = 0.3 * _randn(g, case["out"]) if case["bias"] else None
    return [x, w, b], 1e-3 * _randn(g, rows, case["out"]) if case["op"] == "linear_train" else None


def prepare(case, seed):
    dtype = DTYPES[case["dtype"]]
    operands, grad = _inputs(case, seed)
    operands = [None if t is None else t.to(dtype) for t in operands]
    state = {"case": case, "operands": operands, "grad": None if grad is None else grad.to(dtype)}
    if case["op"] == "linear":
        # the weight as a program that serves it keeps it
        values, e = _quantized(operands[1].float())
        state["weight"] = values.to(torch.float8_e4m3fn), (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)
        if own:
            from vtpack_amd.layers import Blocks
            state["weight"] = Blocks(*state["weight"])
    elif grad is not None:
        state["leaves"] = [t.requires_grad_() for t in operands if t is not None]
    return state


# ------------------------------------------------------------------------------------------------ plain forms
def _blocks_of(x):
    """x [rows, n] filled up with zeros -> [rows, blocks, BLOCK]."""
    return torch.nn.functional.pad(x, (0, -x.shape[1] % BLOCK)).view(x.shape[0], -1, BLOCK)


def _quantized(x):
    """-> fp32 values (e4m3 numbers) [rows, n], exponents [rows, blocks]."""
    t = _blocks_of(x)
    m, e = torch.frexp(t.abs().amax(2))                  # m in [0.5, 1); 448 = 0.875 * 2^9
    e = (e - 9 + (m > 0.875)).clamp(min=LEAST)
    values = (t * torch.exp2(-e.float()).unsqueeze(2)).to(torch.float8_e4m3fn).float()
    return values.view(x.shape[0], -1)[:, :x.shape[1]], e


def _stands_for(values, e):
    return (_blocks_of(values.float()) * torch.exp2(e.float()).unsqueeze(2)).view(values.shape[0], -1)[:, :values.shape[1]]


def _q(x):
    return _stands_for(*_quantized(x))


def _phi(x):
    return 0.5 * torch.erfc(-x * math.sqrt(0.5))


def _plain(state):
    case, operands = state["case"], [None if t is None else t.detach().float() for t in state["operands"]]
    dtype, x = DTYPES[case["dtype"]], operands[0]
    if case["op"] == "checkpoint":
        return [_q(x).to(dtype)]
    if case["op"] == "linear":
        values, scales = state["weight"]
        w = _stands_for(values, scales.view(torch.uint8).int() - 127)
        y = _q(x) @ w.t()
        if operands[2] is not None:
            y = y + operands[2]
        return [(y * _phi(y) if case["act"] == "gelu" else y).to(dtype)]
    dy = state["grad"].float()
    if case["op"] == "linear_train":
        x8, w8, g = _q(x), _q(operands[1]), dy.to(torch.bfloat16).float()
        y = x8 @ w8.t()
        out = [g @ w8, g.t() @ x8]
        if operands[2] is not None:
            y, out = y + operands[2], out + [g.sum(0)]
        return [t.to(dtype) for t in [y] + out]
    if case["op"] == "gelu":
        c = _q(x)
        d = _phi(c) + c * torch.exp(-0.5 * c * c) * (0.5 / math.pi) ** 0.5
        return [(x * _phi(x)).to(dtype), (dy * d).to(dtype)]
    # (the mean next to the row's, whatever the order of the sum: what is rounded to 8 bits goes by it)
    c = x - x.double().mean(1, keepdim=True).float()
    r = torch.rsqrt((c * c).mean(1, keepdim=True) + EPS)
    h, g = _q(c) * r, dy * operands[1]
    dx = r * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
    return [t.to(dtype) for t in (c * r * operands[1] + operands[2], dx, (dy * h).sum(0), dy.sum(0))]


# ------------------------------------------------------------------------------------------------ the framework's
def _own(state):
    from vtpack_amd import layers
    case, (x, *rest) = state["case"], state["operands"]
    if case["op"] == "checkpoint":
        return [layers.quantize_blocks(x).dequantize(x.dtype)]
    if case["op"] == "linear":
        return [layers.linear_8bit(x, state["weight"], rest[1], act=case["act"])]
    if case["op"] == "linear_train":
        y = layers.linear_8bit(x, *rest)
    elif case["op"] == "gelu":
        y = layers.gelu_8bit(x)
    else:
        y = layers.layer_norm_8bit(x, *rest, eps=EPS)
    return [y.detach(), *torch.autograd.grad(y, state["leaves"], state["grad"])]


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------ what it has to do
def work(case):
    s, rows, width = 2 if case["dtype"] == "bf16" else 4, case["rows"], case["width"]
    n = rows * width
    kept = n + rows * -(-width // BLOCK)                 # bytes of the blocks, written and read again
    if case["op"] == "checkpoint":
        return {"bytes": 2 * n * s + 2 * kept, "flops": 4 * n}
    if case["op"] == "gelu":
        return {"bytes": 4 * n * s + 2 * kept, "flops": 40 * n}
    if case["op"] == "layer_norm":
        return {"bytes": 4 * n * s + 2 * kept + 4 * width * s, "flops": 20 * n}
    out, product = case["out"], 2 * n * case["out"]
    if case["op"] == "linear":
        return {"bytes": n * s + out * (width + -(-width // BLOCK)) + rows * out * s, "flops": product}
    return {"bytes": 2 * n * s + 2 * kept + 2 * out * width * s + 2 * rows * out * s, "flops": 3 * product}


# ------------------------------------------------------------------------------------------------ in 64 bits
def _nearest(x):
    """Q(x) of x (float64) from its definition, by logarithms."""
    out = torch.empty_like(x)
    for at in range(0, x.shape[1], BLOCK):
        t = x[:, at:at + BLOCK]
        e = torch.ceil(torch.log2(t.abs().amax(1, keepdim=True) / 448)).clamp(min=LEAST)
        v = t * torch.exp2(-e)
        step = torch.exp2(torch.floor(torch.log2(v.abs())).clamp(min=-6) - 3)
        out[:, at:at + BLOCK] = torch.round(v / step) * step * torch.exp2(e)
    return out


def exact(case, seed):
    dtype = DTYPES[case["dtype"]]
    operands, grad = _inputs(case, seed)
    x, *rest = [None if t is None else t.to(dtype).double() for t in operands]
    dy = None if grad is None else grad.to(dtype)
    if case["op"] == "checkpoint":
        return [_nearest(x)]
    if case["op"] == "gelu":
        c = _nearest(x)
        d = torch.special.ndtr(c) + c * torch.exp(-c * c / 2) / math.sqrt(2 * math.pi)
        return [x * torch.special.ndtr(x), dy.double() * d]
    if case["op"] == "layer_norm":
        mean = x.mean(1, keepdim=True).float()
        kept = _nearest((x.float() - mean).double())
        c, w, b, g = x - mean.double(), rest[0], rest[1], dy.double()
        r = 1 / torch.sqrt((c * c).mean(1, keepdim=True) + EPS)
        h, gw = kept * r, g * w
        dx = r * (gw - gw.mean(1, keepdim=True) - h * (gw * h).mean(1, keepdim=True))
        return [c * r * w + b, dx, (g * h).sum(0), g.sum(0)]
    w, b = rest
    x8, w8 = _nearest(x), _nearest(w)
    y = x8 @ w8.t().contiguous() + (0 if b is None else b)
    if case["op"] == "linear":
        return [y * torch.special.ndtr(y) if case["act"] == "gelu" else y]
    g = dy.to(torch.bfloat16).double()
    return [y, g @ w8, g.t().contiguous() @ x8] + ([] if b is None else [g.sum(0)])
