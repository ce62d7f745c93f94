"""Activations and weights in 8 bits: blocks of 128 numbers with a power of two, the Linear that multiplies them, and the Linear, GELU and
LayerNorm of a training step that keep their input in them (the reference keeps every activation in full, and has no 8-bit product).

A block is 128 consecutive numbers of the last dimension (the last of a row may be shorter): e4m3 values (OCP) and a power of two 2^e, e
the smallest whole number with max |x| 2^-e <= 448, -110 at least.  Values are rounded to nearest, ties to even, half a step being 2^-4
of a value from max |x| 2^-15 on and max |x| 2^-18 at most below.  Infinities and NaN become NaN and do not count in the maximum."""
import torch

from .. import _lib, ops

_ACTS = {"none": _lib.ACT_NONE, "gelu": _lib.ACT_GELU}
_BLOCK = 128


def _pitches(n):
    """Bytes of a row's values and of its scales (include/vtdge.h)."""
    blocks = -(-n // _BLOCK)
    return blocks * _BLOCK, -(-blocks // 4) * 4


class Blocks:
    """Numbers [..., n] in blocks, on a GPU.

    `values` float8_e4m3fn [..., n] and `scales` float8_e8m0fnu [..., ceil(n / 128)] are views of its memory; made from such a pair
    (of a checkpoint, say) it holds a copy.  A scale's byte b stands for 2^(b - 127), 255 for NaN."""

    __slots__ = ("_data", "_shape")

    def __init__(self, values, scales):
        ops._need_gpu(values, scales)
        if values.dtype != torch.float8_e4m3fn or scales.dtype != torch.float8_e8m0fnu:
            raise TypeError(f"values are {values.dtype} and scales {scales.dtype}, expected float8_e4m3fn and float8_e8m0fnu")
        if values.device != scales.device:
            raise TypeError(f"values are on {values.device}, scales on {scales.device}")
        if values.dim() < 1 or values.shape[-1] < 1 or tuple(scales.shape) != (*values.shape[:-1], -(-values.shape[-1] // _BLOCK)):
            raise ValueError(f"scales of {tuple(scales.shape)} do not fit values of {tuple(values.shape)}")
        self._shape = tuple(values.shape)
        rows, (value_pitch, scale_pitch) = self._rows(), _pitches(self._shape[-1])
        values, scales = (t.view(torch.uint8).reshape(rows, t.shape[-1]) for t in (values, scales))
        if values.shape[1] < value_pitch:
            values = torch.nn.functional.pad(values, (0, value_pitch - values.shape[1]))
        if scales.shape[1] < scale_pitch:
            scales = torch.nn.functional.pad(scales, (0, scale_pitch - scales.shape[1]), value=127)
        self._data = torch.cat([values.reshape(-1), scales.reshape(-1)])

    @classmethod
    def _of(cls, data, shape):
        self = cls.__new__(cls)
        self._data, self._shape = data, tuple(shape)
        return self

    def _rows(self):
        return torch.Size(self._shape[:-1]).numel()

    @property
    def shape(self):
        return torch.Size(self._shape)

    @property
    def device(self):
        return self._data.device

    def _view(self, at, pitch, n, dtype):
        rows = self._rows()
        return self._data[at:at + rows * pitch].view(rows, pitch)[:, :n].view(*self._shape[:-1], n).view(dtype)

    @property
    def values(self):
        return self._view(0, _pitches(self._shape[-1])[0], self._shape[-1], torch.float8_e4m3fn)

    @property
    def scales(self):
        value_pitch, scale_pitch = _pitches(self._shape[-1])
        return self._view(self._rows() * value_pitch, scale_pitch, -(-self._shape[-1] // _BLOCK), torch.float8_e8m0fnu)

    def dequantize(self, dtype=torch.float32):
        """The numbers, float32 or bfloat16 (both hold what `quantize_blocks` makes as it is)."""
        if dtype not in (torch.float32, torch.bfloat16):
            raise TypeError(f"vtdge kernels are built for float32 and bfloat16, got {dtype}")
        return _lib.training().dequantize_blocks(self._data, self._shape, dtype == torch.float32)

    def __repr__(self):
        return f"Blocks(shape={self._shape}, device='{self.device}')"


def _check_activation(x):
    if not torch.is_tensor(x):
        raise TypeError(f"expected a tensor, got {type(x).__name__}")
    ops._need_gpu(x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"expected [..., n] with n > 0, got {tuple(x.shape)}")
    if x.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"vtdge kernels are built for float32 and bfloat16, got {x.dtype}")


def quantize_blocks(x):
    """x [..., n], float32 or bfloat16 -> its `Blocks`.  No gradients pass."""
    data = _lib.training().quantize_blocks(x)
    if data is None:
        _check_activation(x)
        raise ValueError("quantize_blocks takes strided tensors")
    return Blocks._of(data, x.shape)


def linear_8bit(x, weight, bias=None, act="none"):
    """act(Q(x) Q(weight)^T + bias) of x's type, Q(.) the numbers that `quantize_blocks` makes.

    x [..., width], float32 or bfloat16; weight [out, width] of x's type, brought into blocks by every call, or `Blocks` of that shape,
    which a program makes once and hands to every call (x is brought into blocks by each; up to 16 rows of 16384 numbers in all read the weight as it
    lies, beyond that a float32 call expands it to bfloat16 first, at some four times the time of its bytes); bias [out] of x's type or None; act "none" or "gelu" (the latter without gradients:
    a training step takes `gelu_8bit`).  Sums are fp32; for bfloat16 results the matrix instructions cut the products of eight neighbours 13 bits
    below the largest of them first: some 2e-5 of the results in the 2-norm, 7 2^-13 of the largest product of each eight at worst.

    Gradients, with g the gradient of the result rounded to bfloat16: dx = g Q(weight), dweight = g^T Q(x), dbias the sum of g over the
    rows.  For them the call keeps Q(x) and Q(weight), a byte a number, and neither x nor weight; weight given as `Blocks` has none.  Traces
    (torch.jit.trace, make_fx), forward-mode derivatives and gradients of the gradients are refused."""
    if act not in _ACTS:
        raise ValueError(f"act is {act!r}, expected 'none' or 'gelu'")
    kept = isinstance(weight, Blocks)
    y = None
    if not kept:
        y = _lib.training().linear_8bit(x, weight, None, bias, _ACTS[act])
    elif len(weight._shape) == 2 and torch.is_tensor(x) and x.shape[-1:] == weight._shape[1:]:
        y = _lib.training().linear_8bit(x, weight._data, weight._shape[0], bias, _ACTS[act])
    if y is not None:
        return y
    _check_activation(x)
    if not kept and not torch.is_tensor(weight):
        raise TypeError(f"expected a weight, got {type(weight).__name__}")
    shape = tuple(weight.shape)
    if len(shape) != 2 or 0 in shape or x.shape[-1] != shape[1]:
        raise ValueError(f"weight {shape} does not take inputs of width {x.shape[-1]}")
    if kept:
        if weight.device != x.device:
            raise TypeError(f"weight is on {weight.device} but the activation is on {x.device}")
        ops._check_like(x, bias=bias)
    else:
        ops._need_gpu(weight, bias)
        ops._check_like(x, weight=weight, bias=bias)
    ops._check_vector("bias", bias, shape[0])
    raise ValueError("linear_8bit takes strided tensors")


def gelu_8bit(x):
    """GELU(x) = x Phi(x) of x [..., n], float32 or bfloat16.  For the gradient it keeps Q(x) alone (see `quantize_blocks`), a byte a number:
    dx = dy (Phi(c) + c phi(c)) with c = Q(x).  bfloat16: Phi is within 3e-4 of its value for x >= -10 (7.2e-5 from -4 on) and below 1e-23 further out, the
    slope within 4e-5 of its value and 2e-6; float32: 3.2e-8 and 6.4e-8 in the 2-norm over unit normals.  Refused as `linear_8bit` does: traces,
    forward mode, second order."""
    y = _lib.training().gelu_8bit(x)
    if y is None:
        _check_activation(x)
        raise ValueError("gelu_8bit takes strided tensors")
    return y


def layer_norm_8bit(x, weight, bias, eps=1e-6):
    """LayerNorm of x [..., n] over its last dimension, n up to 8192, weight and bias [n]; all float32 or all bfloat16.

    For the gradients it keeps Q(x - mean), a byte a number, and each row's 1 / sqrt(var + eps): with h their product and g = dy weight,
    dx = rstd (g - mean g - h mean(g h)), dweight = sum dy h, dbias = sum dy.  The mean is the float32 number next to the row's.  Refused as
    `linear_8bit` does: traces, forward mode, second order."""
    y = _lib.training().layer_norm_8bit(x, weight, bias, eps)
    if y is not None:
        return y
    _check_activation(x)
    n = x.shape[-1]
    if n > 8192:
        raise ValueError(f"layer_norm_8bit takes rows of up to 8192, got {n}")
    if not torch.is_tensor(weight) or not torch.is_tensor(bias):
        raise TypeError("weight and bias have to be tensors")
    if not isinstance(eps, (int, float)) or not eps >= 0:
        raise ValueError(f"eps is {eps}, expected a number from 0 on")
    ops._need_gpu(weight, bias)
    ops._check_like(x, weight=weight, bias=bias)
    ops._check_vector("weight", weight, n)
    ops._check_vector("bias", bias, n)
    y = _lib.training().layer_norm_8bit(x, weight, bias, float(eps))
    if y is None:
        raise ValueError("layer_norm_8bit takes strided tensors")
    return y


def require_plain_module(module):
    """A TypeError unless `call_8bit` can stand in for the module: a Linear, a LayerNorm over the last dimension with weight and bias, or an
    exact GELU, without hooks of its own."""
    hooks = ("_forward_hooks", "_forward_pre_hooks", "_backward_hooks", "_backward_pre_hooks")
    plain = (type(module) in (torch.nn.Linear, torch.nn.LayerNorm, torch.nn.GELU) and "forward" not in vars(module)
             and not any(getattr(module, h, None) for h in hooks))
    if plain and isinstance(module, torch.nn.LayerNorm):
        plain = len(module.normalized_shape) == 1 and module.weight is not None and module.bias is not None
    if plain and isinstance(module, torch.nn.GELU):
        plain = module.approximate == "none"
    if not plain:
        raise TypeError(f"{module} is more than a plain Linear, LayerNorm or GELU, which the operators on 8-bit blocks stand in for")


def call_8bit(module, x):
    """module(x) by `linear_8bit`, `layer_norm_8bit` or `gelu_8bit` (see `require_plain_module`)."""
    require_plain_module(module)
    if isinstance(module, torch.nn.Linear):
        return linear_8bit(x, module.weight, module.bias)
    if isinstance(module, torch.nn.LayerNorm):
        return layer_norm_8bit(x, module.weight, module.bias, module.eps)
    return gelu_8bit(x)


def call(module, x):
    return module(x)
