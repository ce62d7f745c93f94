"""The losses of a training step behind the encoder: the classifier's cross entropy (the reference trains with timm's, main.py:346-352,
on the logits of `model.head`) and the balance of the routers' gates, which stands beside the budget loss of the harness."""
import torch

from .. import _lib, ops


def linear_cross_entropy(x, weight, bias, target, ignore_index=-100, label_smoothing=0.0, reduction="mean"):
    """`F.cross_entropy(F.linear(x, weight, bias), target, ...)` with its gradients, without the logits in memory (see below for
    float32).

    x [..., width], weight [classes, width], bias [classes] or None, all float32 or all bfloat16; target int64 of x's leading
    shape.  -> float32: the mean over the rows that count ("mean"), their sum ("sum"), or every row's own ("none", of target's
    shape).  A row whose target is `ignore_index` is left out, whatever its features hold; so is one whose target is no class
    (F.cross_entropy stops the program there).  Without a row that counts the loss is 0, and so are the gradients.  Traces
    (torch.jit.trace, make_fx), forward-mode derivatives and gradients of the gradients are refused.

    The logits are fp32 sums and are not rounded; in bfloat16 the gradients of the logits are, once, before the products that
    take them to x, weight and bias.  They work in pieces of the classes with some 320 MB of scratch for a piece (more for
    over 160 000 rows, float32 50 000: a piece has 1024 classes at least, or all of them rounded up to 256); float32 operands are
    laid out anew in three parts of two bytes, which stay for the gradients, with logits of up to 256 MB, where all of it is no
    more than 320 MB.  Finite float32 values are multiplied to 24 bits, those below 2^-110 to within 2^-134; the logits that an
    infinity in weight or in a row that counts meets may be NaN where float32 products make an infinity; one in the bias is added
    as it is."""
    how = (ignore_index, label_smoothing, ops.REDUCTIONS.get(reduction))
    loss = _lib.training().linear_cross_entropy(x, weight, bias, target, *how)
    if loss is not None:
        return loss
    # operands that are not the kernels' rows and vectors yet, or none that they can become
    ops._need_gpu(x, weight, bias, target)
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"reduction is {reduction!r}, expected 'mean', 'sum' or 'none'")
    if not 0.0 <= label_smoothing <= 1.0:
        raise ValueError(f"label_smoothing is {label_smoothing}, expected 0 .. 1")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1] or 0 in weight.shape:
        raise ValueError(f"features {tuple(x.shape)} do not match a weight of {tuple(weight.shape)}")
    if x.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"vtdge kernels are built for float32 and bfloat16, got {x.dtype}")
    ops._check_like(x, weight=weight, bias=bias)
    ops._check_vector("bias", bias, weight.shape[0])
    if target.dtype != torch.int64 or target.device != x.device:
        raise TypeError(f"target is {target.dtype} on {target.device}, expected int64 on {x.device}")
    if target.shape != x.shape[:-1]:
        raise ValueError(f"target has shape {tuple(target.shape)}, expected {tuple(x.shape[:-1])}")
    if x.numel() == 0:                           # no row: a loss of 0 that still belongs to its operands
        zero = (x.sum() + weight[:0].sum() + (0 if bias is None else bias[:0].sum())).float()
        return zero if reduction != "none" else zero.expand(target.shape)
    loss = _lib.training().linear_cross_entropy(ops._rows_of(x), ops._rows_of(weight), None if bias is None else bias.contiguous(),
                                                target.reshape(-1).contiguous(), int(ignore_index), float(label_smoothing), how[2])
    if loss is None:
        raise ValueError("linear_cross_entropy takes strided tensors")
    return loss.view(target.shape) if reduction == "none" and target.dim() != 1 else loss


def require_plain_head(head):
    """A TypeError unless a model's classifier is what `linear_cross_entropy` of its weight and bias is."""
    hooks = ("_forward_hooks", "_forward_pre_hooks", "_backward_hooks", "_backward_pre_hooks")
    if (not isinstance(head, torch.nn.Linear) or type(head).forward is not torch.nn.Linear.forward or "forward" in vars(head)
            or any(getattr(head, h, None) for h in hooks)):
        raise TypeError("the model's head is more than a Linear without hooks, and its loss would read the weight and bias alone: take "
                        "F.cross_entropy of the logits, model(images)")


def gate_balance(gate, indices=None, top_k=1, mask=None):
    """How evenly a router's choices fall on its experts (here: granularities): -> (loss, counts).

    gate [..., E] (1 .. 512 logits a token, float32 or bfloat16); loss = E sum_e f_e P_e in float32, f_e the fraction of the choices that
    fell on e and P_e the mean softmax probability of e, with the gradient through P; counts int64 [E] are the choices.  1 is
    even, E is all on one.  The choices are the `top_k` largest logits of a token (among equals the lowest index), or `indices`
    int64 [..., k] (or of gate's leading shape, k = 1) if they were made elsewhere, as by a Gumbel sample; one that is no expert is
    not counted.  `mask` (bool, gate's leading shape): False leaves a token out, whatever its logits are; a token whose logits are
    all -inf is left out too.  Without a token the loss is 0.  Refused as `linear_cross_entropy` does: traces, forward mode, second order."""
    out = _lib.training().balance(gate, indices, mask, top_k) if indices is None else None
    if out is not None:
        return out
    ops._need_gpu(gate, indices, mask)
    if gate.dim() < 1 or not 1 <= gate.shape[-1] <= 512:
        raise ValueError(f"gate has shape {tuple(gate.shape)}, expected 1 .. 512 logits a token")
    if gate.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"vtdge kernels are built for float32 and bfloat16, got {gate.dtype}")
    E, lead = gate.shape[-1], gate.shape[:-1]
    if indices is not None:
        if indices.dtype != torch.int64 or indices.device != gate.device:
            raise TypeError(f"indices are {indices.dtype} on {indices.device}, expected int64 on {gate.device}")
        if indices.shape == lead:
            indices = indices.unsqueeze(-1)
        if indices.shape[:-1] != lead or not 1 <= indices.shape[-1] <= 512:
            raise ValueError(f"indices of shape {tuple(indices.shape)} do not match a gate of {tuple(gate.shape)}")
        top_k = indices.shape[-1]
        indices = indices.reshape(-1, top_k).contiguous()
    elif not 1 <= top_k <= E:
        raise ValueError(f"top_k is {top_k}, expected 1 .. {E}")
    if mask is not None:
        if mask.dtype != torch.bool or mask.device != gate.device:
            raise TypeError(f"mask is {mask.dtype} on {mask.device}, expected bool on {gate.device}")
        if mask.shape != lead:
            raise ValueError(f"mask has shape {tuple(mask.shape)}, expected {tuple(lead)}")
        mask = mask.reshape(-1).contiguous()
    if gate.numel() == 0:
        return gate.sum().float(), torch.zeros((E,), dtype=torch.int64, device=gate.device)
    out = _lib.training().balance(ops._rows_of(gate), indices, mask, int(top_k))
    if out is None:
        raise ValueError("gate_balance takes strided tensors")
    return out
