"""The AdamW step of the reference's training runs (main.py:339-343: `create_optimizer`, `adamw` by default) as one kernel over all
weights, with moments in 32 or in 8 bits.
"""
import itertools
import operator

import numpy as np
import torch
from torch.autograd.graph import increment_version

from . import _lib, ops

__all__ = ["AdamW"]

BLOCK = 256                                    # elements that share a scale
_CODES = {"exp_avg": torch.float8_e4m3fn, "exp_avg_sq": torch.float8_e5m2}
_KEYS = {32: ("exp_avg", "exp_avg_sq"), 8: ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")}
_grad = operator.attrgetter("grad")
_ptr, _dense = torch.Tensor.data_ptr, torch.Tensor.is_contiguous


def _same_layout(a, b):
    return a.shape == b.shape and (a.stride() == b.stride() or a.is_contiguous() and b.is_contiguous())


class _Batch:
    """Weights of one type, device and count of steps, as the rows of the table the library reads.  Every step looks again at all
    that a program can put in another's place: the weights' memory, type, sizes and strides, the tensors in `state` and theirs, the
    gradients."""

    def __init__(self, params, states, bits, skipped):
        self.params, self.states, self.skipped, self.keys = params, states, skipped, _KEYS[bits]
        self.moments = [[s[k] for s in states] for k in self.keys]
        self.tensors = list(itertools.chain(params, *self.moments))
        self.at = _lib.training().places(self.tensors)
        self.plain = all(p.is_contiguous() for p in params)
        self.table = np.zeros((len(params), 7), dtype=np.uint64)
        self.table[:, 0] = [p.data_ptr() for p in params]
        for column, moment in enumerate(self.moments):
            self.table[:, 2 + column] = [t.data_ptr() for t in moment]
        self.table[:, 6] = [p.numel() for p in params]

    def holds(self):
        return (all(all(map(operator.is_, map(operator.itemgetter(k), self.states), old)) for k, old in zip(self.keys, self.moments))
                and _lib.training().places(self.tensors) == self.at)

    def take_gradients(self, grads):
        if not _lib.training().alike(grads, self.params):
            for g, p in zip(grads, self.params):
                if g.dtype != p.dtype or g.shape != p.shape or g.device != p.device:
                    raise ValueError(f"a gradient of {g.dtype} {tuple(g.shape)} on {g.device} for a weight of {p.dtype} {tuple(p.shape)} on {p.device}")
            raise ValueError("AdamW: sparse gradients are not supported")
        if not self.plain or not all(map(_dense, grads)):
            grads = [g if _same_layout(g, p) else torch.empty_like(p).copy_(g) for g, p in zip(grads, self.params)]
        self.table[:, 1] = list(map(_ptr, grads))
        return grads


class AdamW(torch.optim.Optimizer):
    """AdamW with decoupled weight decay (`torch.optim.AdamW` without `amsgrad` and `maximize`) over float32 or bfloat16 weights on
    the GPU, one launch for each 134 tensors (96 with 8-bit moments):

        p *= 1 - lr weight_decay;   m = beta1 m + (1 - beta1) g;   v = beta2 v + (1 - beta2) g^2
        p -= lr / (1 - beta1^t) * m / (sqrt(v / (1 - beta2^t)) + eps)

    `state_bits=8` keeps the moments in a byte each: `exp_avg` as float8_e4m3fn, `exp_avg_sq` as float8_e5m2, each with an fp32
    scale for every 256 consecutive elements of a weight (`exp_avg_scale`, `exp_avg_sq_scale`; element i of a weight stands for
    code[i] * scale[i // 256]).  They are rounded down or up by a hash of the element's place and the step, so that they follow
    slow changes on average, and are the same on every run.  With 32 they are float32, for bfloat16 weights too; those are
    rounded to the nearest, and changes below half a step of theirs are lost, as in torch.

    The group's `"step"` counts the steps; a weight's own count, t, leaves out those it had no gradient for (`"skipped"` in its
    state).  `capturable=True` keeps the count on the device, and `step()` may be captured into a graph once one step has been
    made without: `lr` may then be a float32 tensor of one element on that device, read at every replay.  A replay moves weights
    without torch's knowledge, so that what is derived from them is made anew only after `ops.invalidate_packed`.

    Gradients are read where they lie and have their weight's type; one of other strides than its weight is copied first.
    Refused: types the kernels do not have, sparse gradients, weights with gaps between their elements, weights of a group that lie over
    each other.  A group that is refused is as it was; others may have taken their step."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, capturable=False):
        if torch.is_tensor(lr):
            if not capturable:
                raise ValueError("lr as a tensor goes with capturable=True")
            if lr.dtype != torch.float32 or lr.numel() != 1 or not lr.is_cuda:
                raise ValueError(f"lr is {lr.dtype} {tuple(lr.shape)} on {lr.device}, expected one float32 value on the GPU")
        elif not lr >= 0.0:
            raise ValueError(f"lr is {lr}, expected 0 or more")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise ValueError(f"betas are {tuple(betas)}, expected [0, 1)")
        if not (eps >= 0.0 and weight_decay >= 0.0):
            raise ValueError(f"eps is {eps} and weight_decay {weight_decay}, expected 0 or more")
        if state_bits not in _KEYS:
            raise ValueError(f"state_bits is {state_bits}, expected 32 or 8")
        self._batches, self._natives = {}, {}
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      capturable=capturable, step=0))

    def __setstate__(self, state):
        super().__setstate__(state)
        self._batches, self._natives = {}, {}

    def load_state_dict(self, state_dict):
        """As torch's, but moments keep the type they were saved in (torch casts them to the weight's)."""
        self._batches, self._natives = {}, {}
        super().load_state_dict(state_dict)
        saved = [i for g in state_dict["param_groups"] for i in g["params"]]
        for i, p in zip(saved, (p for g in self.param_groups for p in g["params"])):
            if i in state_dict["state"]:
                self.state[p] = {k: v.detach().to(p.device, copy=True) if torch.is_tensor(v) else v
                                 for k, v in state_dict["state"][i].items()}

    # ---------------------------------------------------------------- what a step works on
    @staticmethod
    def _lay_out(p, bits, skipped):
        """The state of a weight before its first step."""
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW: make one step before the capture; it lays out the moments")
        if bits == 32:
            state = {k: torch.zeros_like(p, dtype=torch.float32, requires_grad=False) for k in _CODES}
        else:
            state = {k: torch.zeros_like(p, dtype=torch.uint8, requires_grad=False).view(t) for k, t in _CODES.items()}
            for k in _CODES:
                state[k + "_scale"] = torch.zeros((-(-p.numel() // BLOCK),), dtype=torch.float32, device=p.device)
        state["skipped"] = skipped
        return state

    @staticmethod
    def _check(p, grad, state, bits):
        if grad.is_sparse or grad.layout != torch.strided:
            raise ValueError("AdamW: sparse gradients are not supported")
        if p.dtype not in (torch.float32, torch.bfloat16):
            raise TypeError(f"vtdge kernels are built for float32 and bfloat16, got a weight of {p.dtype}")
        ops._need_gpu(p)
        if not p.is_contiguous() and torch.empty_like(p).stride() != p.stride():
            raise ValueError(f"a weight of shape {tuple(p.shape)} and strides {p.stride()} has gaps between its elements")
        for k, code in _CODES.items():
            m, want = state.get(k), torch.float32 if bits == 32 else code
            if m is None or m.dtype != want or m.device != p.device or not _same_layout(m, p):
                raise ValueError(f"state {k} does not fit its weight: expected {want} laid out as {tuple(p.shape)} / {p.stride()} on {p.device}, got "
                                 + ("none" if m is None else f"{m.dtype} {tuple(m.shape)} / {m.stride()} on {m.device}"))
            if bits == 8:
                s, n = state.get(k + "_scale"), -(-p.numel() // BLOCK)
                if s is None or s.dtype != torch.float32 or tuple(s.shape) != (n,) or not s.is_contiguous() or s.device != p.device:
                    raise ValueError(f"state {k}_scale does not fit its weight: expected float32 ({n},) on {p.device}")

    def _split(self, group, params, grads):
        """The batches of a group's weights that have a gradient."""
        bits, sets = group["state_bits"], {}
        for p, g in zip(params, grads):
            ops._need_gpu(p)
            state = self.state[p]
            if not any(k in state for k in _CODES):
                state.update(self._lay_out(p, bits, int(group["step"])))
            self._check(p, g, state, bits)
            sets.setdefault((p.dtype, p.device, state.get("skipped", 0)), []).append(p)
        lie = sorted((p.device.index, p.data_ptr(), p.data_ptr() + p.nbytes) for p in params if p.numel())
        if any(a[0] == b[0] and b[1] < a[2] for a, b in zip(lie, lie[1:])):
            raise ValueError("AdamW: weights that lie over each other, or one twice in a group, cannot be moved in one step")
        if group["capturable"] and len({d for _, d, _ in sets}) > 1:
            raise ValueError("AdamW: a capturable group keeps its count of steps on one device")
        return [_Batch(ps, [self.state[p] for p in ps], bits, skipped) for (_, _, skipped), ps in sets.items()]

    def _held(self, index, group, params):
        """The batches of the group's last step that was not one call, where they still hold."""
        kept = self._batches.get(index)
        if kept is not None:
            states, batches, old = kept
            now = list(self.state.values())
            if (len(params) == len(old) and all(map(operator.is_, params, old)) and len(now) == len(states)
                    and all(map(operator.is_, now, states)) and all(b.holds() and b.keys == _KEYS[group["state_bits"]] for b in batches)):
                return batches
        return None

    def _of_group(self, index, group, params, grads):
        batches = self._split(group, params, grads)
        self._batches = {i: b for i, b in self._batches.items() if i != index}
        self._batches[index] = (list(self.state.values()), batches, list(params))
        return batches

    # ---------------------------------------------------------------- the step
    def step(self, closure=None):
        """One step over all weights that have a gradient.  `closure` (optional) works the loss out again and returns it."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        rest = [(i, g) for i, g in enumerate(self.param_groups) if not self._in_one_call(i, g, g["params"])]
        if rest:
            self._step_groups(rest)
        return loss

    @torch.no_grad()
    def _step_groups(self, groups):
        """The step of groups that have to be looked over.  A group's weights, gradients and states are all looked at before the first
        launch, so that one that is refused is as it was; those before it have taken their step."""
        capturing = torch.cuda.is_available() and torch.cuda.is_current_stream_capturing()
        for index, group in groups:
            params = group["params"]
            grads = list(map(_grad, params))
            if capturing and not group["capturable"]:
                raise RuntimeError("AdamW: a step that is captured needs capturable=True (its count of steps would stand still)")
            missing = []
            if not all(map(operator.is_not, grads, itertools.repeat(None))):
                params = [p for p, g in zip(params, grads) if g is not None]
                if not params:
                    continue
                missing = [p for p, g in zip(group["params"], grads) if g is None and any(k in self.state.get(p, ()) for k in _CODES)]
                if missing and capturing:
                    raise RuntimeError("AdamW: a weight that has taken steps has no gradient in the one that is captured")
                grads = [g for g in grads if g is not None]
            batches = self._held(index, group, params)
            if batches is None:
                if not capturing and (params is not group["params"] and self._in_one_call(index, group, params)
                                      or self._in_one_call(index, group, params, anew=True)):
                    self._skip(index, missing)
                    continue
                batches = self._of_group(index, group, params, grads)
            of = dict(zip(map(id, params), grads)) if len(batches) > 1 else None
            held = [b.take_gradients(grads if of is None else [of[id(p)] for p in b.params]) for b in batches]
            for i, b in enumerate(batches):
                self._launch(group, b, i + 1 == len(batches))
            del held                                           # (what was laid out anew is read behind the launch)
            if not group["capturable"]:
                group["step"] += 1
            increment_version(params)
            self._skip(index, missing)

    def _in_one_call(self, index, group, params, anew=False):
        """The step of a group's weights in one native call that looks all of them over and launches; False, and nothing done, where
        something is not as it was when the call was prepared, which `anew` does again, or not as it takes it."""
        if group["capturable"] or _lib.timer is not None:
            return False
        native, bits = _lib.training(), group["state_bits"]
        if anew:
            for p in params:
                ops._need_gpu(p)
            states = [self.state[p] for p in params]
            for p, state in zip(params, states):
                if not any(k in state for k in _CODES):
                    state.update(self._lay_out(p, bits, int(group["step"])))
            # the native call meets the states in the order of their weights
            at = {id(p): i for i, p in enumerate(params)}
            order = [at[id(p)] for p in self.state if id(p) in at]
            if order != list(range(len(params))):
                for p, state in zip(params, states):
                    del self.state[p]
                    self.state[p] = state
            skipped = {state.get("skipped", 0) for state in states}
            batch = native.adamw_batch(params, states, list(_KEYS[bits]), bits) if len(skipped) == 1 else None
            self._natives = {i: b for i, b in self._natives.items() if i != index}
            if batch is None:
                return False
            self._natives[index] = (batch, skipped.pop(), bits, list(params))
        batch, skipped, kept_bits, _ = self._natives.get(index, (None, 0, 0, ()))
        beta1, beta2 = group["betas"]
        if kept_bits != bits or not native.adamw_step(batch, params, self.state, group["lr"], beta1, beta2, group["eps"], group["weight_decay"],
                                                      int(group["step"]) + 1 - skipped, bits):
            return False
        group["step"] += 1
        return True

    def _skip(self, index, params):
        """Weights with states and without a gradient have missed this step.  What was prepared for others only is good for the next
        one too; with one of these in it, its count of steps is no longer theirs."""
        for p in params:
            self.state[p]["skipped"] = self.state[p].get("skipped", 0) + 1
        missed = set(map(id, params))
        for prepared in (self._batches, self._natives):
            if index in prepared and not missed.isdisjoint(map(id, prepared[index][-1])):
                del prepared[index]

    def _launch(self, group, batch, last):
        (b1, b2), eps, decay = group["betas"], group["eps"], group["weight_decay"]
        first, lr, step, scalars = batch.params[0], group["lr"], 0, None
        with ops._on(first):
            if group["capturable"]:
                if not torch.is_tensor(group["step"]):
                    group["step"] = torch.tensor([group["step"]], dtype=torch.int64, device=first.device)
                if group["step"].device != first.device or torch.is_tensor(lr) and lr.device != first.device:
                    raise ValueError(f"AdamW: the count of steps and lr have to be on {first.device}, as the weights are")
                scalars = torch.empty((_lib.ADAMW_SCALARS,), dtype=torch.uint8, device=first.device)
                held = lr if torch.is_tensor(lr) else None
                lr = 0.0 if held is not None else float(lr)
                _lib.call("vtdge_adamw_scalars", ops.ptr(group["step"]), batch.skipped, int(last), ops.ptr(held), lr, b1, b2, eps, decay,
                          ops.ptr(scalars), ops.stream_ptr(), tag=("adamw_scalars",))
            else:
                step = int(group["step"]) + 1 - batch.skipped
            _lib.call("vtdge_adamw", batch.table.ctypes.data, len(batch.params), float(lr), b1, b2, eps, decay, step, ops.ptr(scalars),
                      ops.dtype_code(first), group["state_bits"], ops.stream_ptr(), tag=("adamw", group["state_bits"]))
