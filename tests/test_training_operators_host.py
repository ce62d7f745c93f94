"""The operators of a training step without a GPU: what they refuse, and the checks of the library's arguments."""
import ctypes

import pytest
import torch

from vtpack_amd import _lib
from vtpack_amd.layers import gate_balance, linear_cross_entropy
from vtpack_amd.optim import AdamW


def test_tensors_on_the_cpu_are_refused():
    x, w, t = torch.randn(4, 8), torch.randn(3, 8), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="GPU only"):
        linear_cross_entropy(x, w, None, t)
    with pytest.raises(RuntimeError, match="GPU only"):
        gate_balance(x)
    p = torch.nn.Parameter(x)
    p.grad = x.clone()
    with pytest.raises(RuntimeError, match="GPU only"):
        AdamW([p]).step()


@pytest.mark.parametrize("kw", [{"lr": -1.0}, {"betas": (1.0, 0.9)}, {"betas": (0.9, -0.1)}, {"eps": -1e-8}, {"weight_decay": -1.0},
                                {"state_bits": 16}, {"lr": torch.tensor(1e-3)}, {"lr": torch.tensor(1e-3), "capturable": True},
                                {"lr": float("nan")}])
def test_settings_of_the_optimizer(kw):
    with pytest.raises(ValueError):
        AdamW([torch.nn.Parameter(torch.zeros(3))], **kw)


def test_a_step_without_gradients_does_nothing():
    opt = AdamW([torch.nn.Parameter(torch.zeros(3))])
    assert opt.step(lambda: 5.0) == 5.0 and opt.param_groups[0]["step"] == 0


def test_state_dict_round_trip_without_steps():
    p = torch.nn.Parameter(torch.zeros(3))
    opt = AdamW([p], lr=0.5, state_bits=8)
    other = AdamW([p])
    other.load_state_dict(opt.state_dict())
    assert other.param_groups[0]["state_bits"] == 8 and other.param_groups[0]["lr"] == 0.5


class _Tensor(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("param", "grad", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")] + [("n", ctypes.c_int64)]


def test_arguments_of_the_library():
    """Before anything is launched."""
    lib = _lib.load()
    p = 4096                                              # never read: the sizes are refused first
    ce = [p, 8, p, 8, p, p, 4, 3, 8, -100, 0.0, p, 1 << 40, 0, p, p, p, p, p, 0, None]

    def call(**put):
        args = list(ce)
        for i, v in put.items():
            args[int(i[1:])] = v
        return lib.vtdge_cross_entropy(*args)

    assert call(_0=None) == _lib.ERR_ARG and b"NULL" in lib.vtdge_last_error()
    assert call(_19=7) == _lib.ERR_ARG                    # type
    assert call(_1=7) == _lib.ERR_ARG                     # rows that overlap
    assert call(_6=0) == _lib.ERR_ARG and call(_7=0) == _lib.ERR_ARG and call(_8=0) == _lib.ERR_ARG
    assert call(_6=1 << 24) == _lib.ERR_UNSUPPORTED and call(_8=(1 << 16) + 1) == _lib.ERR_UNSUPPORTED
    assert call(_10=1.5) == _lib.ERR_ARG and call(_10=float("nan")) == _lib.ERR_ARG
    assert call(_12=0) == _lib.ERR_ARG and b"workspace" in lib.vtdge_last_error()
    assert call(_11=p + 16) == _lib.ERR_ARG               # a workspace off its boundary
    assert call(_17=None) == _lib.ERR_ARG                 # a count of rows without their mean
    assert lib.vtdge_cross_entropy_workspace(4, 3, 0, 0, 0) == -1
    back = [p, 8, p, 8, p, p, p, p, p, 1, p, 4, 3, 8, -100, 0.0, None, p, 1 << 40, p, p, p, 0, None]
    assert lib.vtdge_cross_entropy_backward(*back) == _lib.ERR_ARG and b"grad_stride" in lib.vtdge_last_error()
    gb = [p, 3, None, None, 100, 3, 1, None, 0, p, p, p, 0, None]
    for i, v, want in ((4, 0, -1), (5, 0, -1), (5, 513, -1), (6, 4, -1), (6, 0, -1), (1, 2, -1), (12, 5, -1), (4, 1 << 31, -2), (4, 100000, -1)):
        args = list(gb)
        args[i] = v
        assert lib.vtdge_gate_balance(*args) == want, (i, v)
    args = list(gb)
    args[1] = args[5] = 513
    assert lib.vtdge_gate_balance(*args) == _lib.ERR_UNSUPPORTED
    table = (_Tensor * 1)(_Tensor(p, p, p, p, None, None, 10))
    at = ctypes.addressof(table)
    adamw = [at, 1, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, None, 0, 32, None]
    for i, v, want in ((1, -1, -1), (2, -1.0, -1), (3, 1.0, -1), (4, 1.5, -1), (5, -1.0, -1), (6, -1.0, -1), (7, 0, -1), (9, 3, -1), (10, 16, -2),
                       (10, 8, -1)):                     # (8-bit moments without scales)
        args = list(adamw)
        args[i] = v
        assert lib.vtdge_adamw(*args) == want, (i, v)
    assert lib.vtdge_adamw(None, 0, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, None, 0, 32, None) == 0
    table[0].n = 0
    table[0].param = None
    assert lib.vtdge_adamw(*adamw) == 0                   # nothing to do, nothing touched
    assert lib.vtdge_adamw_scalars(None, 0, 1, None, 1e-3, 0.9, 0.999, 1e-8, 0.0, p, None) == _lib.ERR_ARG


def test_workspaces_follow_the_sizes():
    lib = _lib.load()
    size = lib.vtdge_cross_entropy_workspace
    assert size(256, 1000, 384, 1, 0) % 256 == 0 and size(256, 1000, 384, 1, 0) < size(256, 1000, 384, 0, 0)
    # operands that are read where they lie need no room: forward neither, for the gradients x all the same
    full, x, w = size(256, 1000, 384, 1, 0), 256 * 384 * 2, 1000 * 384 * 2
    assert full - size(256, 1000, 384, 1, 2) == x and full - size(256, 1000, 384, 1, 4) == w and full - size(256, 1000, 384, 1, 6) == x + w
    assert size(256, 1000, 384, 1, 1) == size(256, 1000, 384, 1, 3) == size(256, 1000, 384, 1, 7) + w
    # kept logits: fp32, up to 256 MB
    assert size(256, 1001, 384, 0, 8) - size(256, 1001, 384, 0, 0) == 256 * 1008 * 4 and size(256, 1001, 384, 1, 8) == size(256, 1001, 384, 1, 0)
    assert size(1024, 65537, 64, 0, 8) == size(1024, 65537, 64, 0, 0) and size(1024, 65536, 64, 0, 8) - size(1024, 65536, 64, 0, 0) == 256 << 20
    # d of a piece: no more than 320 MB, or 1024 classes, however many classes there are
    assert size(8192, 65536, 1024, 1, 1) < (320 << 20) + 2 * 65536 * 1024 * 2 + 3 * 8192 * 1024 * 4 + (8 << 20) * 4 * 2
    assert lib.vtdge_gate_balance_workspace(100, 8) == 0 and lib.vtdge_gate_balance_workspace(1 << 20, 8) == 256 * 17 * 4


def test_the_native_module_is_named_when_it_is_missing(monkeypatch):
    import sys
    import vtpack_amd
    monkeypatch.setattr(_lib, "_training", None)
    monkeypatch.delattr(vtpack_amd, "_training", raising=False)
    monkeypatch.setitem(sys.modules, "vtpack_amd._training", None)
    with pytest.raises(ImportError, match="_training.so is missing"):
        _lib.training()


def test_arguments_of_the_native_module():
    """Operands it does not take as they are come back as None, for Python to name what is wrong; nothing else passes either."""
    native = _lib.training()
    x, t = torch.randn(4, 8), torch.zeros(4, dtype=torch.int64)
    assert native.linear_cross_entropy(x, x, None, t, -100, 0.0, 1) is None
    assert native.linear_cross_entropy(x, x, None, t, -100, 0.0, None) is None
    assert native.linear_cross_entropy("x", x, None, t, -100, 0.0, 1) is None
    assert native.balance(x, None, None, 1) is None and native.balance(None, None, None, 1) is None
    for name in ("linear_cross_entropy", "cross_entropy", "cross_entropy_backward", "balance", "gate_balance", "gate_balance_backward",
                 "adamw_batch", "adamw_step", "bind"):
        with pytest.raises(RuntimeError, match="arguments"):
            getattr(native, name)(1)
    p = torch.nn.Parameter(x)
    with pytest.raises(RuntimeError, match="do not match"):
        native.adamw_batch([p], [], ["exp_avg", "exp_avg_sq"], 32)
    with pytest.raises(RuntimeError, match="do not match"):
        native.adamw_batch([p], [{}], ["exp_avg"], 8)
    assert native.adamw_batch([p], [{"exp_avg": x.clone(), "exp_avg_sq": x.clone()}], ["exp_avg", "exp_avg_sq"], 32) is None    # on the CPU
    with pytest.raises((RuntimeError, ValueError)):
        native.adamw_step(None, [p], {p: {}}, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, 32)


def _plain_calls():
    """The native calls that take operands as they are: (name, operands that fit one another but for their place)."""
    x, w, b, t = torch.randn(4, 8), torch.randn(3, 8), torch.randn(3), torch.zeros(4, dtype=torch.int64)
    stats, one, share = torch.zeros(13), torch.ones(()), torch.zeros(9)
    kept = torch.zeros(_lib.load().vtdge_cross_entropy_laid_out(4, 3, 8, 0), dtype=torch.uint8)
    return {"cross_entropy": [x, w, b, t, -100, 0.1, 1],
            "cross_entropy_backward": [x, w, b, t, stats, kept, one, -100, 0.1, 1, 1, 1, 1],
            "gate_balance": [x, torch.zeros((4, 2), dtype=torch.int64), torch.ones(4, dtype=torch.bool), 2],
            "gate_balance_backward": [x, torch.ones(4, dtype=torch.bool), share, one]}


@pytest.mark.parametrize("name", ["cross_entropy", "cross_entropy_backward", "gate_balance", "gate_balance_backward"])
def test_operands_of_the_plain_calls(name):
    """Each operand that does not fit is named before anything is launched; the place is looked at last, so that the rest shows here."""
    call = getattr(_lib.training(), name)
    args = _plain_calls()[name]
    with pytest.raises(RuntimeError, match=f"^{name}: .* GPU"):
        call(*args)
    half, longs, flat = torch.randn(4, 8).half(), torch.zeros((4, 8), dtype=torch.int64), torch.randn(32)
    strided, empty = torch.randn(4, 16)[:, ::2], torch.randn(0, 8)
    rows = [half, longs, flat, strided, empty, "x", None]
    bad = {"cross_entropy": {0: rows, 1: rows + [torch.randn(3, 9), torch.randn(3, 8).bfloat16()], 2: [torch.randn(2), torch.randn(3).bfloat16(), torch.randn(6)[::2]],
                             3: [torch.zeros(3, dtype=torch.int64), torch.zeros(4, dtype=torch.int32), torch.zeros((4, 1), dtype=torch.int64), None],
                             5: [-0.1, 1.5, float("nan")], 6: [3, -1]},
           "gate_balance": {0: rows + [torch.randn(4, 513)], 1: [torch.zeros((4, 3), dtype=torch.int64), torch.zeros((3, 2), dtype=torch.int64), torch.zeros((4, 2), dtype=torch.int32)],
                            2: [torch.ones(3, dtype=torch.bool), torch.ones(4), torch.ones(4, 1, dtype=torch.bool)], 3: [0, 3, 513]},
           "gate_balance_backward": {0: rows, 1: [torch.ones(3, dtype=torch.bool), torch.ones(4)], 2: [torch.zeros(8), torch.zeros(9).double(), torch.zeros(18)[::2], None],
                                     3: [torch.ones(2), torch.ones((), dtype=torch.float64), None]}}
    bad["cross_entropy_backward"] = {**{i: bad["cross_entropy"][i] for i in range(4)}, 4: [torch.zeros(12), torch.zeros(14), torch.zeros(13).double(), torch.zeros(26)[::2], None],
                                     5: [args[5][1:] if name == "cross_entropy_backward" else None, torch.zeros(1 << 16)], 6: [torch.ones(4), torch.ones(3), torch.ones((), dtype=torch.bfloat16), None],
                                     8: [-0.1, 1.5], 9: [3, -1]}
    for at, values in bad[name].items():
        for v in values:
            with pytest.raises((RuntimeError, TypeError, ValueError), match=f"^{name}: (?!.*GPU)"):
                call(*args[:at], v, *args[at + 1:])
    if name == "gate_balance":
        with pytest.raises((RuntimeError, ValueError), match="^gate_balance: .*top_k"):
            call(args[0], None, None, 9)
    if name == "cross_entropy_backward":                   # a value for each row goes with a loss for each
        with pytest.raises(RuntimeError, match=f"^{name}: .* GPU"):
            call(*args[:6], torch.ones(4), *args[7:9], 0, *args[10:])
        with pytest.raises(RuntimeError, match=f"^{name}: (?!.*GPU)"):
            call(*args[:6], torch.ones(3), *args[7:9], 0, *args[10:])


@pytest.mark.parametrize("change", ["half", "transposed", "type", "moment", "scale"])
def test_a_table_of_weights_holds_for_their_memory_alone(change):
    """The same address under another size, order or type is another weight."""
    from vtpack_amd.optim import _Batch
    p = torch.nn.Parameter(torch.randn(32, 32))
    state = {k: torch.zeros(32, 32) for k in ("exp_avg", "exp_avg_sq")}
    state.update({k + "_scale": torch.zeros(4) for k in ("exp_avg", "exp_avg_sq")})
    batch = _Batch([p], [state], 8, 0)
    assert batch.holds()
    if change == "half":
        p.data = p.data[:16]
    elif change == "transposed":
        p.data = p.data.t()
    elif change == "type":
        state["exp_avg"].data = state["exp_avg"].data.view(torch.int32)
    elif change == "moment":
        state["exp_avg"].data = state["exp_avg"].data.view(-1)
    else:
        state["exp_avg_sq_scale"].data = state["exp_avg_sq_scale"].data[:3]
    assert not batch.holds()


def test_gradients_of_a_table():
    """One of another type, size or device, or a sparse one, is refused also where its bytes are as many."""
    from vtpack_amd.optim import _Batch
    p, q = (torch.nn.Parameter(torch.randn(32).bfloat16()) for _ in range(2))
    states = [{k: torch.zeros(32) for k in ("exp_avg", "exp_avg_sq")} for _ in range(2)]
    batch = _Batch([p, q], states, 32, 0)
    good = torch.zeros(32, dtype=torch.bfloat16)
    assert all(a is b for a, b in zip(batch.take_gradients([good, good]), [good, good]))
    for bad in (good.half(), torch.zeros(32, dtype=torch.bfloat16, device="meta"), good.view(4, 8), good[:31], good.to_sparse()):
        with pytest.raises(ValueError):
            batch.take_gradients([good, bad])


def test_tracing_is_refused():
    """What a trace would record of a native call is the allocation of its results."""
    from torch.fx.experimental.proxy_tensor import make_fx
    x, w, t = torch.randn(4, 8), torch.randn(3, 8), torch.zeros(4, dtype=torch.int64)
    for call in (lambda x: linear_cross_entropy(x, w, None, t), lambda x: gate_balance(x)[0]):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(call, (x,))
        for mode in ("real", "fake"):
            with pytest.raises(RuntimeError, match="cannot be traced"):
                make_fx(call, tracing_mode=mode, _allow_non_fake_inputs=True)(x)
        with pytest.raises(RuntimeError, match="GPU only"):           # and nothing stays behind of it
            call(x)


@pytest.mark.parametrize("family", ["deit", "pvt"])
def test_a_head_that_is_more_than_its_weight_has_no_fused_loss(family):
    from vtpack_amd.models.dge.deit_dge import VisionTransformer
    from vtpack_amd.models.dge.pvt_dge import PyramidVisionTransformer
    if family == "deit":
        m = VisionTransformer(img_size=64, patch_size=8, embed_dim=64, depth=1, num_heads=1, mlp_ratio=2, num_classes=7, split_sizes=[4, 2, 1])
    else:
        m = PyramidVisionTransformer(img_size=128, patch_size=4, num_classes=7, embed_dims=[64] * 4, num_heads=[1] * 4, mlp_ratios=[2] * 4,
                                     depths=[1] * 4, sr_ratios=[8, 4, 2, 1], split_sizes=[[4, 2, 1]] * 4, qkv_bias=True)
    side = 64 if family == "deit" else 128
    images, target = torch.randn(1, 3, side, side), torch.zeros(1, dtype=torch.int64)
    plain = m.head
    for hook in (plain.register_forward_hook(lambda *a: None), plain.register_forward_pre_hook(lambda *a: None),
                 plain.register_full_backward_hook(lambda *a: None), plain.register_full_backward_pre_hook(lambda *a: None)):
        with pytest.raises(TypeError, match="model's head"):
            m.loss(images, target)
        hook.remove()

    class Scaled(torch.nn.Linear):
        def forward(self, x):
            return 2 * super().forward(x)

    for head in (Scaled(64, 7), torch.nn.Sequential(plain), torch.nn.utils.spectral_norm(torch.nn.Linear(64, 7))):
        m.head = head
        with pytest.raises(TypeError, match="model's head"):
            m(images, target)
    m.head = plain
    plain.forward = lambda x: x                           # as wrappers of modules put theirs in place
    with pytest.raises(TypeError, match="model's head"):
        m(images, target)
    del plain.forward
    with pytest.raises(Exception) as caught:              # on to the kernels, which want a GPU
        m.loss(images, target)
    assert "model's head" not in str(caught.value)


def test_how_a_loss_is_made_goes_with_a_target():
    from vtpack_amd.models.dge.deit_dge import VisionTransformer
    m = VisionTransformer(img_size=64, patch_size=8, embed_dim=64, depth=1, num_heads=1, mlp_ratio=2, num_classes=7, split_sizes=[4, 2, 1])
    with pytest.raises(TypeError, match="label_smoothing without a target"):
        m(torch.randn(1, 3, 64, 64), label_smoothing=0.1)


def test_gradients_with_operands_laid_out_before_need_no_room_for_them():
    size = _lib.load().vtdge_cross_entropy_workspace
    x, w = 2048 * 384 * 6, 21841 * 384 * 6
    assert size(2048, 21841, 384, 0, 1) - size(2048, 21841, 384, 0, 1 + 8) == -(-x // 256) * 256 + -(-w // 256) * 256
    # bf16 that is read where it lies has its x with zeros for the rows that are left out all the same
    assert size(256, 1000, 384, 1, 1 + 2 + 4) == size(256, 1000, 384, 1, 1 + 2 + 4 + 8)


def test_lists_of_a_batch():
    native, p = _lib.training(), torch.nn.Parameter(torch.zeros(3))
    for args in (((p,), [{}], ["exp_avg", "exp_avg_sq"]), ([p], ({},), ["exp_avg", "exp_avg_sq"]), ([p], [{}], ("exp_avg", "exp_avg_sq")), (None, [{}], [])):
        with pytest.raises(RuntimeError, match="lists"):
            native.adamw_batch(*args, 32)
    for name, args in (("places", ((p,),)), ("places", ([None],)), ("alike", ([p], [])), ("alike", (p, [p]))):
        with pytest.raises(RuntimeError, match=name):
            getattr(native, name)(*args)
