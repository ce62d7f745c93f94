"""Blocks of 8-bit numbers without a GPU: what the operators refuse, the checks of the library's arguments, the oracle's own rounding."""
import pytest
import torch

from tests import eight_bit_reference as ref
from vtpack_amd import _lib
from vtpack_amd.layers import Blocks, gelu_8bit, layer_norm_8bit, linear_8bit, quantize_blocks


def test_tensors_on_the_cpu_are_refused():
    x, w = torch.randn(4, 8), torch.randn(3, 8)
    for call in (lambda: quantize_blocks(x), lambda: linear_8bit(x, w), lambda: gelu_8bit(x), lambda: layer_norm_8bit(x, w[0], w[0]),
                 lambda: Blocks(x.to(torch.float8_e4m3fn), torch.ones(4, 1).to(torch.float8_e8m0fnu))):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()


def test_what_is_no_tensor_is_refused():
    for call in (lambda: quantize_blocks([1.0]), lambda: gelu_8bit(None), lambda: linear_8bit(None, torch.zeros(2, 2)), lambda: layer_norm_8bit(1, 2, 3)):
        with pytest.raises(TypeError):
            call()
    with pytest.raises(ValueError, match="act"):
        linear_8bit(torch.zeros(2, 2), torch.zeros(2, 2), act="relu")


def test_the_oracle_rounds_as_e4m3_does():
    """Against torch's own conversion of what the scale leaves."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(50, 300, generator=g) * torch.exp(3 * torch.randn(50, 300, generator=g))
    numbers, e = ref.blocks_of(x)
    for k in range(3):
        t, s = x[:, 128 * k:128 * k + 128], e[:, k:k + 1]
        scaled = (t.double() * torch.exp2(-s)).float()
        assert float(scaled.abs().max()) <= 448 and (scaled.abs().amax(1) > 224).all()
        assert torch.equal(numbers[:, 128 * k:128 * k + 128], scaled.to(torch.float8_e4m3fn).double() * torch.exp2(s))
    assert torch.equal(numbers, numbers.to(torch.bfloat16).double())


def test_sizes_of_buffers():
    lib = _lib.load()
    assert lib.vtdge_blocks_bytes(1, 1) == 128 + 4 and lib.vtdge_blocks_bytes(3, 128) == 3 * 132 and lib.vtdge_blocks_bytes(2, 129) == 2 * 260
    assert lib.vtdge_blocks_bytes(2, 513) == 2 * (640 + 8) and lib.vtdge_blocks_bytes(0, 5) == -1 and lib.vtdge_blocks_bytes(5, 0) == -1
    assert lib.vtdge_blocks_bytes(1 << 31, 1) == -1 and lib.vtdge_blocks_bytes(1, (1 << 20) + 1) == -1 and lib.vtdge_blocks_bytes((1 << 31) - 1, 1 << 20) == -1


def test_more_than_a_launch_takes_is_refused():
    """2^32 threads, sixteen a block, and a workgroup for one to four rows of a norm."""
    lib, p, U = _lib.load(), 4096, _lib.ERR_UNSUPPORTED
    most = 268435440
    assert lib.vtdge_blocks_bytes(most, 1) == most * 132 and lib.vtdge_blocks_bytes(most + 1, 128) == -1 and lib.vtdge_blocks_bytes(most // 2 + 1, 129) == -1
    for rows, n in ((most + 1, 1), (most // 2 + 1, 129)):
        assert lib.vtdge_quantize_blocks(p, n, rows, n, p, 0, None) == U and lib.vtdge_dequantize_blocks(p, rows, n, p, 0, None) == U
        assert lib.vtdge_gelu_8bit(p, n, rows, n, p, p, 0, None) == U and lib.vtdge_gelu_8bit_backward(p, n, rows, n, p, p, 0, None) == U
    assert lib.vtdge_layernorm_8bit(p, 8, p, p, 1e-6, 1 << 24, 8, p, p, p, 0, None) == U
    assert lib.vtdge_layernorm_8bit_backward_workspace(1 << 24, 8) == -1 and lib.vtdge_layernorm_8bit_backward_workspace((1 << 24) - 1, 8) > 0


def _codes(fn, good, table):
    for i, v, want in table:
        args = list(good)
        args[i] = v
        assert fn(*args) == want, (i, v, _lib.load().vtdge_last_error())


def test_arguments_of_the_library():
    """Before anything is launched."""
    lib, p = _lib.load(), 4096                            # never read: the arguments are refused first
    A, U = _lib.ERR_ARG, _lib.ERR_UNSUPPORTED
    blocks = ((0, None, A), (1, 7, A), (2, 0, A), (3, 0, A), (3, -1, A), (4, None, A), (4, p + 16, A), (5, 2, A), (2, 1 << 31, U))
    _codes(lib.vtdge_quantize_blocks, [p, 8, 4, 8, p, 0, None], blocks)
    _codes(lib.vtdge_dequantize_blocks, [p, 4, 8, p, 0, None], ((0, None, A), (0, p + 4, A), (1, 0, A), (2, 0, A), (3, None, A), (4, 9, A), (2, 1 << 21, U)))
    gelu = [p, 8, 4, 8, p, p, 0, None]
    _codes(lib.vtdge_gelu_8bit, gelu, ((0, None, A), (1, 7, A), (2, 0, A), (3, 0, A), (4, None, A), (5, p + 1, A), (6, 5, A)))
    _codes(lib.vtdge_gelu_8bit_backward, [p, 8, 4, 8, p, p, 0, None], ((0, None, A), (1, 7, A), (4, None, A), (5, None, A), (4, p + 1, A), (6, 5, A)))
    _codes(lib.vtdge_layernorm_8bit, [p, 8, p, p, 1e-6, 4, 8, p, p, p, 0, None],
           ((0, None, A), (1, 7, A), (2, None, A), (3, None, A), (5, 0, A), (6, 8193, U), (7, None, A), (8, None, A), (9, None, A), (8, p + 1, A), (10, 3, A)))
    _codes(lib.vtdge_layernorm_8bit_backward, [p, 8, p, p, p, 4, 8, p, 1 << 30, p, p, p, 0, None],
           ((0, None, A), (1, 7, A), (2, None, A), (3, None, A), (4, None, A), (5, 0, A), (6, 8193, U), (7, None, A), (8, 0, A), (7, p + 4, A), (12, 3, A)))
    linear = [p, 8, p, 8, None, p, p, None, 40, 3, 8, 0, p, 1 << 40, 0, None]
    _codes(lib.vtdge_linear_8bit, linear,
           ((0, None, A), (1, 7, A), (3, 7, A), (4, p + 4, A), (6, None, A), (7, p + 4, A), (8, 0, A), (9, 0, A), (10, 0, A), (11, 2, A), (12, None, A),
            (12, p + 16, A), (13, -1, A), (13, 0, A), (14, 2, A), (8, 1 << 31, U), (10, 1 << 21, U)))
    # what lies in the workspace: operands that are neither given nor kept in blocks, none with few rows but a weight
    size = lib.vtdge_linear_8bit_workspace
    assert size(40, 3, 8, 1 | 4, 1) == 0 and size(40, 3, 8, 2 | 4, 1) == 0 and size(40, 3, 8, 0, 1) > 0 and size(40, 3, 8, 1 | 4, 0) > 0
    assert size(16, 3, 8, 1, 0) == 0 and size(16, 3, 8, 0, 0) == 512 and size(17, 3, 8, 1, 0) > 0
    args = list(linear)
    args[2] = args[4] = None
    assert lib.vtdge_linear_8bit(*args) == A and b"NULL" in lib.vtdge_last_error()
    back = [p, 3, p, p, 4, 3, 8, p, 1 << 40, p, p, p, 0, None]
    _codes(lib.vtdge_linear_8bit_backward, back,
           ((0, None, A), (1, 2, A), (2, None, A), (3, None, A), (2, p + 4, A), (3, p + 4, A), (4, 0, A), (5, 0, A), (6, 0, A), (7, None, A), (7, p + 16, A),
            (8, 0, A), (12, 4, A)))
    args = list(back)
    args[0] = args[9] = args[10] = args[11] = None        # nothing asked for
    assert lib.vtdge_linear_8bit_backward(*args) == 0
    assert lib.vtdge_linear_8bit_workspace(0, 3, 8, 0, 0) == -1 and lib.vtdge_linear_8bit_backward_workspace(4, 3, 8, 0, 7) == -1


def test_a_model_in_eight_bits():
    """The setting reaches every block and takes plain modules alone."""
    from vtpack_amd.models.dge.deit_dge import Attention, Block, Mlp, VisionTransformer
    m = VisionTransformer(img_size=32, patch_size=8, embed_dim=32, depth=2, num_heads=1, num_classes=3, split_sizes=[2, 1])
    keys = list(m.state_dict())
    parts = [k for k in m.modules() if isinstance(k, (Block, Attention, Mlp))]
    assert m.set_eight_bit() is m and len(parts) == 6 and all(k.eight_bit for k in parts) and list(m.state_dict()) == keys
    with pytest.raises(RuntimeError, match="GPU only"):
        m.train().blocks[0].mlp(torch.zeros(2, 32))
    m.eval()
    assert m.blocks[0].mlp(torch.zeros(2, 32)).shape == (2, 32)         # eval mode as it was
    assert not any(k.eight_bit for k in (m.set_eight_bit(False), *parts) if k is not m)
    m.blocks[1].mlp.fc1.register_forward_hook(lambda *a: None)
    with pytest.raises(TypeError, match="plain"):
        m.set_eight_bit()
    assert not any(k.eight_bit for k in parts)
    m = VisionTransformer(img_size=32, patch_size=8, embed_dim=32, depth=1, num_heads=1, num_classes=3, split_sizes=[2, 1])
    m.blocks[0].mlp.act = torch.nn.GELU(approximate="tanh")
    with pytest.raises(TypeError, match="plain"):
        m.set_eight_bit()
    from vtpack_amd.layers.eight_bit import require_plain_module
    for bad in (torch.nn.LayerNorm(8, elementwise_affine=False), torch.nn.LayerNorm([2, 4]), torch.nn.Identity(), torch.nn.LayerNorm(8, bias=False)):
        with pytest.raises(TypeError):
            require_plain_module(bad)


def test_a_pyramid_in_eight_bits():
    from vtpack_amd.models.dge.pvt_dge import Attention, Block, PyramidVisionTransformer
    m = PyramidVisionTransformer(img_size=128, patch_size=4, num_classes=9, embed_dims=[64, 64, 64, 64], num_heads=[1, 1, 1, 1], mlp_ratios=[2] * 4,
                                 depths=[1, 1, 1, 1], sr_ratios=[8, 4, 2, 1], split_sizes=[[4, 2, 1]] * 4, qkv_bias=True)
    assert all(k.eight_bit for k in m.set_eight_bit().modules() if isinstance(k, (Block, Attention)))
    m.block1[0].attn.norm = torch.nn.Identity()
    with pytest.raises(TypeError, match="plain"):
        m.set_eight_bit()
