"""What the block-scaled operators (utils/block_scaled.py) refuse, and the arguments their C entries refuse, without a GPU."""
import pytest
import torch

from medicaldetectiontoolkit_amd import _lib
from medicaldetectiontoolkit_amd.utils import block_scaled as bs


def ck(shape, **kw):
    n = torch.Size(shape).numel()
    return bs.Checkpoint8(torch.zeros(n, dtype=torch.uint8), torch.zeros(-(-n // 32), dtype=torch.uint8), shape, **kw)


def test_no_cpu_path():
    x = torch.zeros(4, 32)
    with pytest.raises(RuntimeError, match="GPU"):
        bs.checkpoint8(x)
    with pytest.raises(RuntimeError, match="GPU"):
        ck((4, 32)).restore()
    with pytest.raises(RuntimeError, match="GPU"):
        bs.bias_act_checkpoint8(x, torch.zeros(32))
    with pytest.raises(RuntimeError, match="GPU"):
        bs.conv1x1_backward8(x, torch.zeros(32, 8), ck((4, 8)))
    with pytest.raises(RuntimeError, match="GPU"):
        bs.mx4_quantize(x)
    w4 = bs.Mx4(torch.zeros(3, 16, dtype=torch.uint8), torch.zeros(3, 1, dtype=torch.uint8), 32)
    with pytest.raises(RuntimeError, match="GPU"):
        w4.dequantize()
    with pytest.raises(RuntimeError, match="GPU"):
        bs.mx4_linear(x, w4)


def test_other_types_are_refused():
    for t in (torch.float64, torch.int32, torch.uint8):
        with pytest.raises(TypeError):
            bs.checkpoint8(torch.zeros(4, dtype=t))
        with pytest.raises(TypeError):
            bs.mx4_quantize(torch.zeros(4, dtype=t))
        with pytest.raises(TypeError):
            ck((4,), dtype=t)


def test_checkpoint8_container():
    with pytest.raises(ValueError, match="33 uint8 codes and 2 uint8 scales"):
        bs.Checkpoint8(torch.zeros(33, dtype=torch.uint8), torch.zeros(1, dtype=torch.uint8), (33,))
    with pytest.raises(ValueError):
        bs.Checkpoint8(torch.zeros(32), torch.zeros(1, dtype=torch.uint8), (32,))
    with pytest.raises(ValueError, match="contiguous"):
        bs.Checkpoint8(torch.zeros(64, dtype=torch.uint8)[::2], torch.zeros(1, dtype=torch.uint8), (32,))
    with pytest.raises(ValueError, match="aligned"):
        bs.Checkpoint8(torch.zeros(33, dtype=torch.uint8)[1:], torch.zeros(1, dtype=torch.uint8), (32,))
    with pytest.raises(ValueError, match="channels_last"):
        ck((2, 3, 4), channels_last=True)
    with pytest.raises(ValueError, match="channels_last"):
        ck((2, 3), channels_last=False)


def test_mx4_container():
    with pytest.raises(ValueError, match="rows of 33"):
        bs.Mx4(torch.zeros(2, 16, dtype=torch.uint8), torch.zeros(2, 1, dtype=torch.uint8), 33)
    with pytest.raises(ValueError):
        bs.Mx4(torch.zeros(2, 16, dtype=torch.uint8), torch.zeros(3, 1, dtype=torch.uint8), 32)
    with pytest.raises(ValueError):
        bs.Mx4(torch.zeros(2, 0, dtype=torch.uint8), torch.zeros(2, 0, dtype=torch.uint8), 0)
    with pytest.raises(ValueError, match="contiguous"):
        bs.Mx4(torch.zeros(16, 2, dtype=torch.uint8).t(), torch.zeros(2, 1, dtype=torch.uint8), 32)


def test_division_by_multiplication():
    """the kernels' n / d for n < 2^31, in integers"""
    import random
    rng = random.Random(0)
    for d in [1, 2, 3, 5, 7, 18, 36, 72, 255, 256, 257, 5292, 65537, 2 ** 30 - 1, 2 ** 30, 2 ** 30 + 1] + [rng.randrange(1, 2 ** 31) for _ in range(200)]:
        s = 0
        while s < 32 and (1 << s) < d:
            s += 1
        mul = ((((1 << s) - d) << 32) // d + 1) & 0xffffffff
        for n in [0, 1, d - 1, d, d + 1, 2 * d - 1, 2 * d, 2 ** 31 - 1] + [rng.randrange(2 ** 31) for _ in range(200)]:
            if 0 <= n < 2 ** 31:
                assert (((mul * n) >> 32) + n) >> s == n // d, (n, d)


def test_c_entries_refuse_bad_arguments():
    L = _lib.lib()
    bad, small = -1, -2
    assert L.mdt_act8_quantize(None, None, None, 5, 0, 0, None) == bad
    assert L.mdt_act8_quantize(16, 16, 16, -1, 0, 0, None) == bad
    assert L.mdt_act8_quantize(16, 16, 16, 5, 3, 0, None) == bad
    assert L.mdt_act8_quantize(16, 17, 16, 5, 0, 0, None) == bad
    assert L.mdt_act8_quantize(16, 16, 16, 2 ** 33 + 1, 0, 0, None) == bad
    assert L.mdt_act8_restore(16, 16, None, 5, 0, 0, None) == bad
    assert L.mdt_bias_act_act8_forward(16, 16, None, None, 16, 16, 32, 4, 1, 1, None) == bad
    assert L.mdt_bias_act_act8_forward(16, 16, 16, None, 16, 16, 32, 0, 1, 1, None) == bad
    assert L.mdt_mx4_quantize(16, 16, 16, 4, 0, 0, None) == bad
    assert L.mdt_mx4_quantize(16, 16, 16, 2 ** 40, 2 ** 40, 0, None) == bad
    assert L.mdt_mx4_dequantize(16, 16, 16, 4, 8, 9, None) == bad
    ws = L.mdt_conv1x1_act8_backward_workspace_bytes(100, 18, 72)
    assert L.mdt_conv1x1_act8_backward(16, 16, 16, 16, 1, 16, 16, 16, 16, 16, 100, 18, 72, 16, ws - 1, None) == small
    assert L.mdt_conv1x1_act8_backward(16, 16, 16, 16, 1, 16, 16, 16, 16, 16, 100, 18, 72, None, ws, None) == small
    assert L.mdt_conv1x1_act8_backward(None, 16, 16, 16, 1, 16, 16, 16, 16, 16, 100, 18, 72, 16, ws, None) == bad
    assert L.mdt_conv1x1_act8_backward(16, 16, None, 16, 1, 16, 16, 16, 16, 16, 100, 18, 72, 16, ws, None) == bad
    assert L.mdt_conv1x1_act8_backward(16, 16, 16, 16, 1, 16, 16, 16, 16, 16, 100, 0, 72, 16, ws, None) == bad
    ws = L.mdt_mx4_linear_workspace_bytes(4000, 5292, 144)
    assert ws > 0 and L.mdt_mx4_linear_workspace_bytes(1, 5292, 144) == 0
    assert L.mdt_mx4_linear(16, 0, 16, 16, 16, 16, 4000, 5292, 144, 1, 16, ws - 1, None) == small
    assert L.mdt_mx4_linear(16, 0, 16, 16, 16, 16, 4000, 5292, 144, 1, None, ws, None) == small
    assert L.mdt_mx4_linear(None, 0, 16, 16, 16, 16, 100, 5292, 144, 1, None, 0, None) == bad
    assert L.mdt_mx4_linear(16, 0, 24, 16, 16, 16, 100, 5292, 144, 1, None, 0, None) == bad
    assert L.mdt_mx4_linear(16, 5, 16, 16, 16, 16, 100, 5292, 144, 1, None, 0, None) == bad
    # nothing to do is no error and launches nothing
    assert L.mdt_act8_quantize(None, None, None, 0, 0, 0, None) == 0
    assert L.mdt_act8_restore(None, None, None, 0, 0, 0, None) == 0
    assert L.mdt_bias_act_act8_forward(None, None, None, None, None, None, 0, 4, 1, 1, None) == 0
    assert L.mdt_mx4_quantize(None, None, None, 0, 8, 0, None) == 0
    assert L.mdt_mx4_linear(None, 0, None, None, None, None, 0, 8, 4, 0, None, 0, None) == 0


def test_shapes_that_do_not_belong_together():
    """checked before anything is launched; the operands' device is looked at first, so these run on meta-free CPU tensors with the check stubbed"""
    real = _lib.require_cuda
    _lib.require_cuda = lambda t, name: None
    try:
        gy, w = torch.zeros(4, 32), torch.zeros(32, 8)
        for a in ((gy, torch.zeros(32, 8, 3), ck((4, 8))), (gy, torch.zeros(31, 8), ck((4, 8))), (gy, w, ck((5, 8))), (gy, w, ck((4, 9))), (torch.zeros(4, 32, 3), w, ck((4, 8, 3))),
                  (gy, w, ck((4, 8)), ck((4, 31), relu=True)), (gy, w, ck((4, 8)), ck((4, 32))), (torch.zeros(2, 32, 3, 3), w, ck((2, 8, 3, 3)))):
            with pytest.raises(ValueError):
                bs.conv1x1_backward8(*a)
        with pytest.raises(TypeError):
            bs.conv1x1_backward8(gy.double(), w, ck((4, 8)))
        for a in ((gy, torch.zeros(31)), (gy, torch.zeros(32), torch.zeros(4, 31)), (torch.zeros(32), torch.zeros(32))):
            with pytest.raises(ValueError):
                bs.bias_act_checkpoint8(*a)
        with pytest.raises(TypeError):
            bs.bias_act_checkpoint8(gy.half(), torch.zeros(32))
        with pytest.raises(RuntimeError, match="no_grad"):
            bs.bias_act_checkpoint8(gy, torch.zeros(32, requires_grad=True))
        w4 = bs.Mx4(torch.zeros(3, 16, dtype=torch.uint8), torch.zeros(3, 1, dtype=torch.uint8), 32)
        for a in ((torch.zeros(4, 31), w4), (gy, w4, torch.zeros(4)), (torch.zeros(()), w4)):
            with pytest.raises(ValueError):
                bs.mx4_linear(*a)
        with pytest.raises(RuntimeError, match="no_grad"):
            bs.mx4_linear(gy.clone().requires_grad_(), w4)
        with pytest.raises(ValueError):
            bs.mx4_quantize(torch.zeros(()))
        with pytest.raises(ValueError):
            bs.mx4_quantize(torch.zeros(3, 0))
    finally:
        _lib.require_cuda = real


def test_where_the_framework_uses_them():
    """the options' names and refusals"""
    from medicaldetectiontoolkit_amd import predictor
    from medicaldetectiontoolkit_amd.configs import Configs
    from medicaldetectiontoolkit_amd.models import backbone
    from medicaldetectiontoolkit_amd.utils.model_utils import NDConvGenerator
    cf = Configs(dim=2, model="mrcnn", patch_size=[64, 64], batch_size=1)
    assert cf.act8_checkpoints is False
    for kw in (dict(norm="batch_norm"), dict(relu="leaky_relu")):
        cf = Configs(dim=2, model="mrcnn", patch_size=[64, 64], batch_size=1, act8_checkpoints=True, **kw)
        with pytest.raises(ValueError, match="act8_checkpoints"):
            backbone.FPN(cf, NDConvGenerator(2))
    with pytest.raises(ValueError, match="head_dtype"):
        predictor.predict_patient(None, None, None, head_dtype="int8")
    with pytest.raises(ValueError, match="box head"):
        predictor.predict_patient(torch.nn.Linear(2, 2), None, None, head_dtype="mx4")
    net = torch.nn.Module()
    net.classifier = torch.nn.Module()
    with pytest.raises(ValueError, match="box head"):
        bs.mx4_heads(net).__enter__()
    net.classifier.mx4 = None
    net.classifier.conv1 = net.classifier.conv2 = torch.nn.Sequential(torch.nn.Conv2d(2, 2, 1), torch.nn.BatchNorm2d(2))
    with pytest.raises(ValueError, match="without a norm"):
        bs.mx4_heads(net).__enter__()
    with pytest.raises(RuntimeError, match="GPU"):
        bs.conv_bias_act8(torch.nn.Conv2d(8, 8, 1), torch.zeros(1, 8, 4, 4))
    with pytest.raises(RuntimeError, match="GPU"):
        bs.act_backward8(torch.zeros(4, 8), ck((4, 8), relu=True))
    with pytest.raises(TypeError):
        bs.act_backward8(torch.zeros(4, 8, dtype=torch.float64), ck((4, 8), relu=True))


def test_scratch_sizes_of_every_size():
    need = _lib.lib().mdt_conv1x1_act8_backward_workspace_bytes
    for V in (1, 2, 3, 4, 5, 7, 31, 257, 4096, 1 << 20, 1 << 30):
        for ci in (1, 2, 3, 18, 257, 2048, 65536):
            for co in (1, 2, 3, 18, 255, 257, 514, 1028, 2048, 65536):
                n = need(V, ci, co)
                assert 4 * co <= n <= 4 * 2048 * (ci * co + co) + 4 * 32 * V * ci + 4096, (V, ci, co, n)
