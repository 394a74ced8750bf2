"""The block-scaled operators where the framework uses them: a convolution layer of the autograd graph with 8-bit copies (conv_bias_act8, act_backward8), the
backbone and the training step with cf.act8_checkpoints, and the box head in 4 bits (mx4_heads, head_dtype="mx4").

Layers are compared on small integers with the formulas in 64 bits (all products and sums are exact in fp32: equality), nets with the fp32 path: what does not
depend on a kept input is the same up to the order of fp32 sums, the filters' gradients within what half a step of a block allows."""
import numpy as np
import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from medicaldetectiontoolkit_amd.configs import Configs
from medicaldetectiontoolkit_amd.models import mrcnn, retina_unet
from medicaldetectiontoolkit_amd.utils import block_scaled as bs
from medicaldetectiontoolkit_amd.utils import fused_epilogue as fe
from medicaldetectiontoolkit_amd.utils.synthetic_data import make_batch
from tests.test_block_scaled_gpu import kept4, kept8

pytestmark = pytest.mark.gpu


def mf_of(t):
    return torch.channels_last_3d if t.dim() == 5 else torch.channels_last


# ---- mask and column sums ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("shape", [(1, 1), (2, 1), (1, 5), (7, 1), (33, 3), (1000, 18), (77, 30), (4099, 36), (129, 255), (130, 256), (131, 257), (50, 511), (40, 510), (40, 514),
                                   (300, 1024), (60, 1028), (3, 2052), (70000, 18), (20000, 257), (2, 18, 5, 6, 7), (3, 36, 9, 5), (0, 18)])
def test_act_backward8(cuda, shape):
    gen = torch.Generator().manual_seed(sum(shape))
    y = torch.randn(shape, generator=gen).relu()
    gy = torch.randint(-8, 9, shape, generator=gen).float()
    mf = mf_of(y) if len(shape) > 2 else torch.contiguous_format
    y8 = bs.checkpoint8(y.to(cuda).contiguous(memory_format=mf), relu=True)
    gy_d = gy.to(cuda)
    gy_d[y8.restore() == 0] = float("nan")                     # masked gradients do not show
    g, gb = bs.act_backward8(gy_d, y8)
    want = (gy * (y > 0)).double()
    assert g.is_contiguous(memory_format=mf) and torch.equal(g.cpu().double(), want)
    assert torch.equal(gb.cpu().double(), want.transpose(0, 1).reshape(shape[1], -1).sum(1))          # |sum| < 2^24: exact in any order
    plain, sums = bs.act_backward8(gy.to(cuda))
    assert torch.equal(plain.cpu(), gy) and torch.equal(sums.cpu().double(), gy.double().transpose(0, 1).reshape(shape[1], -1).sum(1))
    # without a mask, and the sums alone, through the products' entry
    if len(shape) == 2 and shape[0] > 0:
        V, C = shape
        w, x8 = torch.zeros(C, 2, device=cuda), bs.checkpoint8(torch.zeros(V, 2, device=cuda))
        out = bs.conv1x1_backward8(gy.to(cuda), w, x8, None, need_gx=False, need_gw=False)
        assert out[0] is None and out[1] is None and out[3] is None and torch.equal(out[2].cpu().double(), gy.double().sum(0))
        out = bs.conv1x1_backward8(gy_d, w, x8, y8, need_gx=False, need_gw=True, need_g=True)
        assert torch.equal(out[3], g) and torch.equal(out[2], gb) and not out[1].any()


def test_layers_on_two_streams_do_not_share_scratch(cuda):
    """forward and backward of two layers at once, each on its own stream, equal to one after the other"""
    jobs = []
    for seed in (1, 2):
        one, x0, gy, _ = int_layer(cuda, 3, 18, 72, 1, (32, 32, 32), 1, seed)
        three, _, gy3, _ = int_layer(cuda, 3, 18, 18, 3, (32, 32, 32), 1, seed + 5)
        jobs.append((one, three, x0.to(cuda).contiguous(memory_format=torch.channels_last_3d), gy.to(cuda), gy3.to(cuda)))

    def run(one, three, x0, gy, gy3):
        one.zero_grad(set_to_none=True)
        three.zero_grad(set_to_none=True)
        x = x0.clone().requires_grad_()
        y, _ = bs.conv_bias_act8(one, x, None, relu=True)
        z, _ = bs.conv_bias_act8(three, x, None, keep=False)
        ga, = torch.autograd.grad(y, x, gy, retain_graph=True)
        gb, = torch.autograd.grad(y, one.bias, gy)
        gc, = torch.autograd.grad(z, three.bias, gy3)
        return ga, gb, gc
    want = [run(*j) for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for rep in range(5):
        got = []
        for j, s in zip(jobs, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(run(*j))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for w, g in zip(want, got) for a, b in zip(w, g))


def test_act_backward8_takes_slices_and_views(cuda):
    """gradients that are not dense, not aligned to 16 bytes, and broadcast"""
    y = torch.randn(2, 18, 4, 4, 4).relu().to(cuda).contiguous(memory_format=torch.channels_last_3d)
    y8 = bs.checkpoint8(y, relu=True)
    big = torch.randint(-8, 9, (2, 20, 4, 4, 5)).float().to(cuda)
    flat = torch.randint(-8, 9, (2 * 18 * 64 + 1,)).float().to(cuda)[1:].reshape(2, 4, 4, 4, 18).permute(0, 4, 1, 2, 3)
    for gy in (big[:, 1:19, :, :, :4], flat, torch.ones(1, 1, 1, 1, 1, device=cuda).expand(2, 18, 4, 4, 4)):
        g, gb = bs.act_backward8(gy, y8)
        assert torch.equal(g, gy * (y > 0)) and torch.equal(gb, (gy * (y > 0)).sum((0, 2, 3, 4)))


# ---- one layer -----------------------------------------------------------------------------------------------------------------------
def int_layer(cuda, nd, ci, co, k, size, B, seed):
    gen = torch.Generator().manual_seed(seed)
    conv = (nn.Conv3d if nd == 3 else nn.Conv2d)(ci, co, k, padding=k // 2)
    with torch.no_grad():
        conv.weight.copy_(torch.randint(-3, 4, conv.weight.shape, generator=gen).float())
        conv.bias.copy_(torch.randint(-8, 9, (co,), generator=gen).float() + 0.5)                  # no value of the layer is 0
    x = torch.randint(0, 16, (B, ci) + size, generator=gen).float()
    gy = torch.randint(-4, 5, (B, co) + size, generator=gen).float()
    res = torch.randint(-30, 31, (B, co) + size, generator=gen).float()
    return conv.to(cuda), x, gy, res


LAYERS = [(3, 18, 72, 1, (5, 6, 7), 2), (3, 72, 18, 1, (4, 4, 4), 1), (2, 36, 100, 1, (9, 5), 3), (3, 200, 40, 1, (3, 4, 5), 1), (3, 18, 18, 1, (64, 64, 32), 1), (2, 8, 8, 1, (1, 1), 1)]


@pytest.mark.parametrize("relu,residual,row_major", [(True, False, False), (True, True, False), (False, False, True), (False, True, False), (True, True, True)])
@pytest.mark.parametrize("nd,ci,co,k,size,B", LAYERS)
def test_conv_bias_act8_1x1_is_exact_on_integers(cuda, nd, ci, co, k, size, B, relu, residual, row_major):
    conv, x0, gy, r0 = int_layer(cuda, nd, ci, co, k, size, B, ci + co)
    mf = torch.contiguous_format if row_major else mf_of(x0)
    x = x0.to(cuda).contiguous(memory_format=mf).requires_grad_()
    r = r0.to(cuda).requires_grad_() if residual else None
    y, y8 = bs.conv_bias_act8(conv, x, None, residual=r, relu=relu)
    y.backward(gy.to(cuda))
    w, b = conv.weight.detach().cpu().double(), conv.bias.detach().cpu().double()
    h = (F.conv3d if nd == 3 else F.conv2d)(x0.double(), w, b) + (r0.double() if residual else 0)
    assert torch.equal(y.detach().cpu().double(), h.relu() if relu else h)
    assert y8.relu == relu and torch.equal(y8.restore(), bs.checkpoint8(y.detach(), relu=relu).restore())
    g = gy.double() * (h > 0) if relu else gy.double()
    rows = lambda t: t.transpose(0, 1).reshape(t.shape[1], -1)
    assert torch.equal(x.grad.cpu().double(), (F.conv_transpose3d if nd == 3 else F.conv_transpose2d)(g, w))
    assert torch.equal(conv.weight.grad.cpu().double().flatten(1), rows(g) @ rows(x0.double()).t())
    assert torch.equal(conv.bias.grad.cpu().double(), rows(g).sum(1))
    if residual:
        assert torch.equal(r.grad.cpu().double(), g)


@pytest.mark.parametrize("nd,ci,co,size,B", [(3, 18, 18, (32, 32, 64), 1), (3, 36, 36, (8, 8, 8), 2), (2, 64, 64, (12, 10), 2), (3, 5, 7, (4, 3, 2), 1)])
@pytest.mark.parametrize("relu", [True, False])
def test_conv_bias_act8_window(cuda, nd, ci, co, size, B, relu):
    """3x3(x3) layers.  Their products are this package's or the library's fp32 convolutions: a sum of n products is off by at most n 2^-24 times the sum of their magnitudes in any
    order, and by 64 times as much through a minimal-filtering transform (its growth factor for tiles of 4 is below that)"""
    conv, x0, gy, _ = int_layer(cuda, nd, ci, co, 3, size, B, ci)
    mf = mf_of(x0)
    x = x0.to(cuda).contiguous(memory_format=mf).requires_grad_()
    y, y8 = bs.conv_bias_act8(conv, x, None, relu=relu, keep=relu)
    assert (y8 is not None) == relu
    y.backward(gy.to(cuda))
    w, b = conv.weight.detach().cpu().double(), conv.bias.detach().cpu().double()
    xd = x0.double().requires_grad_()
    wd = w.clone().requires_grad_()
    fn = F.conv3d if nd == 3 else F.conv2d
    h = fn(xd, wd, b, padding=1)
    mask = y.detach().cpu() > 0 if relu else torch.ones(h.shape, dtype=torch.bool)                  # the layer's own mask
    g = gy.double() * mask
    h.backward(g)

    def close(got, want, mags, n):
        assert bool(((got.detach().cpu().double() - want).abs() <= 64 * n * 2.0 ** -24 * mags).all())
    n = ci * 3 ** nd
    close(y, (h.relu() if relu else h).detach(), fn(x0.double(), w.abs(), b.abs(), padding=1), n)
    aw, ax = w.abs().clone().requires_grad_(), x0.double().clone().requires_grad_()
    fn(ax, aw, None, padding=1).backward(g.abs())
    close(x.grad, xd.grad, ax.grad, co * 3 ** nd)
    close(conv.weight.grad, wd.grad, aw.grad, g.numel() // co)
    assert torch.equal(conv.bias.grad.cpu().double(), g.transpose(0, 1).reshape(co, -1).sum(1))


def test_conv_bias_act8_against_differences(cuda):
    """integers, and steps that flip no unit of the ReLU: the differences are exact"""
    conv, x0, gy, r0 = int_layer(cuda, 3, 18, 40, 1, (4, 5, 6), 2, 3)
    x = x0.to(cuda).contiguous(memory_format=torch.channels_last_3d)
    r, gyd = r0.to(cuda), gy.to(cuda)

    def loss(dx=0, dw=0, db=0, dr=0):
        with torch.no_grad():
            h = F.conv3d((x + dx).cpu().double(), (conv.weight + dw).cpu().double(), (conv.bias + db).cpu().double()) + (r + dr).cpu().double()
            return float((h.relu() * gy).sum())
    leaves = [x.clone().requires_grad_(), r.clone().requires_grad_()]
    y, _ = bs.conv_bias_act8(conv, leaves[0], None, residual=leaves[1], relu=True)
    y.backward(gyd)
    grads = dict(dx=leaves[0].grad, dr=leaves[1].grad, dw=conv.weight.grad, db=conv.bias.grad)
    for name, grad in grads.items():
        d = torch.sign(torch.randn(grad.shape, device=cuda)) * 2.0 ** -12                            # 18 * 15 * 2^-12 < 0.5: no unit flips
        slope = (loss(**{name: d}) - loss(**{name: -d})) / 2
        assert slope == float((grad.double() * d.double()).sum()), name


def test_conv_bias_act8_weight_gradient_uses_the_kept_input(cuda):
    gen = torch.Generator().manual_seed(0)
    conv = nn.Conv3d(18, 72, 1).to(cuda)
    x = torch.randn(2, 18, 6, 7, 8, generator=gen).to(cuda).contiguous(memory_format=torch.channels_last_3d)
    gy = torch.randn(2, 72, 6, 7, 8, generator=gen).to(cuda)
    y, _ = bs.conv_bias_act8(conv, x, None, relu=True)
    y.backward(gy)
    flat = x.permute(0, 2, 3, 4, 1).reshape(-1).cpu().double().numpy()
    kept = torch.from_numpy(kept8(flat, False, float(np.finfo(np.float32).max))[2]).reshape(-1, 18)
    g = (gy * (y > 0)).permute(0, 2, 3, 4, 1).reshape(-1, 72).cpu().double()
    got = conv.weight.grad.flatten(1).cpu().double()
    n = g.shape[0]
    # three bf16 pieces hold a float to 2^-24, one fp32 chain and its joins: (n + 64) additions
    assert bool(((got - g.t() @ kept).abs() <= (n + 64) * 2.0 ** -24 * (g.abs().t() @ kept.abs())).all())


def test_conv_bias_act8_parts_that_are_not_wanted(cuda):
    conv, x0, gy, r0 = int_layer(cuda, 3, 18, 36, 1, (4, 4, 4), 1, 5)
    ref = None
    for frozen in ((), ("weight",), ("bias",), ("weight", "bias")):
        for need_x in (True, False):
            if not need_x and len(frozen) == 2:
                continue
            for n, p in conv.named_parameters():
                p.requires_grad_(n not in frozen)
                p.grad = None
            x = x0.to(cuda).contiguous(memory_format=torch.channels_last_3d).requires_grad_(need_x)
            y, _ = bs.conv_bias_act8(conv, x, None, residual=r0.to(cuda), relu=True)
            y.backward(gy.to(cuda))
            got = (x.grad, conv.weight.grad, conv.bias.grad)
            ref = ref or got
            assert [t is not None for t in got] == [need_x, "weight" not in frozen, "bias" not in frozen]
            assert all(a is None or torch.equal(a, b) for a, b in zip(got, ref))


def test_conv_bias_act8_shared_input_twice_and_second_backward(cuda):
    """one kept copy read by two layers and twice by one; backward a second time with retain_graph"""
    conv, x0, gy, _ = int_layer(cuda, 2, 36, 36, 1, (6, 6), 2, 7)
    x = x0.to(cuda).contiguous(memory_format=torch.channels_last).requires_grad_()
    x8 = bs.checkpoint8(x, relu=True)
    a, _ = bs.conv_bias_act8(conv, x, x8, relu=True)
    b, _ = bs.conv_bias_act8(conv, x, x8, residual=x, relu=True)
    loss = (a * gy.to(cuda)).sum() + (b * gy.to(cuda)).sum()
    loss.backward(retain_graph=True)
    first = (x.grad.clone(), conv.weight.grad.clone())
    xr = x0.double().requires_grad_()
    w = conv.weight.detach().cpu().double().requires_grad_()
    h = F.conv2d(xr, w, conv.bias.detach().cpu().double())
    ((h.relu() + (h + xr).relu()) * gy.double()).sum().backward()
    assert torch.equal(first[0].cpu().double(), xr.grad) and torch.equal(first[1].cpu().double(), w.grad)
    loss.backward()
    assert torch.equal(x.grad, 2 * first[0]) and torch.equal(conv.weight.grad, 2 * first[1])


def test_conv_bias_act8_filters_and_biases_of_any_strides(cuda):
    """a filter that is a transposed view, a bias that is a column: on a map large enough for this package's 1x1 kernel"""
    conv, x0, gy, _ = int_layer(cuda, 3, 18, 18, 1, (64, 64, 32), 1, 9)
    odd = nn.Conv3d(18, 18, 1).to(cuda)
    odd.weight = nn.Parameter(conv.weight.detach().flatten(1).t().contiguous().t().view(18, 18, 1, 1, 1))
    odd.bias = nn.Parameter(torch.stack([conv.bias.detach(), conv.bias.detach()], 1)[:, 0])
    assert odd.weight.stride()[:2] == (1, 18) and odd.bias.stride() == (2,)
    outs = []
    for c in (conv, odd):
        x = x0.to(cuda).contiguous(memory_format=torch.channels_last_3d).requires_grad_()
        y, _ = bs.conv_bias_act8(c, x, None, relu=True)
        y.backward(gy.to(cuda))
        outs.append((y.detach(), x.grad, c.weight.grad, c.bias.grad))
    assert all(torch.equal(a, b) for a, b in zip(*outs))


def test_saved_copies_may_leave_the_card(cuda):
    """what autograd holds goes through its hooks as plain tensors: kept on the host between the passes"""
    conv, x0, gy, _ = int_layer(cuda, 2, 36, 36, 1, (6, 6), 2, 7)
    grads = []
    for hooks in (False, True):
        conv.zero_grad(set_to_none=True)
        x = x0.to(cuda).contiguous(memory_format=torch.channels_last).requires_grad_()
        if hooks:
            with torch.autograd.graph.save_on_cpu():
                y, _ = bs.conv_bias_act8(conv, x, None, relu=True)
        else:
            y, _ = bs.conv_bias_act8(conv, x, None, relu=True)
        y.backward(gy.to(cuda))
        grads.append((x.grad, conv.weight.grad, conv.bias.grad))
    assert all(torch.equal(a, b) for a, b in zip(*grads))


def test_train_py_with_kept_copies(cuda, tmp_path):
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, os.path.join(root, "train.py"), "--patch", "64,64,32", "--batch", "2", "--batches", "2", "--epochs", "1", "--act8", "1", "--exp-dir", str(tmp_path)],
                       capture_output=True, text=True, timeout=110, cwd=root)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]


def test_conv_bias_act8_refusals(cuda):
    x = torch.zeros(1, 8, 4, 4, device=cuda)
    ok = nn.Conv2d(8, 8, 1).to(cuda)
    for conv, what in ((nn.Conv2d(8, 8, 1, bias=False), "a bias"), (nn.Conv2d(8, 8, 1, stride=2), "unit stride"), (nn.Conv2d(8, 8, 1, groups=2), "one group"), (nn.Conv2d(8, 8, 3), "size-preserving"),
                       (nn.Conv2d(8, 8, 3, padding="same"), "zero padding"), (nn.Conv2d(8, 8, 3, padding=1, padding_mode="reflect"), "zero padding"),
                       (nn.Conv2d(8, 8, 3, padding=2, dilation=2), "dilation")):
        with pytest.raises(ValueError, match=what):
            bs.conv_bias_act8(conv.to(cuda), x)
    with pytest.raises(ValueError, match="unit stride"):
        bs.conv_bias_act8(nn.Conv2d(8, 8, 3, padding=1, stride=2).to(cuda), x, subsampled=True)
    with pytest.raises(TypeError):
        half = nn.Conv2d(8, 8, 1).to(cuda)
        half.bias = nn.Parameter(half.bias.detach().half())
        bs.conv_bias_act8(half, x)
    with pytest.raises(ValueError, match="does not fit"):
        bs.conv_bias_act8(ok, x[:, :4])
    with pytest.raises(ValueError, match="residual"):
        bs.conv_bias_act8(ok, x, residual=x[:, :, :2])
    with pytest.raises(ValueError, match="x8"):
        bs.conv_bias_act8(ok, x, bs.checkpoint8(x[:, :, :2].contiguous(memory_format=torch.channels_last)))
    with pytest.raises(TypeError):
        bs.conv_bias_act8(ok, x.half())
    with torch.autocast("cuda", dtype=torch.bfloat16), pytest.raises(TypeError, match="autocast"):
        bs.conv_bias_act8(ok, x)
    y8 = bs.checkpoint8(x.contiguous(memory_format=torch.channels_last), relu=True)
    with pytest.raises(ValueError):
        bs.act_backward8(x[:, :4], y8)
    with pytest.raises(ValueError, match="filter"):
        bs.conv1x1_backward8(torch.zeros(4, 0, device=cuda), torch.zeros(0, 8, device=cuda), bs.checkpoint8(torch.zeros(4, 8, device=cuda)))
    with pytest.raises(ValueError):
        bs.act_backward8(torch.zeros(4, 0, device=cuda), bs.checkpoint8(torch.zeros(4, 0, device=cuda), relu=True))
    with pytest.raises(ValueError):
        bs.act_backward8(x, bs.checkpoint8(x.contiguous(memory_format=torch.channels_last)))
    with pytest.raises(TypeError):
        bs.act_backward8(x.half(), y8)


# ---- the backbone --------------------------------------------------------------------------------------------------------------------
NETS = [dict(dim=3, model="mrcnn", patch_size=[64, 64, 32], batch_size=1), dict(dim=3, model="mrcnn", patch_size=[64, 64, 32], batch_size=1, channels_last=True),
        dict(dim=2, model="mrcnn", patch_size=[96, 64], batch_size=2, channels_last=True), dict(dim=3, model="retina_unet", patch_size=[64, 64, 32], batch_size=1, channels_last=True),
        dict(dim=3, model="mrcnn", patch_size=[128, 128, 64], batch_size=2, channels_last=True)]


def two_nets(cuda, kw):
    nets = []
    for act8 in (False, True):
        torch.manual_seed(0)
        cf = Configs(act8_checkpoints=act8, **kw)
        nets.append((mrcnn if kw["model"] == "mrcnn" else retina_unet).net(cf, device=cuda))
    for a, b in zip(nets[0].parameters(), nets[1].parameters()):
        assert torch.equal(a, b)
    return nets


def rel(a, b):
    a, b = a.detach(), b.detach()
    return float((a.double() - b.double()).norm() / b.double().norm().clamp(min=1e-300))


@pytest.mark.parametrize("kw", NETS)
def test_backbone_with_kept_copies(cuda, kw):
    nets = two_nets(cuda, kw)
    gen = torch.Generator().manual_seed(1)
    img = torch.randn([kw["batch_size"], nets[0].cf.n_channels] + kw["patch_size"], generator=gen).to(cuda)
    if kw.get("channels_last"):
        img = img.contiguous(memory_format=mf_of(img))
    res, held = [], []
    for net in nets:
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        outs = net.Fpn(img) if hasattr(net, "Fpn") else net.fpn(img)
        held.append(torch.cuda.memory_allocated() - before - sum(o.numel() * 4 for o in outs))
        gens = torch.Generator().manual_seed(2)
        loss = sum((o * torch.randn(o.shape, generator=gens).to(cuda)).sum() for o in outs)
        fpn = net.Fpn if hasattr(net, "Fpn") else net.fpn
        fpn.zero_grad(set_to_none=True)
        loss.backward()
        res.append((outs, {n: p.grad for n, p in fpn.named_parameters() if p.grad is not None}))
        with torch.no_grad():
            for a, b in zip(fpn(img), outs):
                assert rel(a, b) < 1e-6
    (o0, g0), (o1, g1) = res
    assert len(o0) == len(o1) and set(g0) == set(g1)
    for a, b in zip(o0, o1):
        assert a.shape == b.shape and rel(b, a) < 1e-6
    # a bias gradient is a sum over the V voxels of its map of values of either sign, about sqrt(V) of their size, and an fp32 product's rounding may lean to one side in
    # every voxel alike: 2^-24 a layer between it and the loss, at most 50 of them, relative to the sum of magnitudes, sqrt(V) times the sum itself
    bias_tol = 50 * 2.0 ** -24 * (img.numel() / img.shape[1]) ** 0.5
    for n in g0:
        # a kept input is off by at most max / 510 of its block (max / 254 with a sign), and a block's maximum is a few times its root mean square
        assert rel(g1[n], g0[n]) < (bias_tol if n.endswith("bias") else 0.02), (n, rel(g1[n], g0[n]))
    # the full-resolution layers in front of and behind the stages of a stride-1 pyramid keep their fp32 inputs (C0's two maps and P0_conv2's input): they
    # are in both sums, (2 * 18 + 36) values a voxel here, 37.7 of 60.2 MB
    full = 4 * (2 * nets[0].cf.start_filts + nets[0].cf.end_filts) * img.numel() if nets[0].cf.operate_stride1 else 0
    assert held[1] - full < 0.55 * (held[0] - full), (held, full)


def test_backbone_copies_need_plain_relu_layers(cuda):
    for kw in (dict(norm="instance_norm"), dict(relu="leaky_relu")):
        with pytest.raises(ValueError, match="act8_checkpoints"):
            mrcnn.net(Configs(dim=3, model="mrcnn", patch_size=[64, 64, 32], batch_size=1, act8_checkpoints=True, **kw), device=cuda)


@pytest.mark.parametrize("model", ["mrcnn", "retina_unet"])
def test_training_step_with_kept_copies(cuda, model):
    """the step as train.py runs it, then inference with the box head in 4 bits on the same weights"""
    from medicaldetectiontoolkit_amd import predictor, training
    kw = dict(dim=3, model=model, patch_size=[64, 64, 32], batch_size=2, channels_last=True)
    losses = []
    for net in two_nets(cuda, kw):
        cf = net.cf
        opt = training.build_optimizer(net, cf)
        torch.manual_seed(5)
        res = training.train_step(net, opt, make_batch(cf.patch_size, 2, seed=3))
        losses.append({n: float(v) for n, v in res["loss_terms"].items()} if "loss_terms" in res else {"loss": float(res["torch_loss"])})
        assert all(bool(torch.isfinite(p).all()) for p in net.parameters())
    for n in losses[0]:
        assert abs(losses[0][n] - losses[1][n]) <= 1e-5 * abs(losses[0][n]) + 1e-6, (n, losses)
    if model == "mrcnn":
        rng = np.random.default_rng(1)
        data = rng.standard_normal((1, 80, 70, 40)).astype(np.float32)
        out = predictor.predict_patient(net, data, cf, head_dtype="mx4")
        assert out is not None and net.classifier.mx4 is None


def test_graphed_training_step_with_kept_copies(cuda):
    from medicaldetectiontoolkit_amd import training
    from tests.golden import step_inputs as si
    from tests.test_step_parity_gpu import _batch
    batch = _batch("small")
    nets = []
    for _ in range(2):
        cf = si.make_cf("mrcnn", "small")
        cf.channels_last, cf.act8_checkpoints = True, True
        net = mrcnn.net(cf, device=cuda)
        si.fill_by_name(net)
        nets.append((net, training.build_optimizer(net, cf, flat=True)))
    (net_e, opt_e), (net_g, opt_g) = nets
    step = training.GraphedTrainStep(net_g, opt_g, gmax=4, max_masks=8)
    step.capture(batch)
    for k in range(3):
        torch.manual_seed(1234)
        res_e = training.train_step(net_e, opt_e, batch, monitor=False)
        grads = {n: p.grad.detach().clone() for n, p in net_e.named_parameters() if p.grad is not None}
        torch.manual_seed(1234)
        res_g = step(batch)
        assert {n: float(v) for n, v in res_g["loss_terms"].items()} == {n: float(v) for n, v in res_e["loss_terms"].items()}, k
        for n, p in net_g.named_parameters():
            if n in grads:
                assert float((p.grad - grads[n]).abs().max()) <= 1e-5 * float(grads[n].abs().max()) + 1e-12, (k, n)
        # every replay starts from the eager step's weights: the library's weight gradients differ in their last bits from run to run, and two trajectories of their own
        # part for good where a proposal or a sampled anchor changes on that (a gradient was off by 10.1 % in the third step, once)
        with torch.no_grad():
            for a, b in zip(net_g.parameters(), net_e.parameters()):
                a.copy_(b)


# ---- the box head in 4 bits ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dim,rows", [(3, 1), (3, 7), (2, 130)])
def test_box_head_equals_its_definition(cuda, monkeypatch, dim, rows):
    kw = dict(dim=3, model="mrcnn", patch_size=[64, 64, 32], batch_size=1) if dim == 3 else dict(dim=2, model="mrcnn", patch_size=[96, 64], batch_size=2)
    net = mrcnn.net(Configs(**kw), device=cuda)
    head = net.classifier
    monkeypatch.setattr(mrcnn, "pyramid_roi_align", lambda x, rois, *a: x)
    gen = torch.Generator().manual_seed(rows)
    size = tuple(head.conv1[0].kernel_size)
    x = torch.randint(-3, 4, (rows, head.in_channels) + size, generator=gen).float()
    # 0, 1, 2, 3 and their negatives are 4-bit numbers: the first layer is exact on integers; the second rounds the first's output by blocks
    with torch.no_grad():
        for c in (head.conv1[0], head.conv2[0]):
            c.weight.copy_(torch.randint(-3, 4, c.weight.shape, generator=gen).float())
            c.bias.copy_(torch.randint(-8, 9, c.bias.shape, generator=gen).float())
    big = float(np.finfo(np.float32).max)
    h = x.double().flatten(1).numpy()
    for c in (head.conv1[0], head.conv2[0]):
        h = np.maximum(kept4(h, big)[0] @ kept4(c.weight.detach().cpu().double().flatten(1).numpy(), big)[0].T + c.bias.detach().cpu().double().numpy(), 0)
    with torch.no_grad():
        want = [F.linear(torch.from_numpy(h).float().to(cuda), l.weight, l.bias) for l in (head.linear_bbox, head.linear_class)]
        plain = head(x.to(cuda), None)
        with bs.mx4_heads(net) as inside:
            assert inside is net
            got = head(x.to(cuda), None)
        assert head.mx4 is None
        after = head(x.to(cuda), None)
        assert all(torch.equal(a, b) for a, b in zip(plain, after))
    shapes = {tuple(t.shape): t for t in got}
    for w in want:
        # (the last layers are the library's fp32 product of the same inputs; its bbox output may come in groups of coordinates)
        cand = [t.reshape(w.shape) for t in got if t.numel() == w.numel()]
        assert cand and any(rel(t, w) < 1e-6 for t in cand), shapes.keys()


def test_box_head_follows_the_weights_and_refuses_training(cuda):
    net = mrcnn.net(Configs(dim=3, model="mrcnn", patch_size=[64, 64, 32], batch_size=1), device=cuda)
    packs = []
    for s in (1.0, 2.0):
        with torch.no_grad():
            net.classifier.conv1[0].weight.fill_(s)
        with bs.mx4_heads(net):
            packs.append(net.classifier.mx4[0].dequantize())
            with pytest.raises(RuntimeError, match="already"):
                with bs.mx4_heads(net):
                    pass
            assert net.classifier.mx4 is not None
    assert bool((packs[0] == 1).all()) and bool((packs[1] == 2).all())
    with pytest.raises(KeyError):
        with bs.mx4_heads(net):
            raise KeyError("from inside")
    assert net.classifier.mx4 is None
    from medicaldetectiontoolkit_amd import training
    opt = training.build_optimizer(net, net.cf)
    with bs.mx4_heads(net), pytest.raises(RuntimeError, match="no autograd graph"):
        training.train_step(net, opt, make_batch(net.cf.patch_size, 1, seed=0))


def test_test_set_prediction_rounds_every_checkpoint(cuda, tmp_path):
    """two checkpoints of an ensemble: each is rounded after it was loaded"""
    from medicaldetectiontoolkit_amd import predictor, training
    from medicaldetectiontoolkit_amd.utils import exp_utils
    cf = Configs(dim=3, model="mrcnn", patch_size=[64, 64, 32], batch_size=4)
    torch.manual_seed(0)
    net = mrcnn.net(cf, device=cuda)
    ck, seen = [], []
    for ep in (1, 2):
        with torch.no_grad():
            net.classifier.conv1[0].weight.fill_(float(ep))
        exp_utils.save_best_checkpoint(str(tmp_path), net, ep)
        ck.append(str(tmp_path / ("%d_best_checkpoint" % ep)))
    patients = [(np.random.default_rng(1).standard_normal((1, 80, 70, 40)).astype(np.float32), "p0")]
    forward = net.classifier._forward

    def spy(x, rois):
        seen.append(float(net.classifier.mx4[0].dequantize().max()))
        return forward(x, rois)
    net.classifier._forward = spy
    res = predictor.predict_test_set(net, patients, cf, checkpoint_paths=ck, test_aug=False, head_dtype="mx4")
    assert len(res) == 1 and set(seen) == {1.0, 2.0}
    for amp in (torch.bfloat16,):
        out = predictor.predict_patient(net, patients[0][0], cf, amp_dtype=amp, head_dtype="mx4")
        assert out is not None
