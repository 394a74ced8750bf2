"""Block-scaled operators (utils/block_scaled.py) at their edges: layers whose passes run on several streams or inside a captured graph, every kernel of the 1x1 backward pass and
of the 4-bit product, the ends of the number range, tensors of more than 2^31 values, backbones with hooks and in other forms.

Compared on numbers whose products and sums are exact in fp32: equality."""
import copy

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from medicaldetectiontoolkit_amd import _lib
from medicaldetectiontoolkit_amd.utils import block_scaled as bs
from medicaldetectiontoolkit_amd.utils import fused_epilogue as fe
from tests.test_block_scaled_gpu import BIG, DTYPES, f64, hard_values, kept4, kept8, layer, same
from tests.test_block_scaled_models_gpu import int_layer, mf_of, rel, two_nets

pytestmark = pytest.mark.gpu


# ---- scratch memory of a 3x3x3 layer -------------------------------------------------------------------------------------------------
def window_job(cuda, ci, co, size, seed):
    """a layer whose three products run on this package's kernels (65536 voxels or more, extents of 32): module, input, output gradient"""
    conv, x, gy, _ = int_layer(cuda, 3, ci, co, 3, size, 1, seed)
    return conv, x.to(cuda).contiguous(memory_format=torch.channels_last_3d), gy.to(cuda).contiguous(memory_format=torch.channels_last_3d)


def window_grads(conv, x0, gy):
    x = x0.clone().requires_grad_()
    y, _ = bs.conv_bias_act8(conv, x, None, keep=False)
    return (y.detach(),) + torch.autograd.grad(y, [x, conv.weight, conv.bias], gy)


def window_definition(conv, x0, gy):
    """64 bits, on the host"""
    x, w, b = x0.cpu().double().requires_grad_(), conv.weight.detach().cpu().double().requires_grad_(), conv.bias.detach().cpu().double().requires_grad_()
    y = F.conv3d(x, w, b, padding=1)
    return (y.detach(),) + torch.autograd.grad(y, [x, w, b], gy.cpu().double())


def test_window_layer_is_exact_and_takes_no_shared_buffers(cuda, monkeypatch):
    """neither the scratch memory nor the flipped filters that the fp32 layers keep for a device"""
    conv, x, gy = window_job(cuda, 18, 18, (32, 32, 64), 1)

    def shared(*a, **k):
        raise AssertionError("a buffer of the device, not of the call")
    monkeypatch.setattr(fe, "_workspace", shared)
    monkeypatch.setattr(fe._FlipCache, "get", shared)
    got = window_grads(conv, x, gy)
    assert all(torch.equal(a.cpu().double(), b) for a, b in zip(got, window_definition(conv, x, gy)))


def test_window_layers_on_two_streams(cuda):
    """input and weight gradients of layers of several sizes, their filters changed between the rounds, equal to one layer after the other"""
    jobs = [window_job(cuda, 18, 18, (32, 32, 64), 1), window_job(cuda, 6, 10, (64, 32, 64), 2), window_job(cuda, 18, 18, (64, 64, 32), 3)]
    streams = [torch.cuda.Stream() for _ in jobs]
    for rep in range(4):
        with torch.no_grad():
            for conv, _, _ in jobs:
                conv.weight.copy_(torch.randint(-3, 4, conv.weight.shape, device=cuda).float())
        plain = [tuple(t.clone() for t in window_grads(*copy.deepcopy(j))) for j in jobs]
        torch.cuda.synchronize()
        got = []
        for j, s in zip(jobs, streams):
            with torch.cuda.stream(s):
                got.append(window_grads(*j))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for p, g in zip(plain, got) for a, b in zip(p, g)), rep
        if rep == 0:
            assert all(torch.equal(a.cpu().double(), b) for j, g in zip(jobs, got) for a, b in zip(g, window_definition(*j)))


def test_layers_captured_and_replayed(cuda):
    """a 3x3x3 and a 1x1x1 layer, both passes, in a graph of torch's own; an eager step of the same layers and larger ones between the replays"""
    window, x, gy = window_job(cuda, 18, 18, (32, 32, 64), 4)
    one = int_layer(cuda, 3, 18, 72, 1, (4, 4, 4), 1, 5)[0]
    gy1 = torch.randint(-4, 5, (1, 72, 32, 32, 64), device=cuda).float().contiguous(memory_format=torch.channels_last_3d)
    large = window_job(cuda, 18, 18, (64, 64, 64), 6)

    def step(window, one):
        xs = x.detach().requires_grad_()
        h, h8 = bs.conv_bias_act8(window, xs, None, relu=True)
        y, _ = bs.conv_bias_act8(one, h, h8, relu=True)
        return torch.autograd.grad(y, [xs, window.weight, window.bias, one.weight, one.bias], gy1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(window, one)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(window, one)
    for rep in range(4):
        with torch.no_grad():
            x.copy_(torch.randint(0, 3, x.shape, device=cuda))
            gy1.copy_(torch.randint(-1, 2, gy1.shape, device=cuda))
            for p in (window.weight, one.weight):
                p.copy_(torch.randint(-1, 2, p.shape, device=cuda))
        want = [t.clone() for t in step(window, one)]               # the eager step before the replay: it must not depend on what the graph prepared
        window_grads(*large)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), rep
        assert all(torch.equal(a, b) for a, b in zip(step(*copy.deepcopy((window, one))), want)), rep


# ---- the tiled and one-pass kernels of the 1x1 backward pass ---------------------------------------------------------------------------
def backward_variant(V, ci, co, need_gx=True, need_gw=True):
    """the kernels that mdt_conv1x1_act8_backward takes, restated: (one-pass tiles,) or (gw tile, gx tile, gx's sum split, input channels a multiple of 4)"""
    if V * ci < 4 or V * co < 4:
        return ("tiny",)
    mt, nt = -(-co // 32), -(-ci // 32)
    if need_gx and need_gw and co <= 160 and ci <= 160 and mt * nt <= 10:
        ks, wave = -(-co // 16), (32 * max(co, ci) + 32 * mt + (32 * ci + 32 * nt) // 2 + 3) // 4 * 4
        lds = max(nt * ks * 3 * 1024 + 4 * wave * 4, (4 if mt * nt <= 9 else 2) * (1024 * mt * nt + 32 * mt) * 4)
        if lds <= 160 * 1024:
            return (mt, nt)
    gw = (128 if co > 64 else 64, 128 if ci > 64 else 64) if need_gw else None
    gx = split = None
    if need_gx:
        dn = 128 if ci > 64 and -(-V // 128) * -(-ci // 128) >= 256 else 64
        dm = 128 if dn == 128 or -(-ci // 64) % 2 == 0 else 64
        now, steps = -(-V // dn) * -(-ci // dm), -(-co // 32)
        gx, split = (dm, dn), max(1, min(-(-256 // now), steps // 4)) > 1
    return gw, gx, split, ci % 4 == 0


# one-pass: a tile a side and the others; tiled: gw 128 x 128, 128 x 64, 64 x 128, gx 64 x 64, 128 x 64, 128 x 128 (split and not), channels that are multiples of 4 or not
VARIANTS = [(700, 18, 72), (700, 72, 18), (1100, 36, 144), (1100, 144, 36), (900, 96, 96), (901, 31, 160), (903, 160, 29), (600, 64, 64), (500, 37, 300), (500, 36, 300), (450, 200, 300), (450, 201, 300),
            (460, 300, 40), (460, 301, 40), (17000, 100, 200), (17000, 101, 200), (20001, 37, 170), (20003, 36, 170), (16389, 200, 65), (16390, 202, 66), (11003, 300, 40), (11003, 301, 63),
            (32771, 101, 200), (32771, 104, 200), (16500, 150, 70), (16500, 148, 70), (450, 150, 300), (450, 152, 300), (20000, 170, 33), (20000, 172, 33), (450, 330, 17), (450, 332, 17), (450, 150, 70), (450, 152, 70),
            (601, 31, 33), (3, 1, 1)]


def test_the_cases_reach_every_kernel_of_the_backward_pass():
    seen = {backward_variant(*s) for s in VARIANTS}
    for ci4 in (True, False):
        for gw in ((128, 128), (128, 64), (64, 128)):
            got = {(v[1], v[2]) for v in seen if len(v) == 4 and v[0] == gw and v[3] == ci4}
            want = {((64, 64), False)} if gw == (128, 64) else {((64, 64), False), ((128, 64), False), ((128, 128), False)}
            assert want <= got, (gw, ci4, want - got)
        assert any(len(v) == 4 and v[2] and v[3] == ci4 and v[1] == t for v in seen for t in ((64, 64),)) and any(len(v) == 4 and v[2] and v[3] == ci4 and v[1] == (128, 64) for v in seen)
    assert {(3, 1), (1, 3), (5, 2), (2, 5), (3, 3), (5, 1), (1, 5), (2, 2)} <= seen


def single_products(V, ci, co, seed, cuda):
    """(g, w, x) of which every gx and every gw is one product: row v of g holds one value, at v % co, and of x the value at (v // co) % ci, rows behind co * ci none; powers
    of two where the other factor has all its bits"""
    gen = torch.Generator().manual_seed(seed)
    v = torch.arange(V)
    at_o, at_i, one = v % co, v // co % ci, v < co * ci
    x = torch.zeros(V, ci)
    x[v[one], at_i[one]] = torch.exp2(torch.randint(0, 4, (int(one.sum()),), generator=gen).float())

    def bits(*shape):
        return torch.randint(2 ** 23, 2 ** 24, shape, generator=gen).float() * (torch.randint(0, 2, shape, generator=gen) * 2 - 1)

    def powers(*shape):
        return torch.exp2(torch.randint(-3, 4, shape, generator=gen).float())
    cases = []
    for gv, w in ((bits(V), powers(co, ci)), (powers(V), bits(co, ci))):
        g = torch.zeros(V, co)
        g[v, at_o] = gv
        cases.append((g, w, torch.exp2(torch.randint(-40, 40, (V, 1), generator=gen).float())))
    return x.to(cuda), [(g.to(cuda), w.to(cuda), s.to(cuda)) for g, w, s in cases]


@pytest.mark.parametrize("V,ci,co", VARIANTS)
def test_conv1x1_backward8_keeps_all_bits_of_a_product(cuda, V, ci, co):
    """gradients and filters of 24 significant bits: the three pieces that a float is cut into are all needed, at any size of the gradient"""
    x, cases = single_products(V, ci, co, V + ci, cuda)
    x8 = bs.checkpoint8(x, relu=True)
    assert torch.equal(x8.restore(), x)
    for g, w, size in cases:
        for scale in (1.0, size):
            gs = g * scale
            gx, gw, gb, _ = bs.conv1x1_backward8(gs, w, x8, None)
            gd, wd, xd = gs.double(), w.double(), x.double()
            assert torch.equal(gx.double(), gd @ wd) and torch.equal(gw.double(), gd.t() @ xd)
            for kw in (dict(need_gx=False), dict(need_gw=False)):
                part = bs.conv1x1_backward8(gs, w, x8, None, **kw)
                assert all(a is None or torch.equal(a, b) for a, b in zip(part[:2], (gx, gw)))


@pytest.mark.parametrize("relu", [True, False])
@pytest.mark.parametrize("V,ci,co", VARIANTS)
def test_conv1x1_backward8_variants_on_integers(cuda, V, ci, co, relu):
    """every kernel, masked or not, with and without the residual's gradient, its parts alone: |sums| < 2^24, so the results are the exact ones"""
    x, gy, w, y = layer(V, ci, co, True, V + ci, cuda)
    gy = gy.clamp(-4, 4)                                              # 32771 voxels of 15 * 4
    x8, y8 = bs.checkpoint8(x, relu=True), bs.checkpoint8(y, relu=True) if relu else None
    m = gy * (y > 0) if relu else gy
    want = (m.double() @ w.double(), m.double().t() @ x.double(), m.double().sum(0))
    for kw in (dict(need_g=True), dict(), dict(need_gx=False), dict(need_gw=False), dict(need_gw=False, need_g=True), dict(need_gx=False, need_g=True)):
        got = bs.conv1x1_backward8(gy, w, x8, y8, **kw)
        assert all(a is None or torch.equal(a.double(), b) for a, b in zip(got, want))
        assert got[3] is None or torch.equal(got[3], m)


@pytest.mark.parametrize("V,ci,co", [s for s in VARIANTS if s[0] > 3])
def test_conv1x1_backward8_variants_keep_fp32_accuracy(cuda, V, ci, co):
    """every kernel on floats, the error in 2-norm: products are off by 2^-23 at most (what three pieces leave out), and an fp32 sum of values of either sign by a random walk of
    roundings that stays below 16 of them for 2^15 values in partial sums"""
    x, gy, w, y = layer(V, ci, co, False, V + co, cuda)
    x8, y8 = bs.checkpoint8(x, relu=True), bs.checkpoint8(y, relu=True)
    gx, gw, gb, _ = bs.conv1x1_backward8(gy, w, x8, y8)
    md, xd = (gy * (y > 0)).double(), x8.restore().double()
    for got, want in ((gw, md.t() @ xd), (gx, md @ w.double()), (gb, md.sum(0))):
        assert float((got.double() - want).norm() / want.norm()) < 16 * 2.0 ** -24


EXTREME = [(40, 18, 72), (40, 72, 18), (40, 37, 300), (40, 300, 40), (40, 200, 300), (33000, 101, 200), (2, 1, 1)]


@pytest.mark.parametrize("V,ci,co", EXTREME)
def test_conv1x1_backward8_of_the_largest_finite_values(cuda, V, ci, co):
    """gradients and filters between the largest bf16 and the largest fp32 number: a finite product stays what it is"""
    x, cases = single_products(V, ci, co, 7, cuda)
    x = x.clamp(max=1)
    x[min(V, co):] = 0
    x8 = bs.checkpoint8(x, relu=True)
    top = torch.finfo(torch.float32).max
    for k, (g, w, _) in enumerate(cases):
        g = torch.sign(g)
        g[min(V, co):] = 0                                            # a value a column: no sum passes the largest number
        w = torch.sign(torch.randn(co, ci, generator=torch.Generator().manual_seed(3))).to(cuda)
        big = torch.rand(g.shape if k == 0 else w.shape, generator=torch.Generator().manual_seed(4)).to(cuda) * (top - 3.39e38) + 3.39e38
        big.view(-1)[0] = top
        g, w = (g * big, w * 0.5) if k == 0 else (g * 0.5, w * big)
        gx, gw, gb, gr = bs.conv1x1_backward8(g, w, x8, None, need_g=True)
        gd = g.double()
        assert torch.isfinite(gd @ w.double()).all() and torch.equal(gx.double(), gd @ w.double())
        assert torch.equal(gw.double(), gd.t() @ x.double()) and torch.equal(gb.double(), gd.sum(0)) and torch.equal(gr, g)


@pytest.mark.parametrize("V,ci,co", [(40, 18, 72), (40, 37, 300), (450, 300, 40)])
def test_conv1x1_backward8_of_the_smallest_values(cuda, V, ci, co):
    """a piece below 2^-133 does not exist in bf16: gradients keep all their bits from 2^-110 on, and smaller ones are off by less than 2^-133"""
    x, cases = single_products(V, ci, co, 11, cuda)
    x = x.clamp(max=1)
    x8 = bs.checkpoint8(x, relu=True)
    g, w, _ = cases[0]
    w = torch.sign(w)
    for e in (-86, -133, -140, -149):                                # the last: numbers around the smallest normal one
        gs = (g.double() * 2.0 ** e).float()
        gx, gw, gb, _ = bs.conv1x1_backward8(gs, w, x8, None)
        gd = gs.double()
        tol = 0 if e >= -133 else 2.0 ** -133
        assert bool(((gx.double() - gd @ w.double()).abs() <= tol).all()) and bool(((gw.double() - gd.t() @ x.double()).abs() <= tol).all()), e


# ---- the 4-bit product's kernels -------------------------------------------------------------------------------------------------------
def linear_variant(rows, k, n, size):
    """the kernel that mdt_mx4_linear takes, restated: (shape, W's form, 16-row tiles of x, 16-column tiles)"""
    wide = n > 144 and (rows >= 2048 or (rows >= 512 and k >= 4096))
    copies = wide or (rows >= 256 and k >= 4096)
    if wide:
        ranges = -(-n // 768)
        short, long = -(-(-(-rows // 16) * ranges) // 256), -(-(-(-rows // 48) * ranges) // 256)
        return "wide", "copied", 1 if 6 * short < 10 * long else 3, min(6, max(2, -(-n // (128 * ranges))))
    if not copies and rows * k < 16 // size:
        return "narrow", "tiny", 1, 1
    t = -(-rows // 16)
    tn = 9 if n > 48 and t * -(-n // 144) >= 96 else 3 if n > 16 and t * -(-n // 48) >= 96 else 1
    return "narrow", "copied" if copies else "one block" if k <= 32 else "kept", 1, tn


LINEAR_MORE = [(261, 4099, 9), (777, 4131, 47), (1601, 4100, 47), (1601, 4100, 141), (600, 4200, 200), (1700, 4097, 300), (2051, 100, 200), (2051, 100, 300), (2051, 100, 500), (2051, 100, 600), (2051, 100, 767),
               (4099, 70, 150), (4099, 70, 380), (4099, 70, 500), (4099, 70, 600), (4099, 70, 767), (4099, 300, 900), (1601, 31, 100), (1601, 29, 47), (40, 17, 300), (1601, 290, 100), (1603, 290, 47),
               (50, 290, 33), (1, 3, 7)]


def test_the_cases_reach_every_kernel_of_the_4_bit_product():
    for size in (2, 4):
        seen = {linear_variant(*s, size) for s in LINEAR_MORE}
        assert {("wide", "copied", tm, tn) for tm in (1, 3) for tn in (2, 3, 4, 5, 6)} <= seen
        assert all((linear_variant(*s, size)[1] == "copied") == (_lib.lib().mdt_mx4_linear_workspace_bytes(*s) > 0) for s in LINEAR_MORE)
        assert {("narrow", w, 1, tn) for w in ("copied", "one block", "kept") for tn in (1, 3, 9)} | {("narrow", "tiny", 1, 1)} <= seen


@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,n", LINEAR_MORE)
def test_mx4_linear_variants_on_integers(cuda, rows, k, n, dtype, relu):
    """numbers that 4 bits hold exactly, sums below 2^24: the exact result, rounded once to the type"""
    g = torch.Generator().manual_seed(rows + n)
    vals = torch.tensor([0.0, 1, 2, 3, 4, 6, -1, -2, -3, -4, -6])
    x, w = vals[torch.randint(0, 11, (rows, k), generator=g)].to(cuda), vals[torch.randint(0, 11, (n, k), generator=g)].to(cuda)
    bias = torch.randint(-9, 9, (n,), generator=g).float().to(cuda)
    y = bs.mx4_linear(x.to(dtype), bs.mx4_quantize(w), bias, relu=relu)
    want = x.double() @ w.double().t() + bias.double()
    assert y.dtype == dtype and torch.equal(y, (want.clamp(min=0) if relu else want).to(dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,n", LINEAR_MORE)
def test_mx4_linear_variants_on_floats(cuda, rows, k, n, dtype):
    """exact products, k fp32 sums and the bias, then one rounding: half a step each"""
    g = torch.Generator().manual_seed(rows + k)
    x = (torch.randn(rows, k, generator=g) * torch.exp(torch.randn(k, generator=g))).to(dtype)
    w, bias = torch.randn(n, k, generator=g) / k ** 0.5, torch.randn(n, generator=g)
    y = bs.mx4_linear(x.to(cuda), bs.mx4_quantize(w.to(cuda)), bias.to(cuda))
    xv, wv = (torch.from_numpy(kept4(f64(t), BIG[t.dtype])[0]).to(cuda) for t in (x, w))
    want = xv @ wv.t() + bias.to(cuda).double()
    tol = (k + 64) * 2.0 ** -24 * (xv.abs() @ wv.abs().t() + bias.to(cuda).abs().double()) + torch.finfo(dtype).eps / 2 * want.abs()
    assert bool(((y.double() - want).abs() <= tol * (1 + 1e-6)).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,n", [(70, 512), (300, 512), (2100, 512)])
def test_mx4_linear_rounds_x_as_mx4_quantize_does(cuda, rows, n, dtype):
    """W = the unit matrix: a row of x comes back as its 4-bit values.  Ties, subnormals and numbers of very different size in whole chunks and ragged ones; a row with an infinity or a NaN is NaN,
    and no other row"""
    x = hard_values(rows * n, dtype, rows)
    x[~torch.isfinite(x)] = 1
    x[x.abs() > BIG[dtype] / 4] = 5                                   # (a sum of one value rounded up across the type's largest is an infinity, no saturated code)
    x = x.view(rows, n)
    x[5] = x[0].roll(32)
    if dtype == torch.float16:
        x[7, :64] = torch.arange(64) * 2.0 ** -24                     # fp16's smallest numbers
        x[8, :64] = torch.arange(64) * 2.0 ** -20 - 2.0 ** -15
    elif dtype == torch.bfloat16:
        x[7, :64] = (torch.arange(64).double() * 2.0 ** -133).to(dtype)
        x[8, :64] = (torch.arange(64).double() * 2.0 ** -126).to(dtype)
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0]).repeat(8)
    x[9, :64], x[10, :64], x[11, :64] = ties, -ties * 2.0 ** 3, ties.to(dtype) * (1 + torch.finfo(dtype).eps)
    eye = bs.mx4_quantize(torch.eye(n, device=cuda))
    xd = x.to(cuda)
    v = torch.from_numpy(kept4(f64(x), BIG[dtype])[0]).to(dtype)
    assert torch.equal(bs.mx4_linear(xd, eye).cpu(), v)
    at = {3: float("inf"), 20: float("nan"), 33: -float("inf"), rows - 1: float("nan")}
    for r, bad in at.items():
        xd[r, 37 * r % n] = bad
    y = bs.mx4_linear(xd, eye).cpu()
    assert all(torch.isnan(y[r]).all() for r in at)
    keep = torch.tensor([r not in at for r in range(rows)])
    assert torch.equal(y[keep], v[keep])


def test_two_streams_and_copies_of_w(cuda):
    """products that copy W into scratch memory, another W and another size on each stream"""
    jobs = []
    for i, (rows, k, n) in enumerate([(300, 5292, 144), (700, 4200, 200), (2500, 600, 400), (300, 4100, 33)]):
        x, w = torch.randn(rows, k, device=cuda), bs.mx4_quantize(torch.randn(n, k, device=cuda))
        assert _lib.lib().mdt_mx4_linear_workspace_bytes(rows, k, n) > 0
        jobs.append((x, w, bs.mx4_linear(x, w)))
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in jobs], []
    for rep in range(6):
        for s, (x, w, want) in zip(streams, jobs):
            with torch.cuda.stream(s):
                outs.append((bs.mx4_linear(x, w), want))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in outs)


# ---- tensors of more than 2^31 values --------------------------------------------------------------------------------------------------
def around(n):
    """ranges of indexes at the start, around 2^31 and at the end"""
    return [slice(0, 4096), slice(2 ** 31 - 4096, min(n, 2 ** 31 + 4096)), slice(n - 4099, n)]


@pytest.mark.parametrize("dtype", DTYPES)
def test_checkpoint8_of_more_than_2_31_values(cuda, dtype):
    n = 2 ** 31 + 100037
    x = torch.empty(n, dtype=dtype, device=cuda)
    x.copy_(torch.randn(10007, device=cuda).repeat(-(-n // 10007))[:n])
    ck = bs.checkpoint8(x, relu=True)
    back = ck.restore()
    for s in around(n):
        first = s.start // 32 * 32
        q, b, v = kept8(f64(x[first:s.stop]), True, BIG[dtype])
        assert same(f64(back[first:s.stop]), v) and same(ck.codes[first:s.stop].cpu().numpy(), q)
        assert same(ck.scales[first // 32:-(-s.stop // 32)].cpu().numpy()[:s.stop // 32 - first // 32], b[:s.stop // 32 - first // 32])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_mx4_of_more_than_2_31_values(cuda, dtype):
    rows, k = 2 ** 31 // 4500 + 23, 4500
    x = torch.empty(rows * k, dtype=dtype, device=cuda)
    x.copy_(torch.randn(10007, device=cuda).repeat(-(-rows * k // 10007))[:rows * k])
    x = x.view(rows, k)
    m = bs.mx4_quantize(x)
    back = m.dequantize()
    picks = [0, 1, 2 ** 31 // 4500 - 1, 2 ** 31 // 4500, 2 ** 31 // 4500 + 1, rows - 1]
    v = kept4(f64(x[picks]), BIG[dtype])[0]
    assert same(f64(back[picks]), v)
    del back
    w = torch.zeros(9, k, device=cuda)
    w[torch.arange(9), torch.arange(9) * 501] = 1
    y = bs.mx4_linear(x, bs.mx4_quantize(w))
    assert same(f64(y[picks]), v[:, ::501][:, :9])


@pytest.mark.parametrize("V,ci,co", [(2 ** 31 // 72 + 1001, 72, 72), (2 ** 31 // 300 + 77, 300, 330)])
def test_conv1x1_backward8_of_more_than_2_31_values(cuda, V, ci, co):
    """gradients at a few voxels of a map whose offsets pass 31 bits; the sums alone, the mask and the epilogue on the same map"""
    at = torch.tensor([0, 1, 2 ** 31 // co - 1, 2 ** 31 // co, 2 ** 31 // co + 1, 2 ** 31 // ci - 1, 2 ** 31 // ci, V - 2, V - 1])
    at = at[at < V].unique().to(cuda)
    x = torch.zeros(V, ci, device=cuda)
    x[at] = torch.randint(1, 16, (len(at), ci), device=cuda).float()
    x8 = bs.checkpoint8(x, relu=True)
    del x
    y8 = bs.Checkpoint8(torch.ones(V * co, dtype=torch.uint8, device=cuda), torch.full((-(-V * co // 32),), 127, dtype=torch.uint8, device=cuda), (V, co), relu=True)
    gy = torch.zeros(V, co, device=cuda)
    gy[at] = torch.randint(-8, 9, (len(at), co), device=cuda).float()
    w = torch.randint(-8, 9, (co, ci), device=cuda).float()
    gx, gw, gb, g = bs.conv1x1_backward8(gy, w, x8, y8, need_g=True)
    gd = gy[at].double()
    xd = x8.codes.view(V, ci)[at].double()
    assert torch.equal(g[at], gy[at]) and int(g.count_nonzero()) == int(gy.count_nonzero())
    want = gd @ w.double()
    assert torch.equal(gx[at].double(), want) and int(gx.count_nonzero()) == int(want.count_nonzero())
    scale = torch.stack([x8.scales[(a * ci + torch.arange(ci, device=cuda)) // 32].double() for a in at])
    assert torch.equal(gw.double(), gd.t() @ (xd * torch.exp2(scale - 127))) and torch.equal(gb.double(), gd.sum(0))
    del gx, g
    g, gb = bs.act_backward8(gy, y8)
    assert torch.equal(g[at], gy[at]) and torch.equal(gb.double(), gd.sum(0)) and int(g.count_nonzero()) == int(gy.count_nonzero())
    del g
    y, ck = bs.bias_act_checkpoint8(gy, torch.full((co,), 2.0, device=cuda), relu=True)
    assert torch.equal(y[at], (gy[at] + 2).clamp(min=0)) and float(y[V // 2].min()) == 2.0 and int((ck.codes > 0).sum()) == int((y > 0).sum())


# ---- the backbone: hooks, switches, other forms ----------------------------------------------------------------------------------------
def pyramid(net, img):
    fpn = net.Fpn if hasattr(net, "Fpn") else net.fpn
    fpn.zero_grad(set_to_none=True)
    outs = fpn(img)
    gen = torch.Generator().manual_seed(2)
    sum((o * torch.randn(o.shape, generator=gen).to(o.device)).sum() for o in outs).backward()
    return fpn, [o.detach() for o in outs], {n: p.grad for n, p in fpn.named_parameters() if p.grad is not None}


def image_of(net, kw, cuda):
    img = torch.randn([kw["batch_size"], net.cf.n_channels] + kw["patch_size"], generator=torch.Generator().manual_seed(1)).to(cuda)
    return img.contiguous(memory_format=mf_of(img)) if kw.get("channels_last") else img


@pytest.fixture
def repeatable(kw):
    """MIOpen's 2D convolutions split sums over atomics: two passes of one net differ in their last bits, and a unit of a ReLU that is zero but for these bits has a gradient in the one and
    none in the other.  Torch's own convolutions there (MIOpen's 3D ones are deterministic): the forward values of two nets are equal, and so are their masks"""
    with torch.backends.cudnn.flags(enabled=kw["dim"] == 3):
        yield


def same_pyramids(a, b, img, kw):
    """channels-last nets: the stages' outputs of the fp32 path bit for bit; bias gradients within 50 layers' roundings of a sum of values of either sign over the map's voxels (2^-24 a layer of
    the sum of magnitudes, sqrt(voxels) times the sum itself), filters' gradients within what half a step of a block allows.  Row-major nets run other kernels of the library with the option than without, so only their outputs are compared (see repeatable)"""
    (_, o0, g0), (_, o1, g1) = a, b
    assert len(o0) == len(o1) and set(g0) == set(g1)
    if not kw.get("channels_last"):
        assert all(p.shape == q.shape and rel(q, p) < 1e-6 for p, q in zip(o0, o1))
        return
    front = len(o0) - (5 if kw.get("sixth_pooling") else 4)          # levels behind the interpolations of a stride-1 pyramid, which have a kernel for each memory layout
    assert all(torch.equal(p, q) for p, q in zip(o0[front:], o1[front:])) and all(rel(q, p) < 1e-6 for p, q in zip(o0[:front], o1[:front]))
    for n in g0:
        level = int(n[1])                                             # C3.0.conv1.0.bias, P5_conv2.weight
        voxels = o0[front + level - 2][:, 0].numel() if level >= 2 else img[:, 0].numel()
        assert rel(g1[n], g0[n]) < (50 * 2.0 ** -24 * voxels ** 0.5 if n.endswith("bias") else 0.02), (n, rel(g1[n], g0[n]))


HOOKED = [dict(dim=3, model="mrcnn", patch_size=[64, 64, 32], batch_size=1, channels_last=True), dict(dim=2, model="mrcnn", patch_size=[96, 64], batch_size=2, channels_last=True),
          dict(dim=2, model="mrcnn", patch_size=[64, 64], batch_size=1)]


@pytest.mark.parametrize("kw", HOOKED)
def test_hooks_run_as_without_copies(cuda, repeatable, kw):
    """hooks of every kind on every module: the same ones run, in the same order"""
    seen, res = [], []
    for net in two_nets(cuda, kw):
        names = []
        fpn = net.Fpn if hasattr(net, "Fpn") else net.fpn
        for n, m in fpn.named_modules():
            m.register_forward_hook(lambda m, i, o, n=n, names=names: names.append(n))
            m.register_forward_pre_hook(lambda m, i, n=n, names=names: names.append("pre " + n))
        img = image_of(net, kw, cuda)
        res.append(pyramid(net, img))
        seen.append(names)
    assert seen[0] == seen[1] and any("C4.1.conv2" == n for n in seen[0]) and any("P2_conv2" == n for n in seen[0])
    same_pyramids(*res, img, kw)


@pytest.mark.parametrize("where", [("C1",), ("C2.0",), ("C2.1",), ("C3.0.conv2", "P5_conv1"), ("C4.2.conv3", "P3_conv2"), ("C5.1.conv1",), ("C5.2",), ("P2_conv2", "P4_conv2")])
@pytest.mark.parametrize("kw", HOOKED[:2])
def test_a_hook_that_changes_an_output(cuda, repeatable, kw, where):
    """also to values of the other sign, behind a ReLU"""
    res = []
    for net in two_nets(cuda, kw):
        fpn = net.Fpn if hasattr(net, "Fpn") else net.fpn
        modules = dict(fpn.named_modules())
        for n in where:
            modules[n].register_forward_hook(lambda m, i, o: o * -1.5)
        img = image_of(net, kw, cuda)
        res.append(pyramid(net, img))
    same_pyramids(*res, img, kw)


def test_the_switch_of_the_1x1_kernel_holds(cuda, monkeypatch):
    """a layer that the kernel would take, with and without it"""
    conv, x0, gy, _ = int_layer(cuda, 3, 18, 72, 1, (64, 64, 32), 1, 9)
    calls, real = [], fe._conv1x1_forward
    monkeypatch.setattr(fe, "_conv1x1_forward", lambda *a: calls.append(1) or real(*a))
    outs = []
    for on, enabled in ((True, True), (False, True), (True, False)):
        monkeypatch.setattr(fe, "CONV1X1_FWD", on)
        monkeypatch.setattr(fe, "ENABLED", enabled)
        x = x0.to(cuda).contiguous(memory_format=torch.channels_last_3d).requires_grad_()
        y, y8 = bs.conv_bias_act8(conv, x, None, relu=True)
        outs.append((y.detach(), y8.restore()) + torch.autograd.grad(y, [x, conv.weight, conv.bias], gy.to(cuda)))
        assert len(calls) == 1
    assert all(torch.equal(a, b) for o in outs[1:] for a, b in zip(o, outs[0]))


@pytest.mark.parametrize("kw", [dict(dim=3, model="mrcnn", patch_size=[64, 64, 32], batch_size=1, channels_last=True, sixth_pooling=True),
                                dict(dim=3, model="mrcnn", patch_size=[128, 128, 64], batch_size=2, channels_last=True),
                                dict(dim=2, model="mrcnn", patch_size=[128, 96], batch_size=2, channels_last=True, res_architecture="resnet101"),
                                dict(dim=2, model="retina_unet", patch_size=[96, 64], batch_size=2, channels_last=True), dict(dim=2, model="retina_unet", patch_size=[64, 64], batch_size=1)])
def test_other_backbones_with_kept_copies(cuda, repeatable, kw):
    """a sixth level, larger maps, the deep architecture, the 2D pyramid at unit stride"""
    res = []
    for net in two_nets(cuda, kw):
        img = image_of(net, kw, cuda)
        res.append(pyramid(net, img))
    same_pyramids(*res, img, kw)


@pytest.mark.parametrize("k,size,B", [(1, (4, 4, 4), 0), (3, (4, 4, 4), 0), (1, (4, 6), 0), (3, (4, 6), 0), (1, (1, 1, 1), 1), (3, (1, 1, 1), 1), (3, (1, 1), 1)])
@pytest.mark.parametrize("relu", [True, False])
def test_layers_without_voxels_and_with_one(cuda, k, size, B, relu):
    nd = len(size)
    conv, x, gy, r = int_layer(cuda, nd, 6, 10, k, size, B, 3)
    x, r = x.to(cuda).requires_grad_(), r.to(cuda).requires_grad_()
    y, y8 = bs.conv_bias_act8(conv, x, None, residual=r, relu=relu)
    got = torch.autograd.grad(y, [x, r, conv.weight, conv.bias], gy.to(cuda))
    assert y.shape == gy.shape and y8.shape == tuple(gy.shape) and y8.restore().shape == gy.shape
    xd, rd, w, b = (t.detach().cpu().double().requires_grad_() for t in (x, r, conv.weight, conv.bias))
    h = (F.conv3d if nd == 3 else F.conv2d)(xd, w, b, padding=k // 2) + rd
    want = torch.autograd.grad(h.relu() if relu else h, [xd, rd, w, b], gy.double())
    # 1x1 layers are exact; the library may take a window through a minimal-filtering transform: sums of at most 10 * 3^3 products, and 64 times their rounding (see the window layers' test)
    xa, ra, wa, ba = (t.detach().abs().requires_grad_() for t in (xd, rd, w, b))
    mags = torch.autograd.grad((F.conv3d if nd == 3 else F.conv2d)(xa, wa, ba, padding=k // 2) + ra, [xa, ra, wa, ba], gy.double().abs())
    tol = 0 if k == 1 else 64 * 270 * 2.0 ** -24
    assert all(p.shape == q.shape and bool(((p.cpu().double() - q).abs() <= tol * m).all()) for p, q, m in zip(got, want, mags))


def test_a_map_without_extent_is_refused_as_by_any_convolution(cuda):
    conv, x, _, _ = int_layer(cuda, 3, 6, 10, 1, (0, 4, 4), 2, 3)
    for call in (lambda t: F.conv3d(t, conv.weight), lambda t: bs.conv_bias_act8(conv, t, None)):
        with pytest.raises(RuntimeError, match="[Kk]ernel size"):
            call(x.to(cuda))


def test_checkpoint8_of_a_single_value_without_axes(cuda):
    for v in (3.0, -0.75, 0.0):
        back = bs.checkpoint8(torch.tensor(v, device=cuda)).restore()
        assert back.shape == () and float(back) == v


def test_calls_are_counted_only_while_they_are(cuda):
    """_lib.count_calls sees these operators' entries, whatever was called before, and nothing of it stays"""
    x = torch.randn(64, device=cuda)
    bs.checkpoint8(x).restore()
    _lib.count_calls(True)
    try:
        bs.checkpoint8(x).restore()
        seen = dict(_lib.CALLS)
    finally:
        _lib.count_calls(False)
    bs.checkpoint8(x).restore()
    assert seen == {"mdt_act8_quantize": 1, "mdt_act8_restore": 1} == _lib.CALLS
