"""Block-scaled operators (utils/block_scaled.py) at their edges: layers whose passes run on several streams or inside a captured graph.

Layers are compared on small integers, where all products and sums are exact in fp32: equality."""
import copy

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from medicaldetectiontoolkit_amd.utils import block_scaled as bs
from medicaldetectiontoolkit_amd.utils import fused_epilogue as fe
from tests.test_block_scaled_models_gpu import int_layer

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
