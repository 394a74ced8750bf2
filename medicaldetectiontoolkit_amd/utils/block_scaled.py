"""Block-scaled numbers (csrc/block_scaled.hip, act8_backward.hip, mx4_linear.hip): activations kept for the backward pass in 8 bits, and products in
4 bits.

32 consecutive values share one power of two 2^e (scale byte e + 127), the smallest with which no value of the block is clipped:
max|x| <= Q * 2^e with Q = 255 for the outputs of a ReLU, 127 for signed values in 8 bits, 6 for the magnitudes 0, .5, 1, 1.5, 2, 3, 4, 6 of 4 bits.
Values are rounded to the nearest code, ties to the even one: a kept value is off by at most half a step of its block, max / 255 (ReLU), max / 127
(signed).  A positive ReLU output keeps at least the code 1 (below half a step it is off by less than a whole one), so the codes hold the ReLU's mask
exactly.  A block with an infinity or a NaN reads back as NaN.

  checkpoint8(x)                      -> Checkpoint8, .restore()      any float32 / bfloat16 / float16 tensor, 33 bytes for 32 values
  bias_act_checkpoint8(h, bias, res)  -> (y, Checkpoint8 of y)        the convolution epilogue of utils/fused_epilogue.bias_act that keeps the copy
  conv1x1_backward8(gy, w, x8, y8)    -> gradients of a 1x1(x1) layer from the kept copies of its input and its output
  conv_bias_act8(conv, x, x8, ...)    -> (y, y8)                      a convolution layer of the autograd graph that keeps x8 and y8 in place of x and y
  mx4_quantize(x) -> Mx4, .dequantize();  mx4_linear(x, w4, bias)     act(x W^T + bias) with both operands in 4 bits (inference)
  mx4_heads(net)                                                      a Mask R-CNN's box head on mx4_linear while the context lasts

What calls them: models/backbone.FPN with cf.act8_checkpoints (train.py --act8 1), predictor.predict_patient / predict_test_set with head_dtype="mx4".

Like every operator of this package they run on the GPU only and are queued on the current stream of the tensors' device; a tensor that was made on
another stream is the caller's to synchronise, as with any torch operator.  Their scratch memory comes from torch's allocator for each call, so
calls on several streams and captured graphs do not share any.  (The backbone around them keeps its fp32 layers, whose buffers belong to one stream.)"""
import contextlib
import math
import threading

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from .. import _lib
from . import fused_epilogue

BLOCK = 32
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _call(device, name, *args):
    """the C entry on `device`'s current stream"""
    fn = getattr(_lib.lib(), name)
    idx = device.index
    if idx == torch._C._cuda_getDevice():                       # (a tensor on the GPU exists: no lazy initialisation to ask for)
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(idx))
    else:
        with torch.cuda.device(idx):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(idx))
    if rc != 0:
        _lib.check(rc, name)


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _on_gpu(device, name):
    if device.type != "cuda":
        raise RuntimeError("%s must live on the GPU: the MI355X HIP path is the only implementation (no CPU fallback in the product path)" % name)


def _float_tensor(x, name):
    if x.dtype not in _DTYPES:
        raise TypeError("%s: float32, bfloat16 or float16, not %s" % (name, x.dtype))
    if not x.is_cuda:
        _lib.require_cuda(x, name)


def _same_device(ref, **tensors):
    for name, t in tensors.items():
        if t is not None and t.device != ref:
            raise ValueError("%s is on %s, the other operands on %s" % (name, t.device, ref))


def _no_graph(what, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError("%s records no autograd graph: call it under torch.no_grad()" % what)


def _rows_format(dim):
    return torch.channels_last_3d if dim == 5 else torch.channels_last if dim == 4 else torch.contiguous_format


def _dense(x):
    """x, or a row-major copy where its storage is neither row-major nor channels-last; and whether its channels (axis 1) are innermost"""
    if x.dim() in (4, 5) and x.is_contiguous(memory_format=_rows_format(x.dim())):
        return x, True
    if not x.is_contiguous():
        x = x.contiguous()
    return x, x.dim() == 2


def _empty(shape, channels_last, dtype, device):
    """a dense tensor, channels innermost or row-major (with 2 axes both are the same)"""
    if channels_last and len(shape) > 2:
        return torch.empty(shape, dtype=dtype, device=device, memory_format=_rows_format(len(shape)))
    return torch.empty(shape, dtype=dtype, device=device)


def _scales_at(n):
    """where the scales of n codes begin in a buffer that holds both"""
    return (n + 15) // 16 * 16


class Checkpoint8(object):
    """An activation kept in 8 bits: `codes` (uint8, one a value, storage order) and `scales` (uint8, one for 32 codes).  `channels_last`: axis 1 is the
    innermost of the storage (for two axes it always is).  What the operators make holds both in one allocation, `buffer`."""
    __slots__ = ("buffer", "_codes", "_scales", "shape", "relu", "dtype", "channels_last", "device")

    def __init__(self, codes, scales, shape, relu=False, dtype=torch.float32, channels_last=None):
        shape = tuple(int(s) for s in shape)
        n = math.prod(shape)
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or codes.numel() != n or scales.numel() != -(-n // BLOCK):
            raise ValueError("Checkpoint8: %d uint8 codes and %d uint8 scales for shape %s, got %d %s and %d %s"
                             % (n, -(-n // BLOCK), shape, codes.numel(), codes.dtype, scales.numel(), scales.dtype))
        if not codes.is_contiguous() or not scales.is_contiguous() or codes.data_ptr() % 4 != 0:
            raise ValueError("Checkpoint8: codes and scales are contiguous, the codes 4-byte aligned")
        if dtype not in _DTYPES:
            raise TypeError("Checkpoint8: float32, bfloat16 or float16, not %s" % dtype)
        if channels_last is None:
            channels_last = len(shape) == 2
        elif (channels_last and len(shape) not in (2, 4, 5)) or (len(shape) == 2 and not channels_last):
            raise ValueError("Checkpoint8: channels_last=%s does not describe %d axes" % (channels_last, len(shape)))
        if scales.device != codes.device:
            _same_device(codes.device, scales=scales)
        self._set(None, codes, scales, shape, bool(relu), dtype, bool(channels_last), codes.device)

    def _set(self, buffer, codes, scales, shape, relu, dtype, channels_last, device):
        self.buffer, self._codes, self._scales, self.shape, self.relu, self.dtype, self.channels_last, self.device = buffer, codes, scales, shape, relu, dtype, channels_last, device
        return self

    @classmethod
    def of_buffer(cls, buffer, shape, relu, dtype, channels_last):
        """codes and, from _scales_at(values) on, scales in one uint8 tensor"""
        return cls.__new__(cls)._set(buffer, None, None, shape, relu, dtype, channels_last, buffer.device)

    @property
    def codes(self):
        return self._codes if self.buffer is None else self.buffer[:math.prod(self.shape)]

    @property
    def scales(self):
        return self._scales if self.buffer is None else self.buffer[_scales_at(math.prod(self.shape)):]

    def pointers(self):
        """(codes, scales) as addresses"""
        if self.buffer is None:
            return self._codes.data_ptr(), self._scales.data_ptr()
        at = self.buffer.data_ptr()
        return at, at + _scales_at(math.prod(self.shape))

    def tensors(self):
        """what holds the copy, for Function.save_for_backward: of_tensors puts it together again"""
        return (self._codes, self._scales) if self.buffer is None else (self.buffer,)

    def meta(self):
        return self.shape, self.relu, self.dtype, self.channels_last

    @classmethod
    def of_tensors(cls, tensors, meta):
        if len(tensors) == 1:
            return cls.of_buffer(tensors[0], *meta)
        return cls.__new__(cls)._set(None, tensors[0], tensors[1], *meta, tensors[0].device)

    def restore(self):
        """the kept values, in the type, shape and storage order of the tensor they were taken from"""
        _on_gpu(self.device, "Checkpoint8")
        x = _empty(self.shape, self.channels_last, self.dtype, self.device)
        codes, scales = self.pointers()
        _call(self.device, "mdt_act8_restore", codes, scales, x.data_ptr(), x.numel(), _DTYPES[self.dtype], self.relu)
        return x


def checkpoint8(x, relu=False):
    """x's values in 8 bits.  relu=True: x is the output of a ReLU (values <= 0 read back as 0) and is kept with twice the resolution."""
    _float_tensor(x, "x")
    x, cl = _dense(x)
    n, device, dtype = x.numel(), x.device, x.dtype
    codes = _scales_at(n)
    buffer = torch.empty(codes + -(-n // BLOCK), dtype=torch.uint8, device=device)
    at = buffer.data_ptr()
    _call(device, "mdt_act8_quantize", x.data_ptr(), at, at + codes, n, _DTYPES[dtype], bool(relu))
    return Checkpoint8.of_buffer(buffer, tuple(x.shape), bool(relu), dtype, cl)


def bias_act_checkpoint8(h, bias, residual=None, relu=True, inplace=False):
    """(y, Checkpoint8 of y), y = act(h + bias[c] (+ residual)): fused_epilogue.bias_act (the same roundings) with y's 8-bit copy from the same pass.
    h: float32 [N, C, ...], row-major or channels-last; inplace: y overwrites h."""
    _float_tensor(h, "h")
    if h.dtype != torch.float32 or bias.dtype != torch.float32 or (residual is not None and residual.dtype != torch.float32):
        raise TypeError("bias_act_checkpoint8: float32 operands")
    shape, device = h.shape, h.device
    if len(shape) < 2 or bias.dim() != 1 or bias.shape[0] != shape[1] or (residual is not None and residual.shape != shape):
        raise ValueError("bias_act_checkpoint8: bias %s and residual %s do not fit h %s" % (tuple(bias.shape), None if residual is None else tuple(residual.shape), tuple(shape)))
    if bias.device != device or (residual is not None and residual.device != device):
        _same_device(device, bias=bias, residual=residual)
    if torch.is_grad_enabled():
        _no_graph("bias_act_checkpoint8", h, bias, residual)
    x, cl = _dense(h)
    if inplace and x is not h:
        raise ValueError("bias_act_checkpoint8: inplace needs a dense row-major or channels-last h")
    inner = 1 if cl else math.prod(shape[2:])
    if residual is not None and residual.stride() != x.stride():
        residual = residual.contiguous(memory_format=_rows_format(x.dim()) if cl else torch.contiguous_format)
    if not bias.is_contiguous():
        bias = bias.contiguous()
    y = x if inplace else torch.empty_like(x)
    n = x.numel()
    codes = _scales_at(n)
    buffer = torch.empty(codes + -(-n // BLOCK), dtype=torch.uint8, device=device)
    if n:
        at = buffer.data_ptr()
        _call(device, "mdt_bias_act_act8_forward", y.data_ptr(), x.data_ptr(), bias.data_ptr(), _ptr(residual), at, at + codes, n, shape[1], inner, bool(relu))
    return y, Checkpoint8.of_buffer(buffer, tuple(shape), bool(relu), x.dtype, cl)


def conv1x1_backward8(gy, w, x8, y8=None, need_g=False, need_gx=True, need_gw=True):
    """(gx, gw, gbias, g) of y = act(conv1x1(x, w) + bias (+ residual)) at unit stride, from the 8-bit copies of x and y.

    gy: float32 [V, C_out] or [N, C_out, ...]; w: float32 [C_out, C_in(, 1, 1(, 1))]; x8: the kept input, channels innermost; y8: the kept ReLU output
    (None: no activation).  g = gy * (y > 0) is the residual's gradient (None unless need_g); gx comes in x's shape and storage order."""
    if gy.dtype != torch.float32 or w.dtype != torch.float32:
        raise TypeError("conv1x1_backward8: float32 gradients and weights")
    _lib.require_cuda(gy, "gy")
    w_shape = tuple(w.shape)
    if len(w_shape) < 2 or math.prod(w_shape[2:]) != 1 or 0 in w_shape:
        raise ValueError("conv1x1_backward8: a 1x1(x1) filter, not %s" % (w_shape,))
    co, ci = w_shape[:2]
    shape = tuple(gy.shape)
    if gy.dim() not in (2, 4, 5) or shape[1] != co or x8.shape != shape[:1] + (ci,) + shape[2:]:
        raise ValueError("conv1x1_backward8: gy %s, w %s and x8 %s do not belong together" % (shape, tuple(w.shape), x8.shape))
    if not x8.channels_last or (y8 is not None and not y8.channels_last):
        raise ValueError("conv1x1_backward8: the kept maps have their channels innermost")
    if y8 is not None and (y8.shape != shape or not y8.relu):
        raise ValueError("conv1x1_backward8: y8 is the kept ReLU output of gy's shape")
    dev = gy.device
    if w.device != dev or x8.device != dev or (y8 is not None and y8.device != dev):
        _same_device(dev, w=w, x8=x8, y8=y8)
    mf = _rows_format(len(shape))
    if not gy.is_contiguous(memory_format=mf):
        gy = gy.contiguous(memory_format=mf)
    if w.stride()[:2] != (ci, 1):
        w = w.detach().reshape(co, ci).contiguous()
    V = gy.numel() // co
    gx = _empty(x8.shape, True, torch.float32, dev) if need_gx else None
    gw = torch.empty(w_shape, dtype=torch.float32, device=dev) if need_gw else None
    gbias = torch.empty(co, dtype=torch.float32, device=dev)
    write_g = need_g and y8 is not None
    g = torch.empty_like(gy) if write_g else None
    ws = torch.empty(_lib.lib().mdt_conv1x1_act8_backward_workspace_bytes(V, ci, co), dtype=torch.uint8, device=dev)
    _call(dev, "mdt_conv1x1_act8_backward", gy.data_ptr(), w.data_ptr(), *x8.pointers(), int(x8.relu), y8.pointers()[0] if y8 is not None else None,
          _ptr(gx), _ptr(gw), gbias.data_ptr(), _ptr(g), V, ci, co, ws.data_ptr(), ws.numel())
    return gx, gw, gbias, (g if write_g else gy if need_g else None)


def act_backward8(gy, y8=None):
    """(g, gbias) of act(h + bias) from the kept output: g = gy * (y > 0) (y8 None, no activation: gy), gbias = the sum of g over everything but axis 1.
    gy: float32, in any storage order; g has its channels innermost."""
    if gy.dtype != torch.float32:
        raise TypeError("act_backward8: float32 gradients")
    _lib.require_cuda(gy, "gy")
    shape, dev = tuple(gy.shape), gy.device
    if len(shape) not in (2, 4, 5) or shape[1] == 0 or (y8 is not None and (y8.shape != shape or not y8.relu or not y8.channels_last)):
        raise ValueError("act_backward8: gy %s has 2, 4 or 5 axes, y8 is the kept ReLU output of its shape, channels innermost" % (shape,))
    _same_device(dev, y8=y8)
    mf = _rows_format(len(shape))
    if not gy.is_contiguous(memory_format=mf):
        gy = gy.contiguous(memory_format=mf)
    V = gy.numel() // shape[1]
    g = torch.empty_like(gy) if y8 is not None else None
    gbias = torch.empty(shape[1], dtype=torch.float32, device=dev)
    ws = torch.empty(_lib.lib().mdt_conv1x1_act8_backward_workspace_bytes(V, 1, shape[1]), dtype=torch.uint8, device=dev)
    _call(dev, "mdt_conv1x1_act8_backward", gy.data_ptr(), None, None, None, 0, y8.pointers()[0] if y8 is not None else None, None, None, gbias.data_ptr(), _ptr(g), V, 1, shape[1],
          ws.data_ptr(), ws.numel())
    return (g if y8 is not None else gy), gbias


class _ConvBiasAct8(Function):
    """y = act(conv(x) + bias (+ residual)) whose backward pass finds x and y in 8 bits: a quarter of the memory that autograd would hold from the forward pass to the
    backward pass.  The forward values are those of the fp32 layer; the ReLU's mask, the input gradient and the bias gradient are exact, the weight
    gradient is taken with the kept x."""

    @staticmethod
    def forward(ctx, x, w, bias, residual, x8, relu, keep, padding):
        nd = w.dim() - 2
        mf = _rows_format(x.dim())
        if residual is not None and not residual.is_contiguous(memory_format=mf):
            residual = residual.contiguous(memory_format=mf)
        one = math.prod(w.shape[2:]) == 1
        bias = bias.detach().contiguous()
        y = y8 = None
        if one and fused_epilogue.ENABLED and fused_epilogue.CONV1X1_FWD and x.numel() >= (1 << 20) and x.data_ptr() % 16 == 0 and w.stride()[:2] == (w.shape[1], 1) and _lib.lib().mdt_conv1x1_forward_supported(int(w.shape[1]), int(w.shape[0])):
            y = fused_epilogue._conv1x1_forward(x, w, bias, residual, relu)
        elif nd == 3 and residual is None and padding == (1, 1, 1) and not x.is_contiguous():
            y = fused_epilogue.conv3x3x3_small(x, w, bias, relu)
        if y is None:
            h = (F.conv3d if nd == 3 else F.conv2d)(x, w, None, 1, padding)
            if not h.is_contiguous(memory_format=mf):
                h = h.contiguous(memory_format=mf)
            if relu or keep:
                y, y8 = bias_act_checkpoint8(h, bias, residual, relu=relu, inplace=True)
            else:
                y = fused_epilogue.bias_act(h, bias, residual, False)
        elif relu or keep:
            y8 = checkpoint8(y, relu=relu)
        kept = x8.tensors()
        ctx.x8, ctx.n_x8, ctx.y8 = x8.meta(), len(kept), y8.meta() if relu else None
        ctx.save_for_backward(w, *kept, *(y8.tensors() if relu else ()))
        ctx.has_res, ctx.padding, ctx.one = residual is not None, padding, one
        return y, y8

    @staticmethod
    @once_differentiable
    def backward(ctx, gy, _gy8):
        w, kept = ctx.saved_tensors[0], ctx.saved_tensors[1:]
        x8 = Checkpoint8.of_tensors(kept[:ctx.n_x8], ctx.x8)
        y8 = Checkpoint8.of_tensors(kept[ctx.n_x8:], ctx.y8) if ctx.y8 is not None else None
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        if ctx.one:
            gx, gw, gbias, g = conv1x1_backward8(gy, w, x8, y8, need_g=ctx.has_res and need_r, need_gx=need_x, need_gw=need_w)
        else:
            g, gbias = act_backward8(gy, y8)
            # w.detach(): the filter is flipped for this call; the buffers that the fp32 layers share belong to one stream
            gx, gw = fused_epilogue._stride1_grads(x8.restore() if need_w else _like(x8), w.detach(), ctx.padding, g, need_x, need_w)
        return gx, gw, (gbias if need_b else None), (g if ctx.has_res and need_r else None), None, None, None, None


def _like(x8):
    """an uninitialised tensor of the kept map's shape and storage order, where only those are asked for"""
    return _empty(x8.shape, x8.channels_last, x8.dtype, x8.device)


def conv_bias_act8(conv, x, x8=None, residual=None, relu=False, keep=True, subsampled=False):
    """(y, y8) for y = act(conv(x) + bias (+ residual)) of a size-preserving convolution module (unit stride; subsampled=True: a strided 1x1 layer whose
    input was sub-sampled already): the autograd node keeps x8, x's 8-bit copy (None: one is made), and y's in place of x and y.  y8 is what the next
    layer takes as its x8; keep=False: there is none (an output that no further layer of this kind reads; None where there is no activation either).
    float32 maps on the GPU; a row-major x is copied to channels-last."""
    if not isinstance(conv, (nn.Conv2d, nn.Conv3d)):
        raise ValueError("conv_bias_act8: a Conv2d or Conv3d, not %s" % type(conv).__name__)
    for name, ok in (("a bias", conv.bias is not None), ("one group", conv.groups == 1), ("unit dilation", all(int(v) == 1 for v in conv.dilation)),
                     ("zero padding", conv.padding_mode == "zeros" and not isinstance(conv.padding, str)),
                     ("a size-preserving window", not isinstance(conv.padding, str) and all(2 * int(p) + 1 == int(k) for p, k in zip(conv.padding, conv.kernel_size))),
                     ("unit stride", all(int(v) == 1 for v in conv.stride) or (subsampled and all(int(k) == 1 for k in conv.kernel_size)))):
        if not ok:
            raise ValueError("conv_bias_act8: a convolution with %s" % name)
    _float_tensor(x, "x")
    if x.dtype != torch.float32 or conv.weight.dtype != torch.float32 or conv.bias.dtype != torch.float32 or torch.is_autocast_enabled():
        raise TypeError("conv_bias_act8: float32 training, not under autocast")
    if x.dim() != conv.weight.dim() or int(x.shape[1]) != int(conv.weight.shape[1]):
        raise ValueError("conv_bias_act8: x %s does not fit the filter %s" % (tuple(x.shape), tuple(conv.weight.shape)))
    shape = (x.shape[0], conv.weight.shape[0]) + tuple(x.shape[2:])
    if residual is not None and (tuple(residual.shape) != tuple(shape) or residual.dtype != torch.float32):
        raise ValueError("conv_bias_act8: residual %s, output %s" % (tuple(residual.shape), tuple(shape)))
    _same_device(x.device, weight=conv.weight, bias=conv.bias, residual=residual, x8=x8)
    if x.device.index != torch.cuda.current_device():
        raise RuntimeError("conv_bias_act8: x is not on the current device (one process per GPU)")
    mf = _rows_format(x.dim())
    if not x.is_contiguous(memory_format=mf):
        x = x.contiguous(memory_format=mf)
    if x8 is None:
        x8 = checkpoint8(x)
    if x8.shape != tuple(x.shape) or not x8.channels_last or x8.dtype != torch.float32:
        raise ValueError("conv_bias_act8: x8 is x's copy, channels innermost: %s for x %s" % (x8.shape, tuple(x.shape)))
    return _ConvBiasAct8.apply(x, conv.weight, conv.bias, residual, x8, bool(relu), bool(keep), tuple(int(p) for p in conv.padding))


class Mx4(object):
    """Rows in 4 bits: `codes` uint8 [..., ceil(k / 32) * 16] (two a byte, the even value in the low half), `scales` uint8 [..., ceil(k / 32)]; blocks run along
    the last axis of length k.  `shape`: the values' shape.  What mx4_quantize makes holds both in one allocation, `buffer`."""
    __slots__ = ("buffer", "_codes", "_scales", "shape", "k", "dtype", "device")

    def __init__(self, codes, scales, k, dtype=torch.float32):
        k = int(k)
        kb = -(-k // BLOCK)
        rows = tuple(codes.shape[:-1])
        if k < 1 or codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or codes.dim() < 1 or codes.shape[-1] != 16 * kb or tuple(scales.shape) != rows + (kb,):
            raise ValueError("Mx4: uint8 codes [..., %d] and scales [..., %d] for rows of %d, got %s %s and %s %s"
                             % (16 * kb, kb, k, tuple(codes.shape), codes.dtype, tuple(scales.shape), scales.dtype))
        if not codes.is_contiguous() or not scales.is_contiguous() or codes.data_ptr() % 16 != 0:
            raise ValueError("Mx4: codes and scales are contiguous, the codes 16-byte aligned")
        if dtype not in _DTYPES:
            raise TypeError("Mx4: float32, bfloat16 or float16, not %s" % dtype)
        if scales.device != codes.device:
            _same_device(codes.device, scales=scales)
        self.buffer, self._codes, self._scales, self.shape, self.k, self.dtype, self.device = None, codes, scales, rows + (k,), k, dtype, codes.device

    @classmethod
    def of_buffer(cls, buffer, shape, dtype):
        """codes, then scales, in one uint8 tensor"""
        m = cls.__new__(cls)
        m.buffer, m._codes, m._scales, m.shape, m.k, m.dtype, m.device = buffer, None, None, shape, shape[-1], dtype, buffer.device
        return m

    def _bytes(self):
        kb = -(-self.k // BLOCK)
        return math.prod(self.shape[:-1]) * kb * 16, kb

    @property
    def codes(self):
        if self.buffer is None:
            return self._codes
        n, kb = self._bytes()
        return self.buffer[:n].view(self.shape[:-1] + (16 * kb,))

    @property
    def scales(self):
        if self.buffer is None:
            return self._scales
        n, kb = self._bytes()
        return self.buffer[n:].view(self.shape[:-1] + (kb,))

    def pointers(self):
        """(codes, scales) as addresses"""
        if self.buffer is None:
            return self._codes.data_ptr(), self._scales.data_ptr()
        at = self.buffer.data_ptr()
        return at, at + self._bytes()[0]

    def dequantize(self):
        """the values the codes stand for, in the type of the tensor they were taken from"""
        _on_gpu(self.device, "Mx4")
        x = torch.empty(self.shape, dtype=self.dtype, device=self.device)
        codes, scales = self.pointers()
        _call(self.device, "mdt_mx4_dequantize", codes, scales, x.data_ptr(), x.numel() // self.k, self.k, _DTYPES[self.dtype])
        return x


def mx4_quantize(x):
    """x's rows (last axis) in 4 bits"""
    _float_tensor(x, "x")
    shape = tuple(x.shape)
    if not shape or shape[-1] < 1:
        raise ValueError("mx4_quantize: rows of at least one value, not %s" % (shape,))
    if not x.is_contiguous():
        x = x.detach().contiguous()
    k, device = shape[-1], x.device
    rows = x.numel() // k
    n = rows * -(-k // BLOCK)
    buffer = torch.empty(17 * n, dtype=torch.uint8, device=device)
    at = buffer.data_ptr()
    _call(device, "mdt_mx4_quantize", x.data_ptr(), at, at + 16 * n, rows, k, _DTYPES[x.dtype])
    return Mx4.of_buffer(buffer, shape, x.dtype)


def mx4_linear(x, w4, bias=None, relu=False):
    """act(x W^T + bias) in x's type: x [..., K] (float32, bfloat16 or float16) is rounded to 4 bits in the call, w4 = mx4_quantize(W) for W [N, K]; products and
    sums in float32.  bias: [N], taken in float32.  For inference: no autograd graph."""
    _float_tensor(x, "x")
    shape, device = x.shape, x.device
    if len(w4.shape) != 2 or not shape or shape[-1] != w4.k or (bias is not None and (bias.dim() != 1 or bias.shape[0] != w4.shape[0])):
        raise ValueError("mx4_linear: x %s, W %s and bias %s do not fit" % (tuple(shape), w4.shape, None if bias is None else tuple(bias.shape)))
    if w4.device != device or (bias is not None and bias.device != device):
        _same_device(device, w4=w4, bias=bias)
    if x.requires_grad or (bias is not None and bias.requires_grad):
        _no_graph("mx4_linear", x, bias)
    n, k = w4.shape
    if not x.is_contiguous():
        x = x.contiguous()
    if bias is not None and (bias.dtype != torch.float32 or not bias.is_contiguous()):
        bias = bias.float().contiguous()
    rows = x.numel() // k
    y = torch.empty(shape[:-1] + (n,), dtype=x.dtype, device=device)
    if y.numel() == 0:
        return y
    need = _lib.lib().mdt_mx4_linear_workspace_bytes(rows, k, n)
    ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    codes, scales = w4.pointers()
    _call(device, "mdt_mx4_linear", x.data_ptr(), _DTYPES[x.dtype], codes, scales, _ptr(bias), y.data_ptr(), rows, k, n, int(relu), _ptr(ws), need)
    return y


_HEADS = threading.Lock()       # a head is looked at and taken in one step


@contextlib.contextmanager
def mx4_heads(net):
    """A Mask R-CNN's box head (the two products of every region, `classifier.conv1` and `conv2`) in 4 bits while the context lasts: the filters are rounded when it is
    entered, so load a checkpoint before, and not inside.  It holds for every call of the net while it lasts; a second one at the same time (nested, or of another thread)
    raises.  Inference only: a training step inside raises."""
    head = getattr(net, "classifier", None)
    if head is None or not hasattr(head, "mx4"):
        raise ValueError("mx4_heads: a net with a box head (Mask R-CNN), not %s" % type(net).__name__)
    if not (isinstance(head.conv1, fused_epilogue.ConvBiasReLU) and isinstance(head.conv2, fused_epilogue.ConvBiasReLU)
            and tuple(head.conv1[0].kernel_size) == tuple(head.pool_size) and not any(head.conv1[0].padding)):
        raise ValueError("mx4_heads: the box head's layers are convolution + ReLU without a norm, the first as large as the pooled region")
    with _HEADS:
        if head.mx4 is not None:
            raise RuntimeError("mx4_heads: the net's head is in 4 bits already")
        head.mx4 = tuple(mx4_quantize(c[0].weight.detach().flatten(1)) for c in (head.conv1, head.conv2))
    try:
        yield net
    finally:
        head.mx4 = None
