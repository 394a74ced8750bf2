"""Cases of the block-scaled operators (utils/block_scaled.py): activations kept for the backward pass in 8 bits, and products in 4 bits.

Both formats cut a tensor into blocks of 32 values that share one power of two.  For a block with the largest magnitude m the
shared exponent e is the smallest for which no value is clipped, m <= Q * 2^e (Q = 255 for the outputs of a ReLU, 127 for signed
values in 8 bits, 6 for the eight magnitudes 0, .5, 1, 1.5, 2, 3, 4, 6 of 4 bits), and each value is rounded to the nearest
code, ties to the even one.  A positive output of a ReLU keeps at least the code 1, so the codes hold the ReLU's mask exactly.

  save      y = act(h + bias (+ residual)) and y's 8-bit copy in one pass, and the copy read back (what a training step does with it)
  keep      any tensor into 8 bits and back
  backward  a 1x1(x1) convolution's backward pass from the 8-bit copies of its input and of its output
  pack      rows into 4 bits and back
  linear    act(x W^T + bias) with x rounded to 4 bits in the call and W kept in 4 bits
"""
import math

import torch

own = False

BLOCK = 32
Q4 = 6.0


# ---- the cases --------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the deepest map of a small patch: what one launch costs
        {"name": "save small map", "op": "save", "batch": 2, "channels": 18, "y": 8, "x": 8, "z": 16, "residual": True, "relu": True, "layout": "cl"},
        # the residual output of the first stage's blocks, 8 patches of 128^3
        {"name": "save C2 output", "op": "save", "batch": 8, "channels": 72, "y": 32, "x": 32, "z": 128, "residual": True, "relu": True, "layout": "cl"},
        # a 2D map in bf16, signed, odd extents, row-major
        {"name": "keep odd 2D bf16", "op": "keep", "batch": 5, "channels": 49, "y": 143, "x": 141, "z": 0, "relu": False, "layout": "rows", "dtype": "bfloat16"},
        # a bottleneck's last layer on a ragged little map
        {"name": "backward ragged small", "op": "backward", "voxels": 693, "cin": 18, "cout": 72, "relu": True, "residual": True},
        # the same layer on the first stage's maps: 8 x 32 x 32 x 128 voxels
        {"name": "backward C2 expand", "op": "backward", "voxels": 1048576, "cin": 18, "cout": 72, "relu": True, "residual": True},
        # the bottleneck's first layer there
        {"name": "backward C2 reduce", "op": "backward", "voxels": 1048576, "cin": 72, "cout": 18, "relu": True, "residual": False},
        # a 2D backbone's deepest stage: 20 maps of 9 x 9 with many channels
        {"name": "backward 2D C5", "op": "backward", "voxels": 1620, "cin": 1536, "cout": 384, "relu": True, "residual": False},
        # the 3D box head's filters, laid out once per checkpoint: K is no multiple of the block
        {"name": "pack 3D head filters", "op": "pack", "rows": 144, "k": 5292, "dtype": "float32"},
        # the 2D box head's pooled regions
        {"name": "pack 2D regions", "op": "pack", "rows": 10000, "k": 9408, "dtype": "bfloat16"},
        # one region through the 3D box head: latency
        {"name": "linear one region", "op": "linear", "rows": 1, "k": 5292, "n": 144, "relu": True, "dtype": "float32"},
        # the regions of 8 patches, 500 each
        {"name": "linear 3D head", "op": "linear", "rows": 4000, "k": 5292, "n": 144, "relu": True, "dtype": "float32"},
        # the regions of 20 slices through the 2D box head, under autocast
        {"name": "linear 2D head bf16", "op": "linear", "rows": 10000, "k": 9408, "n": 768, "relu": True, "dtype": "bfloat16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["save", "save", "keep", "backward", "backward", "backward", "pack", "linear", "linear", "linear"])
    if op in ("save", "keep"):
        n = _log(rng, 2e4, 7e7)                                   # elements, then split over the extents
        c = _log(rng, 3, 400)
        d3 = rng.random() < 0.6
        v = max(4, n // c)
        b = rng.randint(1, min(8, v))
        side = max(1, int((v / b) ** (1 / 3 if d3 else 0.5)))
        y = max(1, int(side * rng.uniform(0.6, 1.4)))
        x = max(1, int(side * rng.uniform(0.6, 1.4)))
        z = max(1, v // (b * y * x)) if d3 else 0
        case = {"op": op, "batch": b, "channels": c, "y": y, "x": x, "z": z, "relu": rng.random() < 0.7, "layout": "cl" if rng.random() < 0.75 else "rows"}
        if op == "save":
            return dict(case, residual=rng.random() < 0.5)
        return dict(case, dtype=rng.choice(["float32", "bfloat16", "float16"]))
    if op == "backward":
        ci, co = _log(rng, 3, 1000), _log(rng, 3, 1000)
        most = min(1000000, 94e6 / (ci + co), 1.3e9 / (ci * co))
        v = _log(rng, 100, most)
        relu = rng.random() < 0.75
        return {"op": op, "voxels": v, "cin": ci, "cout": co, "relu": relu, "residual": relu and rng.random() < 0.5}
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    k = _log(rng, 24, 9400)
    if op == "pack":
        return {"op": op, "rows": _log(rng, 1, min(10000, 9e7 / k)), "k": k, "dtype": dtype}
    return {"op": op, "rows": _log(rng, 1, 9000), "k": k, "n": _log(rng, 3, 768), "relu": rng.random() < 0.5, "dtype": dtype}


def _shape(case):
    sp = [case["y"], case["x"]] + ([case["z"]] if case["z"] else [])
    return [case["batch"], case["channels"]] + sp


def work(case):
    op = case["op"]
    if op in ("save", "keep"):
        n = math.prod(_shape(case))
        code = n + -(-n // BLOCK)
        if op == "save":
            return {"bytes": 4 * n * (3 + (1 if case["residual"] else 0)) + 2 * code, "flops": 8 * n}
        return {"bytes": 2 * n * (4 if case["dtype"] == "float32" else 2) + 2 * code, "flops": 8 * n}
    if op == "backward":
        v, ci, co = case["voxels"], case["cin"], case["cout"]
        b = 4 * v * co + 4 * v * ci + v * ci * 33 / 32 + (v * co * 33 / 32 if case["relu"] else 0) + (4 * v * co if case["residual"] else 0) + 8 * co * ci + 4 * co
        return {"bytes": b, "flops": 4 * v * ci * co + v * co}
    size = 4 if case["dtype"] == "float32" else 2
    r, k = case["rows"], case["k"]
    packed = -(-k // BLOCK) * 17
    if op == "pack":
        return {"bytes": 2 * r * k * size + 2 * r * packed, "flops": 8 * r * k}
    n = case["n"]
    return {"bytes": r * k * size + n * packed + 4 * n + r * n * size, "flops": 2 * r * k * n}


# ---- the formats, in elementary operations ------------------------------------------------------------------------------------
def _exponent(m, q):
    """smallest e with m <= q * 2^e, at least -127: m = f * 2^k with f in [.5, 1)"""
    f, k = torch.frexp(m)
    fq, kq = math.frexp(q)
    e = k - kq + (f > fq).to(k.dtype)
    return torch.where(m > 0, e, torch.full_like(e, -127)).clamp(min=-127)


def _blocks(flat):
    pad = -flat.shape[-1] % BLOCK
    return torch.nn.functional.pad(flat, (0, pad)).unflatten(-1, (-1, BLOCK))


def _quantize8(flat, relu):
    """codes (integers as float32) and exponents of a flat float32 tensor"""
    x = _blocks(flat)
    m = x.clamp(min=0).amax(-1) if relu else x.abs().amax(-1)
    e = _exponent(m, 255.0 if relu else 127.0)
    q = torch.round(x * torch.exp2(-e.float())[:, None])
    if relu:
        q = torch.maximum(q, (x > 0).float())
    return q, e


def _values8(q, e, n):
    return (q * torch.exp2(e.float())[:, None]).reshape(-1)[:n]


def _round4(a):
    """to the nearest of the eight magnitudes, ties to the even code"""
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return torch.round(a / step) * step


def _quantize4(x):
    """magnitudes with their signs (float32) in blocks, and exponents, of float32 rows [r, k]"""
    x = _blocks(x)
    e = _exponent(x.abs().amax(-1), Q4)
    v = x * torch.exp2(-e.float())[..., None]
    return torch.sign(v) * _round4(v.abs()), e


def _values4(q, e, k):
    return (q * torch.exp2(e.float())[..., None]).flatten(-2)[..., :k]


_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _pack4(q, e):
    """[r, blocks, 32] magnitudes -> bytes [r, 16 * blocks] (the even value in the low half) and scales [r, blocks]"""
    grid = torch.tensor(_GRID, device=q.device)
    code = torch.bucketize(q.abs(), grid).to(torch.uint8) + 8 * (q < 0).to(torch.uint8)
    return (code[..., 0::2] | (code[..., 1::2] << 4)).flatten(-2).contiguous(), (e + 127).to(torch.uint8)


def _unpack4(codes, scales, k):
    grid = torch.tensor(_GRID + tuple(-g for g in _GRID), device=codes.device)
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).unflatten(-1, (-1, BLOCK)).int()
    return _values4(grid[c], scales.int() - 127, k)


# ---- inputs ---------------------------------------------------------------------------------------------------------------------
def _dense(t, layout):
    if layout == "rows":
        return t.contiguous()
    return t.contiguous(memory_format=torch.channels_last_3d if t.dim() == 5 else torch.channels_last)


def _activation(gen, shape, dim):
    """pre-activations: each channel with its own spread and offset"""
    c = shape[dim]
    view = [1] * len(shape)
    view[dim] = c
    spread = torch.exp(torch.randn(c, generator=gen, device="cuda") * 0.7).view(view)
    off = (torch.randn(c, generator=gen, device="cuda") * 0.3).view(view)
    return torch.randn(shape, generator=gen, device="cuda") * spread + off


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    op = case["op"]
    s = {"case": case}
    if op in ("save", "keep"):
        shape = _shape(case)
        h = _activation(gen, shape, 1)
        if op == "keep":
            h = h.relu_() if case["relu"] else h
            s["x"] = _dense(h.to(getattr(torch, case["dtype"])), case["layout"])
            return s
        s["h"] = _dense(h, case["layout"])
        s["bias"] = torch.randn(shape[1], generator=gen, device="cuda") * 0.5
        s["residual"] = _dense(torch.randn(shape, generator=gen, device="cuda").relu_(), case["layout"]) if case["residual"] else None
        return s
    if op == "backward":
        v, ci, co = case["voxels"], case["cin"], case["cout"]
        x = _activation(gen, [v, ci], 1).relu_()
        q, e = _quantize8(x.reshape(-1), True)
        s["x_codes"], s["x_scales"] = q.reshape(-1)[:v * ci].to(torch.uint8), (e + 127).to(torch.uint8)
        if case["relu"]:
            q, e = _quantize8(_activation(gen, [v, co], 1).relu_().reshape(-1), True)
            s["y_codes"], s["y_scales"] = q.reshape(-1)[:v * co].to(torch.uint8), (e + 127).to(torch.uint8)
        s["w"] = torch.randn(co, ci, generator=gen, device="cuda") / math.sqrt(ci)
        # gradients: small, and of very different size from voxel to voxel
        s["gy"] = torch.randn(v, co, generator=gen, device="cuda") * torch.exp(torch.randn(v, 1, generator=gen, device="cuda") * 1.5 - 7)
        return s
    dtype = getattr(torch, case["dtype"])
    s["x"] = _activation(gen, [case["rows"], case["k"]], 1).to(dtype)
    if op == "linear":
        w = torch.randn(case["n"], case["k"], generator=gen, device="cuda") / math.sqrt(case["k"])
        s["w_codes"], s["w_scales"] = _pack4(*_quantize4(w))
        s["bias"] = torch.randn(case["n"], generator=gen, device="cuda") * 0.1
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------------------
def _in_memory_order(t, layout):
    return t if layout == "rows" else t.movedim(1, -1)


def _read8(codes, scales, shape):
    n = math.prod(shape)
    return _values8(_blocks(codes.float()), scales.int() - 127, n).view(shape)


def run(s):
    if own:
        return _run_own(s)
    case, op = s["case"], s["case"]["op"]
    if op in ("save", "keep"):
        if op == "save":
            b = s["bias"].view([1, -1] + [1] * (s["h"].dim() - 2))
            y = s["h"] + b
            if s["residual"] is not None:
                y = y + s["residual"]
            y = y.clamp(min=0) if case["relu"] else y
        else:
            y = s["x"]
        m = _in_memory_order(y, case["layout"])
        kept = _values8(*_quantize8(m.float().reshape(-1), case["relu"]), m.numel()).view(m.shape).to(y.dtype)
        kept = kept if case["layout"] == "rows" else kept.movedim(-1, 1)
        return {"y": y, "kept": kept} if op == "save" else {"kept": kept}
    if op == "backward":
        g = s["gy"]
        if case["relu"]:
            g = g * (s["y_codes"].view(g.shape) > 0)
        x = _read8(s["x_codes"], s["x_scales"], [case["voxels"], case["cin"]])
        out = {"gx": g @ s["w"], "gw": g.t() @ x, "gbias": g.sum(0)}
        return dict(out, g=g) if case["residual"] else out
    x = _values4(*_quantize4(s["x"].float()), case["k"])
    if op == "pack":
        return x.to(s["x"].dtype)
    y = x @ _unpack4(s["w_codes"], s["w_scales"], case["k"]).t() + s["bias"]
    return (y.clamp(min=0) if case["relu"] else y).to(s["x"].dtype)


def _run_own(s):
    from medicaldetectiontoolkit_amd.utils import block_scaled as bs
    case, op = s["case"], s["case"]["op"]
    if op == "save":
        y, kept = bs.bias_act_checkpoint8(s["h"], s["bias"], s["residual"], relu=case["relu"])
        return {"y": y, "kept": kept.restore()}
    if op == "keep":
        return {"kept": bs.checkpoint8(s["x"], relu=case["relu"]).restore()}
    if op == "backward":
        v = case["voxels"]
        x = bs.Checkpoint8(s["x_codes"], s["x_scales"], (v, case["cin"]), relu=True)
        y = bs.Checkpoint8(s["y_codes"], s["y_scales"], (v, case["cout"]), relu=True) if case["relu"] else None
        gx, gw, gbias, g = bs.conv1x1_backward8(s["gy"], s["w"], x, y, need_g=case["residual"])
        out = {"gx": gx, "gw": gw, "gbias": gbias}
        return dict(out, g=g) if case["residual"] else out
    if op == "pack":
        return bs.mx4_quantize(s["x"]).dequantize()
    return bs.mx4_linear(s["x"], bs.Mx4(s["w_codes"], s["w_scales"], case["k"]), s["bias"], relu=case["relu"])


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------------------
def _shared(m, q):
    """2^e for the smallest e >= -127 with m <= q * 2^e, found by trying the two exponents around log2(m / q)"""
    e = torch.ceil(torch.log2(m.clamp(min=1e-300) / q)).clamp(min=-127)
    e = torch.where(q * torch.exp2(e) < m, e + 1, e)
    return torch.exp2(torch.where((q * torch.exp2(e - 1) >= m) & (e > -127), e - 1, e))


def _kept64(x, relu):
    n = x.numel()
    x = torch.cat([x.reshape(-1), x.new_zeros(-n % BLOCK)]).view(-1, BLOCK)
    s = _shared((x if relu else x.abs()).amax(1, keepdim=True).clamp(min=0), 255.0 if relu else 127.0)
    t = x / s
    low = torch.floor(t)
    d = t - low
    odd = torch.remainder(low, 2) == 1
    q = low + ((d > 0.5) | ((d == 0.5) & odd)).double()
    if relu:
        q = torch.where(x > 0, torch.where(q < 1, 1.0, q), 0.0)
    return (q * s).reshape(-1)[:n]


def _four64(x):
    k = x.shape[1]
    x = torch.cat([x, x.new_zeros(x.shape[0], -k % BLOCK)], 1).view(x.shape[0], -1, BLOCK)
    s = _shared(x.abs().amax(2, keepdim=True), Q4)
    a = x.abs() / s
    # borders between neighbours; the one below takes a tie where its code is even
    q = torch.zeros_like(a)
    for code in range(1, 8):
        border = (_GRID[code - 1] + _GRID[code]) / 2
        up = a >= border if code % 2 == 0 else a > border
        q = torch.where(up, torch.full_like(q, _GRID[code]), q)
    return (torch.where(x < 0, -q, q) * s).flatten(1)[:, :k]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("save", "keep"):
        if op == "save":
            # the sums are defined with a rounding to float32 after each
            c = s["bias"].double().view([1, -1] + [1] * (s["h"].dim() - 2))
            y = (s["h"].double() + c).float().double()
            if s["residual"] is not None:
                y = (y + s["residual"].double()).float().double()
            if case["relu"]:
                y = torch.where(y > 0, y, torch.zeros_like(y))
        else:
            y = s["x"].double()
        if case["layout"] == "rows":
            kept = _kept64(y, case["relu"]).view(y.shape)
        else:
            t = y.movedim(1, -1)
            kept = _kept64(t, case["relu"]).view(t.shape).movedim(-1, 1)
        return {"y": y, "kept": kept} if op == "save" else {"kept": kept}
    if op == "backward":
        g = s["gy"].double()
        if case["relu"]:
            g = torch.where(s["y_codes"].view(g.shape) != 0, g, torch.zeros_like(g))
        at = torch.arange(s["x_codes"].numel(), device="cuda") // BLOCK
        x = (s["x_codes"].double() * torch.exp2(s["x_scales"].double()[at] - 127)).view(case["voxels"], case["cin"])
        out = {"gx": torch.mm(g, s["w"].double()), "gw": torch.mm(g.t(), x), "gbias": g.sum(0)}
        return dict(out, g=g) if case["residual"] else out
    x = _four64(s["x"].double())
    if op == "pack":
        return x
    c = s["w_codes"].long()
    c = torch.stack([torch.remainder(c, 16), torch.div(c, 16, rounding_mode="floor")], 2).flatten(1)
    mag = torch.tensor(_GRID, dtype=torch.float64, device="cuda")[torch.remainder(c, 8)]
    w = torch.where(c >= 8, -mag, mag) * torch.exp2(s["w_scales"].double() - 127).repeat_interleave(BLOCK, 1)
    y = torch.mm(x, w[:, :case["k"]].t()) + s["bias"].double()
    return torch.where(y > 0, y, torch.zeros_like(y)) if case["relu"] else y
