"""Timed cases of operators around a region decoder's attention: group norm with an activation, rotary positions on
several axes, linear layers with weights in 4 bits.

A map's tokens are normalised before regions look at them, regions and tokens are told their places in the volume, and
a trained head serves a few regions with its weights in 4 bits.  ``listed()`` holds fixed cases, ``draw()`` gives further
ones of the same ranges, ``prepare()`` makes what the caller has in hand on the GPU, ``run()`` makes one pass, ``work()``
says what a pass cannot do without and ``exact()`` gives the same outputs in 64 bits.

Kinds of cases
    group    ``group_norm_act`` of cells [B, cells, C], channels last: forward alone, or with the gradients of the cells,
             the weight and the bias
    rotary   ``rotary_positions`` of heads [B, rows, H, D] at places on one to three axes, forward alone or with the gradient
    linear   ``group_linear``: product with 4-bit weights (e2m1) and a scale for each group of 32, 64 or 128 of a row
"""
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"f16": 2, "bf16": 2, "f32": 4}
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)   # what the codes 0 .. 7 stand for; 8 .. 15: the same, negative


def listed():
    return [
        # serving of one pooled region: a call whose launch counts
        {"name": "group_region_f16", "kind": "group", "dtype": "f16", "train": False, "batch": 1, "cells": 343,
         "channels": 256, "groups": 32, "activation": "silu"},
        # inference on the tokens of a 12 x 48 x 48 level of 256 channels, two samples
        {"name": "group_tokens_bf16", "kind": "group", "dtype": "bf16", "train": False, "batch": 2, "cells": 27648,
         "channels": 256, "groups": 32, "activation": "gelu"},
        # training step on a whole 128^3 volume behind a first layer of 32 channels: larger than what caches hold
        {"name": "group_volume_train_f16", "kind": "group", "dtype": "f16", "train": True, "batch": 2, "cells": 2097152,
         "channels": 32, "groups": 8, "activation": "leaky_relu"},
        # training step at full precision with odd sizes: groups of ten channels, 5 x 17 x 23 cells
        {"name": "group_odd_train_f32", "kind": "group", "dtype": "f32", "train": True, "batch": 3, "cells": 1955,
         "channels": 60, "groups": 6, "activation": "silu"},
        # one query of a decoder at a place between the cells: a call whose launch counts
        {"name": "rotary_query_f16", "kind": "rotary", "dtype": "f16", "train": False, "batch": 1, "rows": 1,
         "heads": 8, "dim": 32, "axes": 3, "pairs": 15, "neighbours": False, "shared": False},
        # keys of the tokens of a 32^3 map, two samples with the same grid
        {"name": "rotary_tokens_bf16", "kind": "rotary", "dtype": "bf16", "train": False, "batch": 2, "rows": 32768,
         "heads": 8, "dim": 64, "axes": 3, "pairs": 30, "neighbours": False, "shared": True},
        # training step: keys of a 12 x 48 x 48 level, scans with a grid each
        {"name": "rotary_tokens_train_f16", "kind": "rotary", "dtype": "f16", "train": True, "batch": 2, "rows": 27648,
         "heads": 8, "dim": 32, "axes": 3, "pairs": 15, "neighbours": True, "shared": False},
        # training step at full precision with odd sizes: regions of images, heads of 40 channels
        {"name": "rotary_odd_train_f32", "kind": "rotary", "dtype": "f32", "train": True, "batch": 3, "rows": 1001,
         "heads": 6, "dim": 40, "axes": 2, "pairs": 18, "neighbours": False, "shared": False},
        # a linear layer of a decoder for one region: a call whose launch counts
        {"name": "linear_one_f16", "kind": "linear", "dtype": "f16", "rows": 1, "inputs": 256, "outputs": 1024,
         "group": 32, "bias": True},
        # first layer of a 3-D head (256 channels x 7^3 cells) for one region: bound by reading the weights
        {"name": "linear_head_bf16", "kind": "linear", "dtype": "bf16", "rows": 1, "inputs": 87808, "outputs": 1024,
         "group": 128, "bias": True},
        # a wide layer for a few regions, odd sizes
        {"name": "linear_few_f16", "kind": "linear", "dtype": "f16", "rows": 13, "inputs": 8100, "outputs": 8190,
         "group": 32, "bias": False},
        # first layer of an image head (256 channels x 7^2 cells) for all regions: bound by the products
        {"name": "linear_regions_bf16", "kind": "linear", "dtype": "bf16", "rows": 2000, "inputs": 12544,
         "outputs": 1024, "group": 64, "bias": True},
    ]


# ---- more cases of the same ranges -------------------------------------------------------------------
def _log(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _draw_group(rng):
    c = {"kind": "group", "dtype": rng.choice(["f16", "f16", "bf16", "bf16", "f32"]), "train": rng.random() < 0.5,
         "batch": _log(rng, 1, 8), "cells": _log(rng, 16, 2097152)}
    c["groups"] = rng.choice([1, 2, 4, 6, 8, 16, 32, 32])
    c["channels"] = c["groups"] * rng.choice([1, 2, 4, 5, 8, 8, 10, 12, 16, 32])
    # (32 bits do not tell on which side of a kink a value next to it lies, and its gradient is another there)
    kinks = [] if c["train"] and c["dtype"] == "f32" else ["relu", "leaky_relu"]
    c["activation"] = rng.choice(["none", "silu", "silu", "gelu", *kinks])
    return c


def _draw_rotary(rng):
    c = {"kind": "rotary", "dtype": rng.choice(["f16", "f16", "bf16", "bf16", "f32"]), "train": rng.random() < 0.5,
         "batch": _log(rng, 1, 8), "rows": _log(rng, 1, 32768), "heads": rng.choice([1, 2, 3, 4, 6, 8, 16]),
         "dim": rng.choice([12, 16, 20, 32, 32, 40, 64, 64, 80, 96, 128]), "axes": rng.choice([1, 2, 3, 3, 3]),
         "neighbours": rng.random() < 0.4, "shared": rng.random() < 0.5}
    most = c["dim"] // 2 // c["axes"]
    c["pairs"] = c["axes"] * rng.choice([most, most, max(1, most // 2)])
    return c


def _draw_linear(rng):
    c = {"kind": "linear", "dtype": rng.choice(["f16", "bf16"]), "rows": rng.choice([1, 1, 2, 5, 8, _log(rng, 1, 64), _log(rng, 1, 4000)]),
         "inputs": _log(rng, 16, 87808), "outputs": _log(rng, 8, 8192), "group": rng.choice([32, 32, 64, 128]),
         "bias": rng.random() < 0.5}
    if rng.random() < 0.6:
        c["inputs"] = -(-c["inputs"] // 64) * 64
        c["outputs"] = -(-c["outputs"] // 16) * 16
    return c


def draw(rng):
    while True:
        c = rng.choice([_draw_group, _draw_rotary, _draw_linear])(rng)
        if _cost(c) <= _MOST[c["kind"]]:
            return c


def _cost(c):
    if c["kind"] == "group":
        return c["batch"] * c["cells"] * c["channels"] * (2 if c["dtype"] == "f32" else 1)
    if c["kind"] == "rotary":
        return c["batch"] * c["rows"] * c["heads"] * c["dim"] * (2 if c["dtype"] == "f32" else 1)
    return (c["rows"] + 128) * c["inputs"] * c["outputs"]   # (the plain form makes the weights first)


_MOST = {"group": 2 * 2097152 * 32, "rotary": 2 * 32768 * 8 * 64, "linear": (2000 + 128) * 12544 * 1024}


# ---- inputs --------------------------------------------------------------------------------------------
def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _to_4_bits(w, group):
    """Codes and scales of a matrix: columns padded with zeros to whole blocks of 128; two codes a byte, the first one in
    its low half; the four bytes of eight neighbouring columns together, and of a block's sixteen such pieces piece
    4 s + g at place 4 g + s."""
    n, k = w.shape
    w = torch.nn.functional.pad(w, (0, -k % 128)).reshape(n, -1, group)
    scales = (w.abs().amax(2) / 6.0).clamp(min=2.0 ** -126)
    t = w * (1.0 / scales)[:, :, None]
    size = t.abs()
    code = ((size > 0.25).byte() + (size >= 0.75).byte() + (size > 1.25).byte() + (size >= 1.75).byte() + (size > 2.5).byte()
            + (size >= 3.5).byte() + (size > 5.0).byte())   # to the nearest level, halves to the even code
    code = (code + 8 * (t < 0).byte()).reshape(n, -1, 4, 4, 8).transpose(2, 3)
    return (code[..., 0::2] + 16 * code[..., 1::2]).reshape(n, -1), scales


def prepare(case, seed):
    c, dtype = case, DTYPES[case["dtype"]]
    g = torch.Generator(device="cuda").manual_seed(seed)
    if c["kind"] == "group":
        shape = (c["batch"], c["cells"], c["channels"])
        # channels of different strength around a value of their own, as a convolution gives them
        middle, strength = _randn(g, c["channels"]), torch.exp(0.5 * _randn(g, c["channels"]))
        s = {"case": c, "x": (_randn(g, *shape).mul_(strength).add_(middle)).to(dtype),
             "weight": (1 + 0.2 * _randn(g, c["channels"])).to(dtype), "bias": (0.3 * _randn(g, c["channels"])).to(dtype)}
        if c["train"]:
            for name in ("x", "weight", "bias"):
                s[name].requires_grad_(True)
            s["grad"] = _randn(g, *shape).to(dtype)
        return s
    if c["kind"] == "rotary":
        rows = c["rows"]
        if c["shared"]:   # cells of a grid, in their order, in voxels of the volume
            side = max(1, round(rows ** (1 / c["axes"])))
            at = torch.arange(rows, device="cuda")
            place = torch.stack([at // side ** a % side if a + 1 < c["axes"] else at // side ** a for a in range(c["axes"])], 1)
            place = place.float() * 4 + 1.5 + 0.01 * torch.rand(c["axes"], generator=g, device="cuda")
        else:             # middles of regions and cells of grids that differ from scan to scan
            place = 128 * torch.rand((c["batch"], rows, c["axes"]), generator=g, device="cuda")
        # a share of the pairs for each axis: turns from one voxel to a few hundred
        each = c["pairs"] // c["axes"]
        turn = 100.0 ** (-torch.arange(each, device="cuda", dtype=torch.float64) / each)
        frequencies = torch.zeros(c["axes"], c["pairs"], device="cuda", dtype=torch.float64)
        for a in range(c["axes"]):
            frequencies[a, a * each:(a + 1) * each] = turn
        shape = (c["batch"], rows, c["heads"], c["dim"])
        s = {"case": c, "x": _randn(g, *shape).to(dtype), "positions": place, "frequencies": frequencies}
        if c["train"]:
            s["x"].requires_grad_(True)
            s["grad"] = _randn(g, *shape).to(dtype)
        return s
    x = _randn(g, c["rows"], c["inputs"]).relu_().mul_(torch.exp(0.5 * _randn(g, c["inputs"])))   # pooled features
    w, scales = _to_4_bits(_randn(g, c["outputs"], c["inputs"]) / math.sqrt(c["inputs"]), c["group"])
    return {"case": c, "x": x.to(dtype), "weight": w, "scales": scales,
            "bias": _randn(g, c["outputs"]).to(dtype) if c["bias"] else None}


# ---- plain forms ---------------------------------------------------------------------------------------
def _activated(z, activation):
    if activation == "none":
        return z
    if activation == "silu":
        return z * torch.sigmoid(z)
    if activation == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return torch.where(z > 0, z, z * (0.01 if activation == "leaky_relu" else 0.0))


def _group_norm(x, groups, weight, bias, activation):
    b, n, ch = x.shape
    f = x.float().reshape(b, n, groups, ch // groups)
    d = f - f.mean((1, 3), keepdim=True)
    h = d * torch.rsqrt(d.square().mean((1, 3), keepdim=True) + 1e-5)
    return _activated(h.reshape(b, n, ch) * weight.float() + bias.float(), activation).to(x.dtype)


def _rotated(x, positions, frequencies, neighbours):
    pairs = frequencies.shape[1]
    angle = positions.double() @ frequencies   # far places: 32 bits would lose the turn
    cos, sin = angle.cos().float()[..., None, :], angle.sin().float()[..., None, :]
    f = x.float()
    if neighbours:
        a, b = f[..., 0:2 * pairs:2], f[..., 1:2 * pairs:2]
        y = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = f[..., :pairs], f[..., pairs:2 * pairs]
        y = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((y, f[..., 2 * pairs:]), -1).to(x.dtype)


def _values(weight, scales, inputs):
    """What 4-bit weights and their scales stand for, in 32 bits."""
    n = weight.shape[0]
    code = torch.stack((weight & 15, weight >> 4), -1).reshape(n, -1, 4, 4, 8).transpose(2, 3).reshape(n, scales.shape[1], -1)
    level = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=weight.device)
    return (level[code.int()] * scales[:, :, None]).reshape(n, -1)[:, :inputs]


# ---- one pass ------------------------------------------------------------------------------------------
def run(state):
    if own:
        import medvision_amd.ops as ops
    s, c = state, state["case"]
    if c["kind"] == "group":
        x, w, b, kind = s["x"], s["weight"], s["bias"], c["activation"]
        if own:
            y = ops.group_norm_act(x, c["groups"], w, b, eps=1e-5, activation=None if kind == "none" else kind)
        else:
            y = _group_norm(x, c["groups"], w, b, kind)
        return (y, *torch.autograd.grad(y, (x, w, b), s["grad"])) if c["train"] else y
    if c["kind"] == "rotary":
        x, p, f = s["x"], s["positions"], s["frequencies"]
        if own:
            y = ops.rotary_positions(x, p, f, neighbours=c["neighbours"])
        else:
            y = _rotated(x, p, f, c["neighbours"])
        return (y, *torch.autograd.grad(y, (x,), s["grad"])) if c["train"] else y
    if own:
        return ops.group_linear(s["x"], s["weight"], s["scales"], s["bias"])
    y = s["x"].float() @ _values(s["weight"], s["scales"], c["inputs"]).t()
    return (y if s["bias"] is None else y + s["bias"].float()).to(s["x"].dtype)


# ---- what a pass cannot do without ---------------------------------------------------------------------
def work(case):
    c, size = case, BYTES[case["dtype"]]
    if c["kind"] == "group":   # training: cells and incoming gradient read, result and gradient written
        n = c["batch"] * c["cells"] * c["channels"]
        return {"bytes": n * size * (4 if c["train"] else 2) + c["channels"] * size * (4 if c["train"] else 2),
                "flops": n * (24 if c["train"] else 10)}
    if c["kind"] == "rotary":
        n = c["batch"] * c["rows"] * c["heads"] * c["dim"]
        places = (1 if c["shared"] else c["batch"]) * c["rows"] * c["axes"]
        return {"bytes": n * size * (4 if c["train"] else 2) + 4 * places, "flops": 3 * n * (2 if c["train"] else 1)}
    padded = -(-c["inputs"] // 128) * 128
    return {"bytes": c["outputs"] * (padded // 2 + padded // c["group"] * 4) + c["rows"] * (c["inputs"] + c["outputs"]) * size,
            "flops": 2 * c["rows"] * c["inputs"] * c["outputs"]}


# ---- the same in 64 bits -------------------------------------------------------------------------------
def _slope(z, kind):
    """An activation and its derivative."""
    if kind == "none":
        return z, torch.ones_like(z)
    if kind == "silu":
        p = 1.0 / (1.0 + torch.exp(-z))
        return z * p, p * (1.0 + z * (1.0 - p))
    if kind == "gelu":
        p = 0.5 * torch.erfc(-z / math.sqrt(2.0))
        return z * p, p + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    low = 0.01 if kind == "leaky_relu" else 0.0
    d = (z > 0).double() * (1.0 - low) + low
    return z * d, d


def _exact_group(s):
    c = s["case"]
    each = c["channels"] // c["groups"]
    w, b = s["weight"].detach().double(), s["bias"].detach().double()
    y = torch.empty(s["x"].shape, device=w.device, dtype=torch.float64)
    dx, dw, db = (torch.empty_like(y), torch.zeros_like(w), torch.zeros_like(b)) if c["train"] else (None, None, None)
    for i in range(c["batch"]):
        for g in range(c["groups"]):
            at = slice(g * each, (g + 1) * each)
            x = s["x"][i, :, at].detach().double()
            var, mean = torch.var_mean(x, unbiased=False)
            r = 1.0 / torch.sqrt(var + 1e-5)
            h = (x - mean) * r
            y[i, :, at], d = _slope(h * w[at] + b[at], c["activation"])
            if not c["train"]:
                continue
            gz = s["grad"][i, :, at].double() * d
            db[at] += gz.sum(0)
            dw[at] += (gz * h).sum(0)
            gz = gz * w[at]
            dx[i, :, at] = r * (gz - gz.mean() - h * (gz * h).mean())
    return (y, dx, dw, db) if c["train"] else y


def _exact_rotary(s):
    c, turn = s["case"], s["frequencies"]
    n = c["pairs"]
    first = torch.arange(n, device=turn.device) * (2 if c["neighbours"] else 1)
    second = first + (1 if c["neighbours"] else n)
    angle = sum(s["positions"].double()[..., a, None] * turn[a] for a in range(c["axes"])).unsqueeze(-2)
    unit = torch.polar(torch.ones_like(angle), angle)

    def turned(t, unit):
        t = t.detach().double()
        z = torch.complex(t[..., first], t[..., second]) * unit
        t[..., first], t[..., second] = z.real, z.imag
        return t

    y = turned(s["x"], unit)
    return (y, turned(s["grad"], unit.conj())) if c["train"] else y


def _exact_linear(s):
    c = s["case"]
    x = s["x"].double()
    level = torch.tensor(LEVELS, device=x.device, dtype=torch.float64)
    column = torch.arange(c["inputs"], device=x.device)
    piece = column // 8 % 16
    byte = column // 128 * 64 + (piece % 4 * 4 + piece // 4) * 4 + column % 8 // 2
    y = torch.zeros(c["rows"], c["outputs"], dtype=torch.float64, device=x.device)
    for first in range(0, c["outputs"], 128):
        code = s["weight"][first:first + 128][:, byte] >> (4 * (column % 2)) & 15
        w = level[(code & 7).long()] * (1.0 - 2.0 * (code >> 3).double())
        y[:, first:first + 128] = x @ (w * s["scales"][first:first + 128].double()[:, column // c["group"]]).t()
    return y if s["bias"] is None else y + s["bias"].double()


def exact(case, seed):
    s = prepare(case, seed)
    return {"group": _exact_group, "rotary": _exact_rotary, "linear": _exact_linear}[case["kind"]](s)
