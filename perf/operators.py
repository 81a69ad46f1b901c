"""The int8 projections of an attention layer, as they are timed.

An attention layer's projections are most of its time beside the attention. On
int8 weights a program rounds each row of its bf16 activations to int8 with one
scale for the row, multiplies that with weights rounded once, one scale for each
output channel, and gets bf16 back:

    a[m] = max_k |x[m, k]|,  q[m, k] = round_half_even(127 x[m, k] / a[m]),  s[m] = a[m] / 127
    y[m, n] = (sum_k q[m, k] wq[n, k]) s[m] t[n]

``linear`` is that product (an out-projection, or any layer without a bias);
``qkv`` is the fused Q | K | V projection, whose Q and K heads are then RMS
normalised and rotated by the tokens' (t, h, w) positions and written head-major
with V. Activations arrive in bf16, so both include the rounding to int8; the
weights, their scales, the gammas and the rotation table are what a program keeps.

The sizes are this repository's configurations (``h3hip.configs`` and the
reference model's width) from one token to the longest clip, and odd ones.
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

D = 128                       # channels of a head
TILE = 128                    # head-major rows are padded to this
EPS = 1e-6
DEV = "cuda:0"
PAIR_DIMS = {128: (32, 48, 48), 96: (32, 32, 32)}   # rot -> t, h, w channels


# ------------------------------------------------------------------ the cases

def _linear(name, tokens, inp, out):
    return dict(name=name, op="linear", tokens=tokens, inp=inp, out=out)


def _qkv(name, tokens, inp, heads, rot):
    return dict(name=name, op="qkv", tokens=tokens, inp=inp, heads=heads, rot=rot)


def listed():
    return [
        # One token's out-projection: what a conditioning vector or a single
        # appended token costs, where the weights' bytes and the launch count.
        _linear("linear_1x5120", 1, 5120, 5120),
        # The audio tokens of a 5 s clip on their own.
        _linear("linear_125x5120", 125, 5120, 5120),
        # Odd sizes: a reduction and a width that no tile divides.
        _linear("linear_637x1000_777", 637, 1000, 777),
        # One 864x480 frame behind its text at the reference model's width.
        _linear("linear_1151x7168_5376", 1151, 7168, 5376),
        # The out-projection of the 864x480, 7 s clip.
        _linear("linear_18102x5120", 18102, 5120, 5120),
        # The out-projection of the headline clip, 1344x768, 5 s.
        _linear("linear_31885x5120", 31885, 5120, 5120),
        # One token's Q, K and V.
        _qkv("qkv_1x40", 1, 5120, 40, 128),
        # The text and audio prefix of the headline clip.
        _qkv("qkv_637x40", 637, 5120, 40, 128),
        # One frame at the reference model's width, 96 of 128 channels rotated.
        _qkv("qkv_1151x56", 1151, 5376, 56, 96),
        # A small layer: 4 heads, 4,096 tokens, a short reduction.
        _qkv("qkv_4096x4", 4096, 512, 4, 128),
        # The QKV projection of the 864x480, 7 s clip, and of the headline clip.
        _qkv("qkv_18102x40", 18102, 5120, 40, 128),
        _qkv("qkv_31885x40", 31885, 5120, 40, 128),
    ]


_CAP = {"linear": 31885 * 5120 * 5120, "qkv": 31885 * 5120 * 15360}


def _width(c):
    return c["out"] if c["op"] == "linear" else 3 * c["heads"] * D


def draw(rng):
    """One more case: one token to the headline clip (over the logarithm), the
    layers of both models and others between them, odd widths among them."""
    while True:
        tokens = int(math.exp(rng.uniform(0.0, math.log(31885))))
        model = rng.choice(["small", "wide", "any", "any"])
        if rng.random() < 0.5:
            inp, out = {"small": (5120, 5120), "wide": (7168, 5376)}.get(
                model, (int(math.exp(rng.uniform(math.log(100), math.log(8000)))),
                        int(math.exp(rng.uniform(math.log(100), math.log(8000))))))
            if model == "any" and rng.random() < 0.5:
                inp, out = -(-inp // 64) * 64, -(-out // 64) * 64
            c = dict(op="linear", tokens=tokens, inp=inp, out=out)
        else:
            inp, heads, rot = {"small": (5120, 40, 128), "wide": (5376, 56, 96)}.get(
                model, (8 * rng.randint(16, 700), rng.randint(1, 48), rng.choice([96, 128])))
            c = dict(op="qkv", tokens=tokens, inp=inp, heads=heads, rot=rot)
        if tokens * c["inp"] * _width(c) <= _CAP[c["op"]]:
            return c


# -------------------------------------------------------------------- inputs

def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def _activations(g, tokens, inp):
    """bf16 rows as a layer meets them: tokens of different magnitude, channels of
    different spread with a few outliers among them, and a padding token."""
    channel = torch.exp(0.4 * _randn(g, inp))
    channel[::97] *= 6.0
    x = _randn(g, tokens, inp) * channel * torch.exp(0.3 * _randn(g, tokens, 1))
    if tokens > 8:
        x[tokens // 2] = 0.0
    return x.to(torch.bfloat16)


def _weights(g, out, inp):
    """Int8 rows, padded with zeros to a multiple of 128, and their scales."""
    w = 0.02 * _randn(g, out, inp)
    top = w.abs().amax(1, keepdim=True)
    q = torch.zeros((out, -(-inp // 128) * 128), dtype=torch.int8, device=DEV)
    q[:, :inp] = torch.round(w * (127.0 / top)).to(torch.int8)
    return q, (top[:, 0] / 127.0).contiguous()


def _rotation(tokens, rot):
    """The rotation table of a clip's tokens, [tokens, rot/2, 2, 2] holding
    [[c, -s], [s, c]]: text at the origin, then a (t, h, w) lattice."""
    prefix = min(tokens // 4, 637)
    v = torch.arange(tokens - prefix, device=DEV)
    pos = torch.zeros((tokens, 3), dtype=torch.float64, device=DEV)
    pos[prefix:, 0], pos[prefix:, 1], pos[prefix:, 2] = v // (24 * 42), v // 42 % 24, v % 42
    angles = torch.cat([pos[:, a:a + 1] * 10000.0 ** (-2.0 * torch.arange(d // 2, device=DEV) / d)
                        for a, d in enumerate(PAIR_DIMS[rot])], dim=1)
    c, s = angles.cos(), angles.sin()
    return torch.stack([c, -s, s, c], dim=-1).reshape(tokens, rot // 2, 2, 2).float().contiguous()


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    st = {"case": c, "x": _activations(g, c["tokens"], c["inp"])}
    st["wq"], st["t"] = _weights(g, _width(c), c["inp"])
    if c["op"] == "qkv":
        st["gammas"] = [(0.9 + 0.2 * torch.rand(D, generator=g, device=DEV)).to(torch.bfloat16)
                        for _ in range(2)]
        st["table"] = _rotation(c["tokens"], c["rot"])
    return st


# ------------------------------------------------------------- the plain form

def _product(x, wq, t):
    """The int8 product in fp32. 127 x / a is compared with half steps: in 64 bits."""
    xd = x.double()
    a = xd.abs().amax(1, keepdim=True)
    q = torch.round(127.0 * xd / torch.where(a > 0, a, 1.0)).float()
    y = torch.matmul(q, wq[:, :x.shape[1]].float().t())
    return y * (a / 127.0).float() * t


def _rotate(y, table, rot):
    """[S, H, D]: channels p and p + rot/2 by token angles, the rest unchanged."""
    c, s = table[:, None, :, 0, 0], table[:, None, :, 1, 0]
    a, b = y[..., :rot // 2], y[..., rot // 2:rot]
    return torch.cat([c * a - s * b, s * a + c * b, y[..., rot:]], dim=-1)


def _head_major(y):
    """[S, H, D] -> bf16 [H, S padded, D], rows past S zero."""
    S, H, _ = y.shape
    out = torch.zeros((H, -(-S // TILE) * TILE, D), dtype=torch.bfloat16, device=y.device)
    out[:, :S] = y.transpose(0, 1).to(torch.bfloat16)
    return out


def _plain(st):
    c = st["case"]
    y = _product(st["x"], st["wq"], st["t"])
    if c["op"] == "linear":
        return y.to(torch.bfloat16)
    y = y.view(c["tokens"], 3, c["heads"], D)
    parts = []
    for i, gamma in enumerate(st["gammas"]):
        z = y[:, i]
        z = z * torch.rsqrt(z.square().mean(-1, keepdim=True) + EPS) * gamma.float()
        parts.append(_head_major(_rotate(z, st["table"], c["rot"])))
    return (*parts, _head_major(y[:, 2]))


def run(state):
    if not own:
        return _plain(state)
    c, ops, L = state["case"], *_framework()
    q, s = ops.quant_rows(state["x"])
    if c["op"] == "linear":
        return ops.proj_i8(q, s, state["wq"], state["t"])
    return ops.qkv_proj_i8(q, s, state["wq"], state["t"], *state["gammas"], state["table"],
                           heads=c["heads"], eps=EPS, rounding=L.ROUND_ONCE)


def _framework():
    path = os.path.abspath("minimax-h3-swift_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from h3hip import _lib, ops
    return ops, _lib


# ---------------------------------------------------------------- work, exact

def work(case):
    c, n, m = case, _width(case), case["tokens"]
    moved = 2.0 * m * c["inp"] + n * c["inp"] + 4.0 * n
    if c["op"] == "linear":
        moved += 2.0 * m * n
    else:
        moved += 2.0 * n * -(-m // TILE) * TILE + 8.0 * m * c["rot"]
    return {"bytes": moved, "flops": 2.0 * m * n * c["inp"]}


def exact(case, seed):
    c, st = case, prepare(case, seed)
    x = st["x"].to(torch.float64)
    top = x.abs().max(dim=1).values
    unit = torch.where(top == 0, torch.ones_like(top), top)
    codes = torch.round(x / unit[:, None] * 127.0)
    # A quotient within rounding of a half step is decided in whole numbers:
    # bf16 rows times a power of two are whole, and 254 x against odd multiples of a.
    scaled = x / unit[:, None] * 127.0
    near = ((scaled - torch.floor(scaled) - 0.5).abs() < 1e-9).nonzero()
    if near.numel():
        xs, tops = x[near[:, 0], near[:, 1]].tolist(), unit[near[:, 0]].tolist()
        codes[near[:, 0], near[:, 1]] = torch.tensor(
            [float(_half_even(a, b)) for a, b in zip(xs, tops)], dtype=torch.float64, device=DEV)
    w = st["wq"][:, :c["inp"]].to(torch.float64) * st["t"].to(torch.float64)[:, None]
    y = torch.mm(codes * (top / 127.0)[:, None], w.t().contiguous())
    if c["op"] == "linear":
        return y
    H, S = c["heads"], c["tokens"]
    pad = (S + TILE - 1) // TILE * TILE
    table = st["table"].to(torch.float64)
    res = []
    for part in range(3):
        out = torch.zeros((H, pad, D), dtype=torch.float64, device=DEV)
        for h in range(H):
            col = (part * H + h) * D
            z = y[:, col:col + D]
            if part < 2:
                r = 1.0 / torch.sqrt((z * z).sum(1, keepdim=True) / D + EPS)
                z = z * r * st["gammas"][part].to(torch.float64)
                half = c["rot"] // 2
                turned = z.clone()
                for lo, hi, k in ((0, half, 0), (half, 2 * half, 1)):
                    turned[:, lo:hi] = (table[:, :, k, 0] * z[:, :half]
                                        + table[:, :, k, 1] * z[:, half:2 * half])
                z = turned
            out[h, :S] = z
        res.append(out)
    return tuple(res)


def _half_even(x, a):
    """127 x / a rounded to a whole number, ties to even, from the exact ratio."""
    (p, q), (r, s) = x.as_integer_ratio(), a.as_integer_ratio()
    num, den = 127 * p * s, q * r
    lo, rest = divmod(num, den)
    return lo + (2 * rest > den or (2 * rest == den and lo % 2 != 0))
