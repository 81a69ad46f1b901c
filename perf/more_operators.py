"""An attention block in microscaled 4-bit floats, as its operators are timed.

A DiT block computes r = a x + gate * norm(attention(modulate(norm(x)))) for a residual
stream x. Its projections can run on 4-bit operands: 32 consecutive values of a row
share a power of two and are sign, two exponent bits and one mantissa bit each
(magnitudes 0, 0.5, 1, 1.5, 2, 3, 4, 6):

    a = max |x|,  e = max(floor(log2 a) - 2, -127),  q = round_half_even_e2m1(min(|x| / 2^e, 6))

``rows``    bf16 rows to 4 bits and back: the values that the 4 bits stand for.
``linear``  y = q(x) . w^T, x bf16 and w kept in 4 bits (an out-projection, or any layer
            without a bias).
``qkv``     the same for Q | K | V rows of w; Q and K heads are then RMS normalised and
            rotated by the tokens' (t, h, w) positions, all written head-major.
``before``  h = rms(x) gamma (1 + scale[s]) + shift[s], s being the token's segment.
``after``   r = a x + gate[s] rms(y) gamma, and where asked for the next block's h of it.

Text, audio and video tokens of one sequence are segments with modulations of their own.
The sizes are this repository's configurations (``h3hip.configs`` and the reference
model's width) from one token to the longest clip, and odd ones.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

D = 128                       # channels of a head
TILE = 128                    # head-major rows are padded to this
EPS = 1e-6
BLOCK = 32                    # values that share an exponent
DEV = "cuda:0"
PAIR_DIMS = {128: (32, 48, 48), 96: (32, 32, 32)}   # rot -> t, h, w channels


# ------------------------------------------------------------------ the cases

def _rows(name, tokens, inp):
    return dict(name=name, op="rows", tokens=tokens, inp=inp)


def _linear(name, tokens, inp, out):
    return dict(name=name, op="linear", tokens=tokens, inp=inp, out=out)


def _qkv(name, tokens, inp, heads, rot):
    return dict(name=name, op="qkv", tokens=tokens, inp=inp, heads=heads, rot=rot)


def _before(name, tokens, inp, segments):
    return dict(name=name, op="before", tokens=tokens, inp=inp, segments=segments)


def _after(name, tokens, inp, segments, norm, chained):
    return dict(name=name, op="after", tokens=tokens, inp=inp, segments=segments, norm=norm,
                chained=chained)


def listed():
    return [
        # The headline clip's text and audio at a width that no block divides.
        _rows("rows_637x1001", 637, 1001),
        # The activations of the headline clip, 1344x768, 5 s.
        _rows("rows_31885x5120", 31885, 5120),
        # One token's out-projection: what a conditioning vector or a single appended
        # token costs, where the weights' bytes and the launch count.
        _linear("linear_1x5120", 1, 5120, 5120),
        # Odd sizes: a reduction and a width that no tile divides.
        _linear("linear_637x1000_777", 637, 1000, 777),
        # The out-projection of the headline clip.
        _linear("linear_31885x5120", 31885, 5120, 5120),
        # One token's Q, K and V.
        _qkv("qkv_1x40", 1, 5120, 40, 128),
        # One 864x480 frame behind its text at the reference model's width, 96 of 128
        # channels rotated.
        _qkv("qkv_1151x56", 1151, 5376, 56, 96),
        # The QKV projection of the headline clip.
        _qkv("qkv_31885x40", 31885, 5120, 40, 128),
        # The audio tokens of a 5 s clip on their own, one modulation.
        _before("before_125x5120", 125, 5120, 1),
        # The 864x480, 7 s clip: text, audio and video modulated apart.
        _before("before_18102x5120", 18102, 5120, 3),
        # One token at the reference model's width, the last block's end.
        _after("after_1x5376", 1, 5376, 1, True, False),
        # The headline clip between two blocks: post-norm, gate, residual, next pre-norm.
        _after("after_31885x5120", 31885, 5120, 3, True, True),
    ]


def _width(c):
    return c["out"] if c["op"] == "linear" else 3 * c["heads"] * D


def _log_int(rng, lo, hi):
    return int(math.exp(rng.uniform(math.log(lo), math.log(hi))))


_CAP = {"rows": 31885 * 5120, "linear": 31885 * 5120 * 5120, "qkv": 31885 * 5120 * 15360,
        "before": 18102 * 5120, "after": 31885 * 5120}


def draw(rng):
    """One more case: one token to the headline clip (over the logarithm), the layers of
    both models and others between them, odd widths among them."""
    while True:
        op = rng.choice(["rows", "linear", "linear", "qkv", "qkv", "before", "after"])
        tokens = _log_int(rng, 1.0, 31885.0)
        inp = rng.choice([5120, 5376, _log_int(rng, 33, 8192), 8 * rng.randint(16, 900)])
        c = dict(op=op, tokens=tokens, inp=inp)
        if op == "linear":
            c["out"] = rng.choice([5120, 5376, _log_int(rng, 100, 8000), 64 * rng.randint(2, 120)])
        elif op == "qkv":
            c["heads"], c["rot"] = rng.choice([40, 56, rng.randint(1, 48)]), rng.choice([96, 128])
        elif op in ("before", "after"):
            c["segments"] = rng.randint(1, 4)
            if op == "after":
                c["norm"], c["chained"] = rng.random() < 0.7, rng.random() < 0.6
        if tokens * inp * (_width(c) if op in ("linear", "qkv") else 1) <= _CAP[op]:
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
    """A weight in 4 bits as checkpoints hold it: [out, inp / 2] bytes of two codes, the
    earlier in the low half, and [out, inp / 32] biased exponents; the row is padded with
    zeros to a whole block."""
    pad = -(-inp // BLOCK) * BLOCK
    w = torch.zeros((out, pad), device=DEV)
    w[:, :inp] = 0.02 * _randn(g, out, inp)
    w = w.view(out, -1, BLOCK)
    top = w.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(torch.clamp(top, min=1e-30))) - 2
    mag = torch.clamp((w * torch.exp2(-e)).abs(), max=6.0)
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=DEV)
    code = torch.bucketize(mag, (grid[1:] + grid[:-1]) / 2) + 8 * (w < 0)
    code = code.view(out, pad).to(torch.uint8)
    return code[:, 0::2] | code[:, 1::2] << 4, (e[..., 0] + 127).to(torch.uint8)


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


def _gamma(g, n):
    return (0.9 + 0.2 * torch.rand(n, generator=g, device=DEV)).to(torch.bfloat16)


def _starts(tokens, segments):
    """First token of each segment: text, audio and video lie 512 : 125 : the rest in
    the headline clip. A short sequence leaves some of them empty."""
    return [min(tokens, s) for s in (0, 512, 637, 637 + 24 * 42)[:segments]]


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    st = {"case": c, "x": _activations(g, c["tokens"], c["inp"])}
    if c["op"] in ("linear", "qkv"):
        st["codes"], st["exponents"] = _weights(g, _width(c), c["inp"])
        if own:
            st["w"] = _framework()[0].Mx4Rows.pack(st["codes"], st["exponents"], c["inp"])
    if c["op"] == "qkv":
        st["gammas"] = [_gamma(g, D) for _ in range(2)]
        st["table"] = _rotation(c["tokens"], c["rot"])
    if c["op"] in ("before", "after"):
        def modulation(size):
            return (size * _randn(g, c["segments"], c["inp"])).to(torch.bfloat16)
        st["starts"] = _starts(c["tokens"], c["segments"])
        st["gamma"], st["scale"], st["shift"] = _gamma(g, c["inp"]), modulation(0.3), modulation(0.3)
        if c["op"] == "after":
            st["y"] = _activations(g, c["tokens"], c["inp"])
            st["gate"], st["post"] = modulation(0.5), _gamma(g, c["inp"])
            st["alpha"] = 0.875
    return st


# ------------------------------------------------------------- the plain form

def _pow2(e):
    """fp32 powers of two of int32 exponents from -127 on, exactly."""
    bits = torch.where(e < -126, torch.full_like(e, 1 << 22), (e + 127) << 23)
    return bits.view(torch.float32)


def _round4(x):
    """fp32 rows to the values that their 4-bit form stands for. Every step is exact in
    fp32: the inputs are bf16 and the scales powers of two."""
    rows, cols = x.shape
    pad = -(-cols // BLOCK) * BLOCK
    if pad != cols:
        x = torch.cat([x, x.new_zeros((rows, pad - cols))], dim=1)
    x = x.reshape(rows, -1, BLOCK)
    top = x.abs().amax(-1, keepdim=True)
    e = torch.clamp(torch.frexp(top).exponent - 3, min=-127)
    t = x * _pow2(-e)
    step = _pow2(torch.clamp(torch.frexp(t).exponent - 2, -1, 1))
    t = torch.clamp(torch.round(t / step) * step, -6.0, 6.0)
    return (t * _pow2(e)).view(rows, pad)[:, :cols]


def _decoded(codes, exponents, cols):
    """The fp32 values of a 4-bit weight."""
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=DEV)
    grid = torch.cat([grid, -grid])
    w = torch.stack([grid[(codes & 15).long()], grid[(codes >> 4).long()]], dim=-1)
    w = w.view(codes.shape[0], -1, BLOCK) * _pow2(exponents.int() - 127)[..., None]
    return w.view(codes.shape[0], -1)[:, :cols]


def _rms(x):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)


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


def _per_token(starts, table, tokens):
    """Each token's row of a modulation [segments, inp]."""
    at = torch.zeros(tokens + 1, dtype=torch.long, device=DEV)
    for s in starts[1:]:
        at[s] += 1
    return table.float()[torch.cumsum(at, 0)[:tokens]]


def _plain(st):
    c = st["case"]
    op, tokens, x = c["op"], c["tokens"], st["x"].float()
    if op == "rows":
        return _round4(x).to(torch.bfloat16)
    if op in ("linear", "qkv"):
        y = torch.matmul(_round4(x), _decoded(st["codes"], st["exponents"], c["inp"]).t())
        if op == "linear":
            return y.to(torch.bfloat16)
        y = y.view(tokens, 3, c["heads"], D)
        parts = [_head_major(_rotate(_rms(y[:, i]) * gamma.float(), st["table"], c["rot"]))
                 for i, gamma in enumerate(st["gammas"])]
        return (*parts, _head_major(y[:, 2]))

    def modulated(v):
        scale, shift = (_per_token(st["starts"], st[k], tokens) for k in ("scale", "shift"))
        return (_rms(v) * st["gamma"].float() * (1 + scale) + shift).to(torch.bfloat16)
    if op == "before":
        return modulated(x)
    y = st["y"].float()
    if c["norm"]:
        y = _rms(y) * st["post"].float()
    r = st["alpha"] * x + _per_token(st["starts"], st["gate"], tokens) * y
    return (r.to(torch.bfloat16), modulated(r)) if c["chained"] else r.to(torch.bfloat16)


def run(state):
    if not own:
        return _plain(state)
    st, c, (ops, L) = state, state["case"], _framework()
    if c["op"] == "rows":
        return ops.dequant_rows_mx4(ops.quant_rows_mx4(st["x"]))
    if c["op"] == "linear":
        return ops.proj_mx4(st["x"], st["w"])
    if c["op"] == "qkv":
        return ops.qkv_proj_mx4(st["x"], st["w"], *st["gammas"], st["table"], heads=c["heads"],
                                eps=EPS, rounding=L.ROUND_ONCE)
    norm = dict(gamma=st["gamma"], scale=st["scale"], shift=st["shift"])
    if c["op"] == "before":
        return ops.norm_modulate(st["x"], **norm, segments=st["starts"], eps=EPS)
    return ops.gated_residual(st["x"], st["y"], st["gate"], post_gamma=st["post"] if c["norm"] else None,
                              residual_scale=st["alpha"], segments=st["starts"], eps=EPS,
                              next_norm=norm if c["chained"] else None)


def _framework():
    path = os.path.abspath("minimax-h3-swift_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from h3hip import _lib, ops
    return ops, _lib


# ---------------------------------------------------------------- work, exact

def work(case):
    c, m = case, case["tokens"]
    cells = float(m * c["inp"])
    if c["op"] == "rows":             # to 4 bits and an exponent a block, and back
        return {"bytes": 4.0 * cells + 2 * cells * (0.5 + 1 / BLOCK), "flops": 4.0 * cells}
    if c["op"] == "before":
        return {"bytes": 4.0 * cells + 2.0 * c["inp"] * (1 + 2 * c["segments"]), "flops": 6.0 * cells}
    if c["op"] == "after":
        tables = (1 if c["norm"] else 0) + c["segments"] + (1 + 2 * c["segments"] if c["chained"] else 0)
        return {"bytes": (8.0 if c["chained"] else 6.0) * cells + 2.0 * c["inp"] * tables,
                "flops": (14.0 if c["chained"] else 8.0) * cells}
    n = _width(c)
    moved = 2.0 * cells + n * c["inp"] * (0.5 + 1 / BLOCK)
    if c["op"] == "linear":
        moved += 2.0 * m * n
    else:
        moved += 2.0 * n * -(-m // TILE) * TILE + 8.0 * m * c["rot"]
    return {"bytes": moved, "flops": 2.0 * n * cells}


def _exact4(x):
    """float64 rows to the values of their 4-bit form, by distance to the eight magnitudes;
    a value halfway between two takes the one whose code is even."""
    rows, cols = x.shape
    out = torch.empty_like(x)
    grid = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    for lo in range(0, cols, BLOCK):
        part = x[:, lo:lo + BLOCK]
        top = part.abs().max(dim=1, keepdim=True).values
        exponent = torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top))))
        # log2 next to a whole number may land on its other side.
        exponent = torch.where(2.0 ** exponent > top, exponent - 1, exponent)
        exponent = torch.where(2.0 ** (exponent + 1) <= top, exponent + 1, exponent)
        unit = 2.0 ** torch.clamp(exponent - 2, min=-127)
        mag = part.abs() / unit
        best = torch.zeros_like(mag)
        for code in range(1, 8):
            half = (grid[code - 1] + grid[code]) / 2
            up = mag >= half if code % 2 == 0 else mag > half
            best = torch.where(up, torch.full_like(mag, grid[code]), best)
        out[:, lo:lo + BLOCK] = torch.sign(part) * best * unit
    return out


def _exact_norm(v, gamma):
    v = v / torch.sqrt((v * v).sum(1, keepdim=True) / v.shape[1] + EPS)
    return v * gamma.to(torch.float64)


def exact(case, seed):
    c, st = case, prepare(case, seed)
    S, x = c["tokens"], st["x"].to(torch.float64)
    if c["op"] == "rows":
        return _exact4(x)
    if c["op"] in ("before", "after"):
        ends = st["starts"][1:] + [S]

        def spread(table):
            return torch.cat([table[i].to(torch.float64).expand(max(0, b - a), -1)
                              for i, (a, b) in enumerate(zip(st["starts"], ends))])

        def modulated(v):
            return _exact_norm(v, st["gamma"]) * (1 + spread(st["scale"])) + spread(st["shift"])
        if c["op"] == "before":
            return modulated(x)
        y = st["y"].to(torch.float64)
        r = st["alpha"] * x + spread(st["gate"]) * (_exact_norm(y, st["post"]) if c["norm"] else y)
        return (r, modulated(r)) if c["chained"] else r
    # Two codes a byte, sign in the high bit of each, and a power of two every 32.
    n, pad = _width(c), 2 * st["codes"].shape[1]
    code = torch.empty((n, pad), dtype=torch.int64, device=DEV)
    code[:, 0::2], code[:, 1::2] = st["codes"] % 16, st["codes"] // 16
    low, high = code % 2, code // 2 % 4
    w = torch.where(high == 0, 0.5 * low, 2.0 ** (high - 1).to(torch.float64) * (1 + 0.5 * low))
    w = torch.where(code >= 8, -w, w)
    w *= (2.0 ** (st["exponents"].to(torch.float64) - 127)).repeat_interleave(BLOCK, dim=1)
    y = torch.mm(_exact4(x), w[:, :c["inp"]].t().contiguous())
    if c["op"] == "linear":
        return y
    H, rows = c["heads"], (S + TILE - 1) // TILE * TILE
    table, res = st["table"].to(torch.float64), []
    for part in range(3):
        out = torch.zeros((H, rows, D), dtype=torch.float64, device=DEV)
        for h in range(H):
            z = y[:, (part * H + h) * D:(part * H + h + 1) * D]
            if part < 2:
                z = _exact_norm(z, st["gammas"][part])
                half = c["rot"] // 2
                turned = z.clone()
                for lo, hi, k in ((0, half, 0), (half, 2 * half, 1)):
                    turned[:, lo:hi] = (table[:, :, k, 0] * z[:, :half]
                                        + table[:, :, k, 1] * z[:, half:2 * half])
                z = turned
            out[h, :S] = z
        res.append(out)
    return tuple(res)
