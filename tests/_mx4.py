"""What the 4-bit projection tests share: the format and the operators' definitions in 64
bits, inputs with the values where they can go wrong, and the error bounds.

A product of two e2m1 values is a whole number of quarters up to 36. With exponents 0, 1 and
2 of either operand a sum of K <= 7,168 products is a whole number of quarters below
7,168 * 36 * 16 * 4 < 2^24, so every fp32 sum of any of them in any order is exact and y is
the exact sum rounded to bf16 once, whatever adds: those tests ask for equal bits.

With other exponents each 128 products join a sum in one instruction. However it adds them, as
a tree of seven levels and the sum behind it, each of these eight additions is off by at most
2^-23 (a rounding or a truncation) of magnitudes that together are at most S = sum |x w|: the
sum by K / 16 * 2^-23 S, and the store by 2^-8 of the value; a bf16 subnormal by 2^-134."""
import numpy as np
import torch

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
BLOCK = 32


def bits16(t: torch.Tensor) -> np.ndarray:
    return t.detach().contiguous().view(torch.int16).cpu().numpy()


def quant64(x: np.ndarray):
    """(codes [S, K], biased exponents [S, ceil(K/32)]) of float64 rows that are exact bf16
    values, by the format's definition: the nearest of the grid's magnitudes at most 6, ties to
    the even code. Blocks holding an infinity or a NaN: exponent 255, codes 0."""
    S, K = x.shape
    nb = -(-K // BLOCK)
    pad = np.zeros((S, nb * BLOCK))
    pad[:, :K] = x
    b = pad.reshape(S, nb, BLOCK)
    bad = ~np.isfinite(b).all(-1)
    b = np.where(bad[..., None], 0.0, b)
    top = np.abs(b).max(-1)
    m, e = np.frexp(top)                         # top = m 2^e, m in [0.5, 1)
    e = np.where(top == 0, -127, np.maximum(e - 1 - 2, -127))
    mag = np.abs(b) / np.ldexp(1.0, e)[..., None]
    codes = np.zeros(b.shape, dtype=np.int64)
    for c in range(1, 8):
        half = (GRID[c - 1] + GRID[c]) / 2
        codes = np.where((mag >= half) if c % 2 == 0 else (mag > half), c, codes)
    codes |= np.where(np.signbit(b), 8, 0)
    codes = np.where(bad[..., None], 0, codes).reshape(S, nb * BLOCK)
    return codes[:, :K], np.where(bad, 255, e + 127)


def unpack(values: torch.Tensor) -> np.ndarray:
    """[S, n/2] bytes to [S, n] codes."""
    v = values.cpu().numpy()
    return np.stack([v & 15, v >> 4], -1).reshape(v.shape[0], -1)


def decode64(rows) -> torch.Tensor:
    """An Mx4Rows' values in float64 on its device, from the layout's definition."""
    v = rows.values
    grid = torch.tensor(np.concatenate([GRID, -GRID]), device=v.device)
    codes = torch.stack([v & 15, v >> 4], -1).reshape(v.shape[0], -1)[:, :rows.cols]
    r = torch.arange(v.shape[0], device=v.device)[:, None]
    b = torch.arange(-(-rows.cols // BLOCK), device=v.device)[None, :]
    e = rows.scale[b // 16, r // 16, 16 * (b % 4) + r % 16, b // 4 % 4].double()
    s = torch.where(e == 255, torch.full_like(e, float("nan")), torch.exp2(e - 127))
    return grid[codes.long()] * s.repeat_interleave(BLOCK, 1)[:, :rows.cols]


def mx4_operand(S, K, seed, low=0, span=3, stride=None):
    """Random codes and exponents (biased 127 + low ..), in an Mx4Rows; values with a row
    stride where asked."""
    from h3hip import ops
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    n = -(-K // 2)
    codes = torch.randint(0, 256, (S, n), generator=g, device="cuda", dtype=torch.uint8)
    e = torch.randint(127 + low, 127 + low + span, (S, -(-2 * n // BLOCK)), generator=g, device="cuda",
                      dtype=torch.uint8)
    rows = ops.Mx4Rows.pack(codes, e, K)
    if stride:
        wide = torch.full((S, stride), 0x77, dtype=torch.uint8, device="cuda")
        wide[:, :rows.values.shape[1]] = rows.values
        rows = rows._replace(values=wide[:, :rows.values.shape[1]])
    return rows


def product64(x, w):
    return torch.mm(decode64(x), decode64(w).t().contiguous())


def check_exact(y, want):
    """Bits of the exact sums rounded once."""
    ref = want.float()
    assert torch.equal(ref.double(), want)      # the sums are exact in fp32, as promised
    ref = ref.to(torch.bfloat16)
    same = (y == ref) | (torch.isnan(y) & torch.isnan(ref))
    assert same.all(), f"{int((~same).sum())} of {y.numel()} differ, first at {(~same).nonzero()[0]}"


def product_bound(x, w, want):
    size = torch.mm(decode64(x).abs(), decode64(w).abs().t().contiguous())
    return size * (max(x.cols, 128) / 16 * 2.0 ** -23) + want.abs() * 2.0 ** -8 + 2.0 ** -133


def check_product(y, x, w):
    want = product64(x, w)
    d = (y.double() - want).abs()
    worst = float((d / product_bound(x, w, want)).max()) if d.numel() else 0.0
    print(f"4-bit product: worst error / bound {worst:.3f}", flush=True)
    assert worst <= 1.0
