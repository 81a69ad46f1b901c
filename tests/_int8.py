"""What the int8 projection tests share: the operators' definitions in 64 bits, inputs
with the rows where they can go wrong, and the error bounds.

A product y = sum * x_scale * w_scale has an exact sum; its conversion to fp32 and the
two fp32 products round by at most 2^-24 each (relative), the store to bf16 by 2^-8:
(1 + 2^-24)^3 (1 + 2^-8) - 1 < 2^-8 + 2^-22. A bf16 subnormal is off by at most 2^-134."""
import numpy as np
import torch

Y_REL, Y_ABS = 2.0 ** -8 + 2.0 ** -22, 2.0 ** -133


def quant64(x: np.ndarray):
    """(codes, scales) of float64 rows that are exact bf16 values. 254 x / a is an odd
    whole number for a tie and at least 2^-16 (relative) from one otherwise, far more
    than the quotient's rounding in 64 bits."""
    bad = ~np.isfinite(x).all(axis=1)
    xf = np.where(bad[:, None], 0.0, x)
    a = np.abs(xf).max(axis=1)
    q = np.rint(127.0 * xf / np.where(a == 0, 1.0, a)[:, None]).astype(np.int64)
    s = a.astype(np.float32) / np.float32(127)
    return q, np.where(bad, np.float32(np.nan), s).astype(np.float32)


def bits16(t: torch.Tensor) -> np.ndarray:
    return t.detach().contiguous().view(torch.int16).cpu().numpy()


def to64(t: torch.Tensor) -> np.ndarray:
    return t.detach().double().cpu().numpy()


def rows_bf16(S, K, seed, special=True):
    """bf16 rows on the GPU: normal ones and, among them, what is hard to round."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.randn((S, K), generator=g, device="cuda") * torch.exp(
        2 * torch.randn((S, 1), generator=g, device="cuda"))
    x = x.to(torch.bfloat16)
    if special:
        half = torch.randint(-126, 127, (K,), generator=g, device="cuda") + 0.5
        half[0] = 127.0                     # quotients n + 1/2: every one a tie
        for i, row in enumerate([
                half, half * 2.0 ** -9, half * 2.0 ** 60, -half * 2.0 ** 119,
                torch.zeros(K, device="cuda"),
                x[0].float() * 1e-39,       # bf16 subnormals
                torch.sign(x[0].float()) * 3.3e38,
                x[0].float() * 2.0 ** -118]):
            if 2 * i + 1 < S:
                x[2 * i + 1] = row.to(torch.bfloat16)
    return x


def int8_operands(S, K, N, seed, ldx=None, ldw=None):
    """Random int8 operands over the whole range, -128 too, and fp32 scales of mixed
    magnitude; strided where asked."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.randint(-128, 128, (S, ldx or K), generator=g, device="cuda", dtype=torch.int8)[:, :K]
    w = torch.randint(-128, 128, (N, ldw or K), generator=g, device="cuda", dtype=torch.int8)[:, :K]
    xs = torch.exp(torch.randn((S,), generator=g, device="cuda"))
    ws = torch.exp(torch.randn((N,), generator=g, device="cuda")) * 0.01
    return x, xs, w, ws


def product64(x, xs, w, ws):
    """float64 on the GPU: whole sums below 2^53, scales applied in 64 bits."""
    return torch.mm(x.double(), w.double().t().contiguous()) * xs.double()[:, None] * ws.double()


def check_product(y, want):
    """y (bf16) against float64 values, both on the GPU."""
    d = (y.double() - want).abs()
    bound = want.abs() * Y_REL + Y_ABS
    worst = float((d / bound).max()) if d.numel() else 0.0
    print(f"int8 product: worst error / bound {worst:.3f}", flush=True)
    assert worst <= 1.0
