"""Torch-facing calls into libch3hip.

torch supplies device memory and the current HIP stream; every computation is
one of the library's HIP kernels. Inputs must already be on the GPU: there is
no host or torch fallback, and a declined call returns ``None`` so the caller
can run its own dense path, exactly as the reference's backends decline.
"""
from __future__ import annotations

import ctypes
import functools
import math
from typing import NamedTuple

import numpy as np
import torch

from . import _lib as L
from .topology import TilePlan


def _ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _stream(t: torch.Tensor):
    return ctypes.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def _require_gpu_bf16(name: str, t: torch.Tensor):
    if not t.is_cuda:
        raise ValueError(f"{name} must be a GPU tensor (no host fallback exists)")
    if t.dtype != torch.bfloat16:
        raise ValueError(f"{name} must be bfloat16, got {t.dtype}")


# ------------------------------------------------------------------ host tables

def rope_pairs_axes(theta: float = 10000.0, dims=(32, 48, 48)):
    """Per-pair (axis, inv_freq) for three-axis RoPE with the given channel split."""
    n = sum(dims) // 2
    ax = np.zeros(n, dtype=np.int32)
    inv = np.zeros(n, dtype=np.float32)
    got = L.lib().h3hip_rope_pairs_axes(theta, dims[0], dims[1], dims[2],
                                        ax.ctypes.data_as(ctypes.POINTER(ctypes.c_int32)),
                                        inv.ctypes.data_as(ctypes.POINTER(ctypes.c_float)))
    L.check(min(got, 0))
    return ax, inv


def rope_pairs_h3(inv_freq: np.ndarray):
    """H3RoPE's pair table from the checkpoint's inv_freq (H3Transformer.swift:64-78)."""
    f = np.ascontiguousarray(inv_freq, dtype=np.float32)
    ax = np.zeros(3 * len(f), dtype=np.int32)
    inv = np.zeros(3 * len(f), dtype=np.float32)
    got = L.lib().h3hip_rope_pairs_h3(f.ctypes.data_as(ctypes.POINTER(ctypes.c_float)), len(f),
                                      ax.ctypes.data_as(ctypes.POINTER(ctypes.c_int32)),
                                      inv.ctypes.data_as(ctypes.POINTER(ctypes.c_float)))
    L.check(min(got, 0))
    return ax, inv


def positions_grid(prefix_len: int, frames: int, height: int, width: int) -> np.ndarray:
    pos = np.zeros((prefix_len + frames * height * width, 3), dtype=np.float32)
    got = L.lib().h3hip_positions_grid(prefix_len, frames, height, width,
                                       pos.ctypes.data_as(ctypes.POINTER(ctypes.c_float)))
    L.check(min(got, 0))
    return pos


def positions_packed(text_tokens: int, audio_t: int, latent_t: int, latent_h: int,
                     latent_w: int, patch: int = 2) -> np.ndarray:
    n = text_tokens + 2 * audio_t + latent_t * (latent_h // patch) * (latent_w // patch)
    pos = np.zeros((n, 3), dtype=np.float64)
    got = L.lib().h3hip_positions_packed(text_tokens, audio_t, latent_t, latent_h, latent_w,
                                         patch,
                                         pos.ctypes.data_as(ctypes.POINTER(ctypes.c_double)))
    L.check(min(got, 0))
    return pos


# --------------------------------------------------------------------- prologue

def qk_norm_rope(q_in: torch.Tensor, k_in: torch.Tensor, q_gamma: torch.Tensor,
                 k_gamma: torch.Tensor, pos: torch.Tensor, pair_axis: torch.Tensor,
                 pair_inv: torch.Tensor, *, heads: int, head_dim: int = 128,
                 eps: float = 1e-6, rot: int | None = None, seq_pad: int | None = None,
                 v_in: torch.Tensor | None = None, rounding: int = L.ROUND_REFERENCE,
                 out=None):
    """Fused RMSNorm + RoPE + head-major relayout of token-major Q and K.

    q_in/k_in: [S, >= heads*head_dim] bf16 views sharing one row stride (e.g.
    slices of a fused qkv projection). Returns (q_out, k_out, v_out) as
    [heads, seq_pad, head_dim] bf16, or None when the geometry is declined."""
    for name, t in (("q_in", q_in), ("k_in", k_in), ("q_gamma", q_gamma),
                    ("k_gamma", k_gamma)):
        _require_gpu_bf16(name, t)
    if q_in.dim() != 2 or q_in.stride(1) != 1 or k_in.stride() != q_in.stride():
        raise ValueError("q_in and k_in must be row-major 2-D views with the same row stride")
    S = q_in.shape[0]
    seq_pad = seq_pad or ((S + L.TILE - 1) // L.TILE) * L.TILE
    rot = rot if rot is not None else 2 * pair_axis.numel()
    if v_in is not None:
        _require_gpu_bf16("v_in", v_in)
        if v_in.stride() != q_in.stride():
            raise ValueError("v_in must share q_in's row stride")
    for name, t, dt in (("pos", pos, torch.float32), ("pair_axis", pair_axis, torch.int32),
                        ("pair_inv", pair_inv, torch.float32)):
        if not t.is_cuda or t.dtype != dt or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous {dt} GPU tensor")
    if pos.dim() != 2 or pos.shape[0] < S or pos.shape[1] != 3:
        raise ValueError(f"pos must be [>= {S}, 3]")
    if pair_axis.numel() < rot // 2 or pair_inv.numel() < rot // 2:
        raise ValueError(f"pair tables must hold rot/2 = {rot // 2} entries")
    if q_in.shape[1] < heads * head_dim or seq_pad % 4 or seq_pad < S:
        raise ValueError("q_in narrower than heads*head_dim, or bad seq_pad")
    if out is None:
        dev = q_in.device
        shape = (heads, seq_pad, head_dim)
        q_out = torch.empty(shape, dtype=torch.bfloat16, device=dev)
        k_out = torch.empty(shape, dtype=torch.bfloat16, device=dev)
        v_out = torch.empty(shape, dtype=torch.bfloat16, device=dev) if v_in is not None else None
    else:
        q_out, k_out, v_out = out
        for t in (q_out, k_out) + ((v_out,) if v_in is not None else ()):
            if t.shape != (heads, seq_pad, head_dim) or not t.is_contiguous():
                raise ValueError("outputs must be contiguous [heads, seq_pad, head_dim]")
    rc = L.lib().h3hip_qk_norm_rope(_ptr(q_in), _ptr(k_in), q_in.stride(0), _ptr(v_in),
                                    _ptr(q_gamma), _ptr(k_gamma), eps, _ptr(pos),
                                    _ptr(pair_axis), _ptr(pair_inv), rot, rounding, S, seq_pad,
                                    heads, head_dim, _ptr(q_out), _ptr(k_out), _ptr(v_out),
                                    _stream(q_in))
    if L.check(rc, allow_declined=True) == L.DECLINED:
        return None
    return q_out, k_out, v_out


def head_major(x: torch.Tensor, *, heads: int, head_dim: int = 128, seq_pad: int | None = None,
               out: torch.Tensor | None = None):
    """Token-major [S, >= heads*head_dim] bf16 (row stride free, unit column
    stride) -> head-major [heads, seq_pad, head_dim], rows >= S zero: the
    materialised transpose of AttentionLayer.sdpa. Returns None when declined."""
    if x.dim() != 2 or x.stride(1) != 1 or x.shape[1] < heads * head_dim:
        raise ValueError(f"x must be a 2-D view [S, >= {heads * head_dim}] with unit column "
                         f"stride, got shape {tuple(x.shape)} strides {x.stride()}")
    S = x.shape[0]
    seq_pad = seq_pad or ((S + L.TILE - 1) // L.TILE) * L.TILE
    shape = (heads, seq_pad, head_dim)
    if out is not None:
        _require_out(out, shape, x.device)
    _require_gpu_bf16("x", x)
    if out is None:
        out = torch.empty(shape, dtype=torch.bfloat16, device=x.device)
    rc = L.lib().h3hip_head_major(_ptr(x), x.stride(0), S, seq_pad, heads, head_dim, _ptr(out),
                                  _stream(x))
    if L.check(rc, allow_declined=True) == L.DECLINED:
        return None
    return out


def rope_table(pos: torch.Tensor, pair_axis: torch.Tensor, pair_inv: torch.Tensor, *,
               rot: int | None = None, rounding: int = L.ROUND_REFERENCE,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """The render's rotation table (H3RoPE.rotationTable): [S, rot/2, 2, 2]
    holding [[c, -s], [s, c]], bf16 for REFERENCE rounding, fp32 for FP32 and ONCE."""
    for name, t, dt in (("pos", pos, torch.float32), ("pair_axis", pair_axis, torch.int32),
                        ("pair_inv", pair_inv, torch.float32)):
        if not t.is_cuda or t.dtype != dt or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous {dt} GPU tensor")
    rot = rot if rot is not None else 2 * pair_axis.numel()
    if pos.dim() != 2 or pos.shape[1] != 3:
        raise ValueError("pos must be [S, 3]")
    if pair_axis.numel() < rot // 2 or pair_inv.numel() < rot // 2:
        raise ValueError(f"pair tables must hold rot/2 = {rot // 2} entries")
    S = pos.shape[0]
    dt = torch.bfloat16 if rounding == L.ROUND_REFERENCE else torch.float32
    shape = (S, rot // 2, 2, 2)
    if out is None:
        out = torch.empty(shape, dtype=dt, device=pos.device)
    elif out.shape != shape or out.dtype != dt or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous {dt} tensor of shape {shape}")
    L.check(L.lib().h3hip_rope_table(_ptr(pos), _ptr(pair_axis), _ptr(pair_inv), rot, rounding,
                                     S, _ptr(out), _stream(pos)))
    return out


def qkv_proj(x: torch.Tensor, w: torch.Tensor, q_gamma: torch.Tensor | None = None,
             k_gamma: torch.Tensor | None = None, table: torch.Tensor | None = None, *,
             heads: int, head_dim: int = 128, eps: float = 1e-6,
             seq_pad: int | None = None, rounding: int = L.ROUND_REFERENCE, out=None):
    """QKV projection x . w^T with the Q/K norm + RoPE prologue in its epilogue.

    x: [S, hidden] bf16 (row stride free, unit column stride); w: [3*heads*head_dim,
    hidden] bf16 (Q | K | V rows); table: the render's rotation table from
    rope_table() for the same rounding mode ([>= S, rot/2, 2, 2]). With q_gamma =
    k_gamma = None this is the plain GEMM written head-major. Returns (q, k, v)
    as [heads, seq_pad, head_dim] bf16, or None when the geometry is declined."""
    _require_gpu_bf16("x", x)
    _require_gpu_bf16("w", w)
    if x.dim() != 2 or w.dim() != 2 or x.stride(1) != 1 or w.stride(1) != 1:
        raise ValueError("x and w must be 2-D with unit column stride")
    S, hidden = x.shape
    if w.shape != (3 * heads * head_dim, hidden):
        raise ValueError(f"w must be [{3 * heads * head_dim}, {hidden}], got {tuple(w.shape)}")
    seq_pad = seq_pad or ((S + L.TILE - 1) // L.TILE) * L.TILE
    plain = q_gamma is None and k_gamma is None
    if plain:
        rot = head_dim
    else:
        for name, t in (("q_gamma", q_gamma), ("k_gamma", k_gamma)):
            _require_gpu_bf16(name, t)
        dt = torch.bfloat16 if rounding == L.ROUND_REFERENCE else torch.float32
        if (table is None or not table.is_cuda or table.dtype != dt or not table.is_contiguous()
                or table.dim() != 4 or table.shape[0] < S or table.shape[2:] != (2, 2)):
            raise ValueError(f"table must be a contiguous {dt} [>= {S}, rot/2, 2, 2] GPU tensor "
                             "(rope_table() with the same rounding mode)")
        rot = 2 * table.shape[1]
    shape = (heads, seq_pad, head_dim)
    if out is None:
        q_out, k_out, v_out = (torch.empty(shape, dtype=torch.bfloat16, device=x.device)
                               for _ in range(3))
    else:
        q_out, k_out, v_out = out
        for t in (q_out, k_out, v_out):
            if t.shape != shape or not t.is_contiguous() or t.dtype != torch.bfloat16:
                raise ValueError("outputs must be contiguous bf16 [heads, seq_pad, head_dim]")
    rc = L.lib().h3hip_qkv_proj(_ptr(x), x.stride(0), _ptr(w), w.stride(0), hidden,
                                _ptr(q_gamma), _ptr(k_gamma), eps, _ptr(table), rot, rounding,
                                S, seq_pad, heads, head_dim, _ptr(q_out), _ptr(k_out),
                                _ptr(v_out), _stream(x))
    if L.check(rc, allow_declined=True) == L.DECLINED:
        return None
    return q_out, k_out, v_out


def out_proj(x: torch.Tensor, w: torch.Tensor, out: torch.Tensor | None = None):
    """Out-projection y = x . w^T (DiTBlock.swift:359, matmul(merged,
    outWeight.T)): x [S, in_features] bf16 (the attention's token-major
    output), w [out_features, in_features] bf16; returns y [S, out_features]
    bf16 (or writes ``out``, any row stride), or None when declined."""
    _require_gpu_bf16("x", x)
    _require_gpu_bf16("w", w)
    if x.dim() != 2 or w.dim() != 2 or x.stride(1) != 1 or w.stride(1) != 1:
        raise ValueError("x and w must be 2-D with unit column stride")
    S, fin = x.shape
    if w.shape[1] != fin:
        raise ValueError(f"w must be [out_features, {fin}], got {tuple(w.shape)}")
    fout = w.shape[0]
    if out is None:
        out = torch.empty((S, fout), dtype=torch.bfloat16, device=x.device)
    elif (out.dim() != 2 or out.shape != (S, fout) or out.stride(1) != 1
          or out.dtype != torch.bfloat16 or not out.is_cuda):
        raise ValueError(f"out must be a bf16 GPU [{S}, {fout}] view with unit column stride")
    rc = L.lib().h3hip_out_proj(_ptr(x), x.stride(0), _ptr(w), w.stride(0), fin, fout, S,
                                _ptr(out), out.stride(0), _stream(x))
    if L.check(rc, allow_declined=True) == L.DECLINED:
        return None
    return out


# ------------------------------------------------------------- int8 projections

# These calls can be as short as their launches (2.5 us), so the host work around them is kept
# small: the raw stream handle without a Stream object, the device switched only where the
# operands are not on the current one, sizes given to torch.empty one by one (1.3 us; as a
# tuple 1.7).
INT8_MAX_REDUCTION = 131071      # in features whose sums stay in int32, whatever the values
_I8, _F32, _BF16 = torch.int8, torch.float32, torch.bfloat16
_empty = torch.empty
# A torch built without a GPU backend has neither function (and no tensor that needs them).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_current_device = getattr(torch._C, "_cuda_getDevice", None)


def _run(fn, device: torch.device, *args) -> int:
    """fn(*args, stream) on the current stream of ``device``; DECLINED or OK."""
    index = device.index
    if _current_device() == index:
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    return rc if rc == L.OK else L.check(rc, allow_declined=True)


# Sizes go to 32-bit parameters, into which ctypes cuts a larger number without an error.
_INT32_MAX = 2 ** 31 - 1


def _require_int32(name: str, t: torch.Tensor):
    if max(t.shape) > _INT32_MAX:
        raise ValueError(f"{name} must have sizes below 2^31, got {tuple(t.shape)}")


def _require_same_device(device: torch.device, **others):
    for name, t in others.items():
        if t.device != device:
            raise ValueError(f"{name} must be on {device}, got {t.device}")


def _rows(name: str, t: torch.Tensor, dtype) -> int:
    """The row stride of a 2-D tensor whose rows are contiguous. A single row has none that
    matters: the least that covers it and keeps the next one aligned."""
    if t.dtype != dtype or t.dim() != 2:
        raise ValueError(f"{name} must be 2-D {dtype}, got {t.dim()}-D {t.dtype}")
    ld, step = t.stride()
    rows, cols = t.shape
    if step != 1 and cols > 1:
        raise ValueError(f"{name} must have unit column stride, got strides {t.stride()}")
    return ld if rows > 1 else (cols + 15) // 16 * 16


def _vector(name: str, t: torch.Tensor, n: int, device: torch.device):
    if t.dtype != torch.float32 or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous fp32 [{n}], got {t.dtype} {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}, got {t.device}")


def quant_rows(x: torch.Tensor, out=None):
    """Rows of bf16 rounded to int8 with one scale a row.

    x: [S, K] bf16 (row stride free, unit column stride). Returns (q, scale): int8
    [S, K padded to a multiple of 128] (zeros past K) and fp32 [S], x being about
    q * scale: the activations of an int8 projection, or its weights, rounded once.
    A row holding an infinity or a NaN gets the scale NaN. ``out`` is such a pair to
    write into."""
    ldx = _rows("x", x, _BF16)
    S, K = x.shape
    if K == 0:
        raise ValueError("x must be [S, K > 0]")
    if S > _INT32_MAX or K > _INT32_MAX:
        _require_int32("x", x)
    if not x.is_cuda:
        raise ValueError("x must be a GPU tensor (no host fallback exists)")
    device, pad = x.device, (K + 127) // 128 * 128
    if out is None:
        q = _empty(S, pad, dtype=_I8, device=device)
        scale = _empty(S, dtype=_F32, device=device)
        ldq = pad
    else:
        q, scale = out
        ldq = _rows("out[0]", q, _I8)
        if q.shape != (S, pad):
            raise ValueError(f"out[0] must be [{S}, {pad}], got {tuple(q.shape)}")
        _require_same_device(device, q=q)
        _vector("out[1]", scale, S, device)
    _run(L.lib().h3hip_quant_rows, device, x.data_ptr(), ldx, S, K, q.data_ptr(), ldq,
         scale.data_ptr())
    return q, scale


def _int8_operands(x, x_scale, w, w_scale):
    """Checks the operands of an int8 projection; returns (device, S, K, N, ldx, ldw)."""
    if x.dim() == w.dim() == 2:
        (S, K), (N, k) = x.shape, w.shape
        if S > _INT32_MAX or K > _INT32_MAX or N > _INT32_MAX:
            _require_int32("x", x)
            _require_int32("w", w)
        (ldx, step), (ldw, step_w) = x.stride(), w.stride()
        device = x.device
        if (x.dtype is _I8 and w.dtype is _I8 and x_scale.dtype is _F32 and w_scale.dtype is _F32
                and k == K and step == 1 and step_w == 1 and x_scale.shape == (S,)
                and w_scale.shape == (N,) and x_scale.is_contiguous() and w_scale.is_contiguous()
                and x.is_cuda and w.device == device and x_scale.device == device
                and w_scale.device == device):
            return device, S, K, N, (ldx if S > 1 else K), (ldw if N > 1 else K)
    # What of it is refused, one by one.
    _rows("x", x, _I8)
    _rows("w", w, _I8)
    if w.shape[1] != x.shape[1]:
        raise ValueError(f"w must be [out, {x.shape[1]}], got {tuple(w.shape)}")
    _require_same_device(x.device, w=w)
    _vector("x_scale", x_scale, x.shape[0], x.device)
    _vector("w_scale", w_scale, w.shape[0], x.device)
    raise ValueError("x must be a GPU tensor of more than one column (no host fallback exists)")


def proj_i8(x: torch.Tensor, x_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
            out: torch.Tensor | None = None):
    """A projection on int8 operands: y = (x . w^T) * w_scale * x_scale[:, None].

    x: [S, K] int8 and x_scale: [S] fp32, w: [N, K] int8 and w_scale: [N] fp32, as
    quant_rows() makes them (K a multiple of 128; S and N up to 16,776,960). Returns y [S, N] bf16 (or writes
    ``out``, any row stride), or None when declined."""
    device, S, K, N, ldx, ldw = _int8_operands(x, x_scale, w, w_scale)
    if out is None:
        out = _empty(S, N, dtype=_BF16, device=device)
        ldy = N
    else:
        ldy = _rows("out", out, _BF16)
        if out.shape != (S, N):
            raise ValueError(f"out must be [{S}, {N}], got {tuple(out.shape)}")
        _require_same_device(device, out=out)
    rc = _run(L.lib().h3hip_proj_i8, device, x.data_ptr(), ldx, x_scale.data_ptr(), w.data_ptr(),
              ldw, w_scale.data_ptr(), K, N, S, out.data_ptr(), ldy)
    return None if rc == L.DECLINED else out


def qkv_proj_i8(x: torch.Tensor, x_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
                q_gamma: torch.Tensor | None = None, k_gamma: torch.Tensor | None = None,
                table: torch.Tensor | None = None, *, heads: int, head_dim: int = 128,
                eps: float = 1e-6, seq_pad: int | None = None,
                rounding: int = L.ROUND_REFERENCE, out=None):
    """qkv_proj() on int8 operands (x, x_scale, w, w_scale as for proj_i8(), w
    [3*heads*head_dim, hidden]): the QKV product with the Q/K norm + RoPE in its
    epilogue. ROUND_REFERENCE and ROUND_FP32 normalise the bf16 product, as qkv_proj()
    does; ROUND_ONCE keeps it in fp32 up to the one rounding of Q and K. Returns (q, k, v)
    as [heads, seq_pad, head_dim] bf16, or None when the geometry is declined."""
    device, S, K, N, ldx, ldw = _int8_operands(x, x_scale, w, w_scale)
    if N != 3 * heads * head_dim:
        raise ValueError(f"w must be [{3 * heads * head_dim}, {K}], got {tuple(w.shape)}")
    seq_pad = seq_pad or (S + L.TILE - 1) // L.TILE * L.TILE
    if q_gamma is None and k_gamma is None:
        rot, gq, gk, tab = head_dim, None, None, None
    else:
        rot = _check_norm_rope(device, S, head_dim, q_gamma, k_gamma, table, rounding)
        gq, gk, tab = q_gamma.data_ptr(), k_gamma.data_ptr(), table.data_ptr()
    shape = (heads, seq_pad, head_dim)
    if out is None:
        # One allocation: three take 2 us more of a call that can be as short as 20.
        out = _empty(3, heads, seq_pad, head_dim, dtype=_BF16, device=device).unbind(0)
    else:
        out = tuple(out)
        for t in out:
            _require_out(t, shape, device)
    q_out, k_out, v_out = out
    rc = _run(L.lib().h3hip_qkv_proj_i8, device, x.data_ptr(), ldx, x_scale.data_ptr(),
              w.data_ptr(), ldw, w_scale.data_ptr(), K, gq, gk, eps, tab, rot, rounding, S, seq_pad,
              heads, head_dim, q_out.data_ptr(), k_out.data_ptr(), v_out.data_ptr())
    return None if rc == L.DECLINED else out


def _check_norm_rope(device, S, head_dim, q_gamma, k_gamma, table, rounding) -> int:
    """Checks what the Q/K norm and rotation read; returns rot."""
    for name, t in (("q_gamma", q_gamma), ("k_gamma", k_gamma)):
        if (t is None or t.dtype is not _BF16 or t.shape != (head_dim,)
                or not t.is_contiguous() or t.device != device):
            raise ValueError(f"{name} must be contiguous bfloat16 [{head_dim}] on {device}")
    dt = _BF16 if rounding == L.ROUND_REFERENCE else _F32
    if (table is None or table.dtype is not dt or table.dim() != 4 or table.shape[0] < S
            or table.shape[2:] != (2, 2) or not table.is_contiguous() or table.device != device):
        raise ValueError(f"table must be a contiguous {dt} [>= {S}, rot/2, 2, 2] tensor on {device} "
                         "(rope_table() with the same rounding mode)")
    return 2 * table.shape[1]


# ------------------------------------------- microscaled 4-bit projections

_U8 = torch.uint8
MX4_BLOCK = 32                   # consecutive values of a row that share a scale


class Mx4Rows(NamedTuple):
    """Rows of microscaled 4-bit floats (MXFP4): what the 4-bit projections multiply.

    values: [S, cols padded to a multiple of 256, / 2] uint8, two values a byte, the earlier in
    the low half (row stride free). scale: [slabs, ceil(S/16), 64, 4] uint8, the blocks' biased
    exponents in the order in which the kernels read them: row r's and block b's at
    [b // 16, r // 16, 16 * (b % 4) + r % 16, b // 4 % 4]. cols: values of a row.
    quant_rows_mx4() makes them of bf16 rows, pack() of what a checkpoint holds, rows() of some of
    the rows (the scales belong to all rows from the first on: values alone are not sliced)."""
    values: torch.Tensor
    scale: torch.Tensor
    cols: int

    @property
    def shape(self):
        return self.values.shape[0], self.cols

    @classmethod
    def pack(cls, codes: torch.Tensor, exponents: torch.Tensor, cols: int | None = None):
        """Of row-major MXFP4 (codes [S, n/2] uint8, exponents [S, ceil(n/32)] uint8), laid out
        once; values past ``cols`` (n by default) become zeros."""
        if codes.dim() != 2 or codes.dtype != _U8 or codes.shape[1] == 0:
            raise ValueError(f"codes must be uint8 [S, n/2], got {codes.dtype} {tuple(codes.shape)}")
        S, n = codes.shape[0], 2 * codes.shape[1]
        blocks = (n + MX4_BLOCK - 1) // MX4_BLOCK
        if exponents.dtype != _U8 or tuple(exponents.shape) != (S, blocks):
            raise ValueError(f"exponents must be uint8 [{S}, {blocks}], got {exponents.dtype} "
                             f"{tuple(exponents.shape)}")
        _require_same_device(codes.device, exponents=exponents)
        cols = n if cols is None else cols
        if not 0 < cols <= n:
            raise ValueError(f"cols must be in 1..{n}, got {cols}")
        values = codes.new_zeros((S, (cols + 255) // 256 * 128))
        used = (cols + 1) // 2
        values[:, :used] = codes[:, :used]
        if cols % 2:
            values[:, used - 1] &= 15
        blocks, slabs, groups = (cols + MX4_BLOCK - 1) // MX4_BLOCK, (cols + 511) // 512, (S + 15) // 16
        rows = codes.new_zeros((16 * groups, 16 * slabs))
        rows[:S, :blocks] = exponents[:, :blocks]
        # [group, row, slab, byte, quarter] -> [slab, group, quarter, row, byte]
        scale = rows.view(groups, 16, slabs, 4, 4).permute(2, 0, 4, 1, 3)
        return cls(values, scale.reshape(slabs, groups, 64, 4).contiguous(), cols)

    def rows(self, first: int, count: int) -> "Mx4Rows":
        """Some of the rows (a weight's channels of one rank, a part of the tokens), from a
        multiple of 16 on: the values in place, their scales copied."""
        S = self.values.shape[0]
        if first % 16 or not 0 <= first <= first + count <= S:
            raise ValueError(f"rows must begin at a multiple of 16 and lie in 0..{S}, got {first} + "
                             f"{count}")
        scale = self.scale[:, first // 16:(first + count + 15) // 16].contiguous()
        return Mx4Rows(self.values[first:first + count], scale, self.cols)

    def exponents(self) -> torch.Tensor:
        """The biased exponents row-major, [S, ceil(cols/32)] uint8: what pack() takes."""
        slabs, groups = self.scale.shape[:2]
        rows = self.scale.view(slabs, groups, 4, 16, 4).permute(1, 3, 0, 4, 2)
        rows = rows.reshape(16 * groups, 16 * slabs)
        return rows[:self.values.shape[0], :(self.cols + MX4_BLOCK - 1) // MX4_BLOCK].contiguous()


def _bf16_rows(x: torch.Tensor):
    """Checks the bf16 rows that a call begins with; returns (stride, rows, columns, device)."""
    if x.dim() == 2 and x.dtype is _BF16 and x.is_cuda:
        (S, K), (ld, step) = x.shape, x.stride()
        if step == 1 and 0 < K <= _INT32_MAX and S <= _INT32_MAX:
            return (ld if S > 1 else K), S, K, x.device
    ld = _rows("x", x, _BF16)
    S, K = x.shape
    if K == 0:
        raise ValueError("x must be [S, K > 0]")
    if S > _INT32_MAX or K > _INT32_MAX:
        _require_int32("x", x)
    if not x.is_cuda:
        raise ValueError("x must be a GPU tensor (no host fallback exists)")
    return ld, S, K, x.device


def _mx4_sizes(S: int, K: int):
    """(bytes of a row of values, shape of the scales)."""
    return (K + 255) // 256 * 128, ((K + 511) // 512, (S + 15) // 16, 64, 4)


def _mx4_operand(name: str, t, device: torch.device | None = None):
    """Checks an Mx4Rows; returns (device, rows, bytes of a row, row stride in bytes)."""
    if not isinstance(t, Mx4Rows):
        raise ValueError(f"{name} must be an Mx4Rows (quant_rows_mx4() or Mx4Rows.pack()), "
                         f"got {type(t).__name__}")
    v, s, cols = t
    if v.dim() == 2 and v.dtype is _U8 and s.dtype is _U8 and v.is_cuda and 0 < cols <= _INT32_MAX:
        (S, n), (ld, step) = v.shape, v.stride()
        where = v.device
        if (S <= _INT32_MAX and n == (cols + 255) // 256 * 128 and step == 1
                and (device is None or where == device) and s.device == where
                and s.shape == ((cols + 511) // 512, (S + 15) // 16, 64, 4) and s.is_contiguous()):
            return where, S, n, (ld if S > 1 else n)
    ld = _rows(f"{name}.values", v, _U8)
    S, n = v.shape
    if S > _INT32_MAX or not 0 < cols <= _INT32_MAX:
        raise ValueError(f"{name} must have sizes from 1 to below 2^31, got {S} x {cols}")
    width, shape = _mx4_sizes(S, cols)
    if n != width:
        raise ValueError(f"{name}.values must be [{S}, {width}] for {cols} columns, got "
                         f"{tuple(v.shape)}")
    if s.dtype is not _U8 or s.shape != shape or not s.is_contiguous():
        raise ValueError(f"{name}.scale must be contiguous uint8 {shape}, got {s.dtype} "
                         f"{tuple(s.shape)}")
    if not v.is_cuda:
        raise ValueError(f"{name} must be on a GPU (no host fallback exists)")
    device = v.device if device is None else device
    if v.device != device or s.device != device:
        raise ValueError(f"{name} must be on {device}, got {v.device} and {s.device}")
    return device, S, n, ld


def quant_rows_mx4(x: torch.Tensor, out: Mx4Rows | None = None) -> Mx4Rows:
    """Rows of bf16 rounded to 4-bit floats, a power of two for every 32 consecutive values.

    x: [S, K] bf16 (row stride free, unit column stride): the activations of a 4-bit
    projection, or its weights, rounded once. A block holding an infinity or a NaN gets the
    scale NaN. ``out`` is an Mx4Rows of these sizes to write into."""
    ldx, S, K, device = _bf16_rows(x)
    if out is None:
        ldq = (K + 255) // 256 * 128
        out = Mx4Rows(_empty(S, ldq, dtype=_U8, device=device),
                      _empty((K + 511) // 512, (S + 15) // 16, 64, 4, dtype=_U8, device=device), K)
    else:
        _, rows, _, ldq = _mx4_operand("out", out, device)
        if (rows, out.cols) != (S, K):
            raise ValueError(f"out must hold [{S}, {K}], got {out.shape}")
    _run(L.lib().h3hip_quant_rows_mx4, device, x.data_ptr(), ldx, S, K, out.values.data_ptr(), ldq,
         out.scale.data_ptr())
    return out


def dequant_rows_mx4(rows: Mx4Rows, out: torch.Tensor | None = None) -> torch.Tensor:
    """The values that 4-bit rows stand for, [S, cols] bf16, exactly."""
    device, S, _, ldq = _mx4_operand("rows", rows)
    values, scale, cols = rows
    if out is None:
        out, ldx = _empty(S, cols, dtype=_BF16, device=device), cols
    else:
        ldx = _rows("out", out, _BF16)
        if out.shape != (S, cols):
            raise ValueError(f"out must be [{S}, {cols}], got {tuple(out.shape)}")
        _require_same_device(device, out=out)
    _run(L.lib().h3hip_dequant_rows_mx4, device, values.data_ptr(), ldq, scale.data_ptr(), S, cols,
         out.data_ptr(), ldx)
    return out


@functools.lru_cache(maxsize=1024)
def _mx4_workspace(S: int, K: int) -> int:
    return L.lib().h3hip_linear_mx4_workspace(S, K)


def _mx4_operands(x, w):
    """Checks the operands of a 4-bit product, x in bf16 or an Mx4Rows; returns
    (device, S, N, x's row stride, w's)."""
    bf16 = isinstance(x, torch.Tensor)
    if type(w) is Mx4Rows and (bf16 or type(x) is Mx4Rows):
        v, s, K = w
        xv = x if bf16 else x.values
        if v.dim() == xv.dim() == 2:
            (S, k), (N, n) = xv.shape, v.shape
            (ldx, step), (ldw, step_w) = xv.stride(), v.stride()
            device = xv.device
            # The common case in one test (2 us less of a call that can be as short as 10); what
            # of it is refused, one by one, below.
            if (0 < K <= _INT32_MAX and S <= _INT32_MAX and N <= _INT32_MAX
                    and n == (K + 255) // 256 * 128 and v.dtype is _U8 and s.dtype is _U8
                    and step == 1 and step_w == 1 and s.is_contiguous() and xv.is_cuda
                    and v.device == device and s.device == device
                    and s.shape == ((K + 511) // 512, (N + 15) // 16, 64, 4)
                    and (k == K and xv.dtype is _BF16 if bf16 else
                         k == n and x.cols == K and _mx4_operand("x", x, device))):
                return device, S, N, (ldx if S > 1 else (k + 15) // 16 * 16), (ldw if N > 1 else n)
    if bf16:
        ldx = _rows("x", x, _BF16)
        device, N, _, ldw = _mx4_operand("w", w)
        if x.shape[1] != w.cols:
            raise ValueError(f"x must be [S, {w.cols}], got {tuple(x.shape)}")
        if x.shape[0] > _INT32_MAX:
            _require_int32("x", x)
        _require_same_device(device, x=x)
        return device, x.shape[0], N, ldx, ldw
    device, S, _, ldx = _mx4_operand("x", x)
    _, N, _, ldw = _mx4_operand("w", w, device)
    if x.cols != w.cols:
        raise ValueError(f"w must hold [out, {x.cols}], got {w.shape}")
    return device, S, N, ldx, ldw


def proj_mx4(x: torch.Tensor | Mx4Rows, w: Mx4Rows, out: torch.Tensor | None = None):
    """A projection on 4-bit operands: y = x . w^T with fp32 sums.

    x: [S, K] bf16 (row stride free), rounded as by quant_rows_mx4() on the way, or an
    Mx4Rows; w: [N, K], rounded or laid out once (S, N and K up to 16,776,960). One or two bf16
    rows take one launch, whose sums add in another order than those of more. Returns y [S, N]
    bf16 (or writes ``out``, any row stride; not on top of one or two rows of x), or None when
    declined."""
    device, S, N, ldx, ldw = _mx4_operands(x, w)
    if out is None:
        out = _empty(S, N, dtype=_BF16, device=device)
        ldy = N
    else:
        ldy = _rows("out", out, _BF16)
        if out.shape != (S, N):
            raise ValueError(f"out must be [{S}, {N}], got {tuple(out.shape)}")
        _require_same_device(device, out=out)
    v, s, K = w
    if type(x) is Mx4Rows:
        rc = _run(L.lib().h3hip_proj_mx4, device, x.values.data_ptr(), ldx, x.scale.data_ptr(),
                  v.data_ptr(), ldw, s.data_ptr(), 2 * v.shape[1], N, S, out.data_ptr(), ldy)
    else:
        size, work = _mx4_workspace(S, K), None
        if size:
            work = _empty(size, dtype=_U8, device=device)
        rc = _run(L.lib().h3hip_linear_mx4, device, x.data_ptr(), ldx, v.data_ptr(), ldw,
                  s.data_ptr(), K, N, S, out.data_ptr(), ldy, work.data_ptr() if size else None, size)
    return None if rc == L.DECLINED else out


def qkv_proj_mx4(x: torch.Tensor | Mx4Rows, w: Mx4Rows, q_gamma: torch.Tensor | None = None,
                 k_gamma: torch.Tensor | None = None, table: torch.Tensor | None = None, *,
                 heads: int, head_dim: int = 128, eps: float = 1e-6, seq_pad: int | None = None,
                 rounding: int = L.ROUND_REFERENCE, out=None):
    """qkv_proj() on 4-bit operands (x and w as for proj_mx4(), w [3*heads*head_dim, hidden]):
    the QKV product with the Q/K norm + RoPE in its epilogue. ROUND_REFERENCE and ROUND_FP32
    normalise the bf16 product, as qkv_proj() does; ROUND_ONCE keeps it in fp32 up to the one
    rounding of Q and K. Returns (q, k, v) as [heads, seq_pad, head_dim] bf16, or None when the
    geometry is declined."""
    device, S, N, ldx, ldw = _mx4_operands(x, w)
    if N != 3 * heads * head_dim:
        raise ValueError(f"w must hold [{3 * heads * head_dim}, {w.cols}], got {w.shape}")
    seq_pad = seq_pad or (S + L.TILE - 1) // L.TILE * L.TILE
    if q_gamma is None and k_gamma is None:
        rot, gq, gk, tab = head_dim, None, None, None
    else:
        rot = _check_norm_rope(device, S, head_dim, q_gamma, k_gamma, table, rounding)
        gq, gk, tab = q_gamma.data_ptr(), k_gamma.data_ptr(), table.data_ptr()
    shape = (heads, seq_pad, head_dim)
    if out is None:
        out = _empty(3, heads, seq_pad, head_dim, dtype=_BF16, device=device).unbind(0)
    else:
        out = tuple(out)
        for t in out:
            _require_out(t, shape, device)
    q, k, o = out
    v, s, K = w
    norm = (gq, gk, eps, tab, rot, rounding, S, seq_pad, heads, head_dim, q.data_ptr(),
            k.data_ptr(), o.data_ptr())
    if type(x) is Mx4Rows:
        rc = _run(L.lib().h3hip_qkv_proj_mx4, device, x.values.data_ptr(), ldx, x.scale.data_ptr(),
                  v.data_ptr(), ldw, s.data_ptr(), 2 * v.shape[1], *norm)
    else:
        size, work = _mx4_workspace(S, K), None
        if size:
            work = _empty(size, dtype=_U8, device=device)
        rc = _run(L.lib().h3hip_qkv_linear_mx4, device, x.data_ptr(), ldx, v.data_ptr(), ldw,
                  s.data_ptr(), K, *norm, work.data_ptr() if size else None, size)
    return None if rc == L.DECLINED else out


# -------------------------------------- norm, modulation, gate and residual

NORM_MAX_HIDDEN = 16384          # widths that a workgroup's registers hold


def _norm_rows(name: str, t: torch.Tensor, S: int, hidden: int, device) -> int:
    """Checks bf16 rows of a norm; returns their stride."""
    if t.dtype is _BF16 and t.device == device and t.shape == (S, hidden):
        ld, step = t.stride()
        if step == 1:
            return ld if S > 1 else hidden
    ld = _rows(name, t, _BF16)
    if t.shape != (S, hidden):
        raise ValueError(f"{name} must be [{S}, {hidden}], got {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}, got {t.device}")
    return ld


def _norm_gamma(name: str, t, hidden: int, device):
    if t is None:
        return None
    if t.dtype is not _BF16 or t.shape != (hidden,) or not t.is_contiguous() or t.device != device:
        raise ValueError(f"{name} must be contiguous bfloat16 [{hidden}] on {device}")
    return t.data_ptr()


def _norm_table(name: str, t, segments: int, hidden: int, device):
    """(address, row stride) of a modulation [segments, hidden] or, of one segment, [hidden]."""
    if t is None:
        return None, hidden
    if (t.dtype is _BF16 and t.device == device
            and (t.shape == (segments, hidden) or (segments == 1 and t.shape == (hidden,)))
            and (t.stride(-1) == 1 or hidden == 1)):
        return t.data_ptr(), (t.stride(0) if segments > 1 else hidden)
    raise ValueError(f"{name} must be bfloat16 [{segments}, {hidden}] on {device} with unit column "
                     f"stride, got {t.dtype} {tuple(t.shape)} on {t.device}")


def _norm_c(gamma, scale, shift, segments, hidden, device) -> L.NormC:
    # All three, contiguous, in one test (0.5 us less of a call that can be as short as 8); what
    # of it is missing or refused, one by one.
    if (gamma is not None and scale is not None and shift is not None
            and gamma.dtype is _BF16 and scale.dtype is _BF16 and shift.dtype is _BF16
            and gamma.device == device and scale.device == device and shift.device == device
            and gamma.shape == (hidden,) and scale.shape == shift.shape == (segments, hidden)
            and gamma.is_contiguous() and scale.is_contiguous() and shift.is_contiguous()):
        return L.NormC(gamma.data_ptr(), scale.data_ptr(), shift.data_ptr(), hidden, hidden)
    scale, ld_scale = _norm_table("scale", scale, segments, hidden, device)
    shift, ld_shift = _norm_table("shift", shift, segments, hidden, device)
    return L.NormC(_norm_gamma("gamma", gamma, hidden, device), scale, shift, ld_scale, ld_shift)


_Starts = [ctypes.c_int32 * n for n in range(17)]


def _segments(starts):
    """(host array or None, how many) of the segments' first rows."""
    if starts is None:
        return None, 1
    n = len(starts)
    if n == 1 and starts[0] == 0:
        return None, 1
    if not 1 <= n <= 16:
        raise ValueError(f"segments must be 1 to 16 first rows, got {n}")
    if min(starts) < 0 or max(starts) > _INT32_MAX:
        raise ValueError(f"segments must be rows from 0 to below 2^31, got {list(starts)}")
    return _Starts[n](*map(int, starts)), n


def norm_modulate(x: torch.Tensor, gamma: torch.Tensor | None = None,
                  scale: torch.Tensor | None = None, shift: torch.Tensor | None = None, *,
                  segments=None, eps: float = 1e-6, out: torch.Tensor | None = None):
    """The norm before a block: x rsqrt(mean x^2 + eps) gamma (1 + scale[s]) + shift[s].

    x: [S, hidden] bf16 (row stride free). gamma: [hidden]; scale, shift: [segments, hidden] bf16
    (or [hidden], of one segment), each optional. segments: the first row of each, not
    descending, from 0 on (None: one segment). Returns h [S, hidden] bf16 (or writes ``out``, any
    row stride; x itself is allowed), or None when declined (hidden above 16,384)."""
    ldx, S, hidden, device = _bf16_rows(x)
    starts, n = (None, 1) if segments is None else _segments(segments)
    norm = _norm_c(gamma, scale, shift, n, hidden, device)
    if out is None:
        out, ldh = _empty(S, hidden, dtype=_BF16, device=device), hidden
    else:
        ldh = _norm_rows("out", out, S, hidden, device)
    rc = _run(L.lib().h3hip_norm_modulate, device, x.data_ptr(), ldx, S, hidden, norm, eps, starts,
              n, out.data_ptr(), ldh)
    return None if rc == L.DECLINED else out


def gated_residual(x: torch.Tensor, y: torch.Tensor, gate: torch.Tensor | None = None, *,
                   post_gamma: torch.Tensor | None = None, residual_scale: float = 1.0,
                   segments=None, eps: float = 1e-6, next_norm: dict | None = None, out=None):
    """The end of a block's half: r = residual_scale x + gate[s] z, z being y or, with
    post_gamma, y rsqrt(mean y^2 + eps) post_gamma.

    x, y: [S, hidden] bf16 (row strides free); gate: [segments, hidden] bf16 (or [hidden], of one
    segment) or None (1); segments as for norm_modulate(). next_norm: a dict of the gamma,
    scale and shift (any of them) of the norm that the next half begins with; it is taken of r
    before r is rounded. Returns r, with next_norm (r, h), [S, hidden] bf16 each, or None when
    declined (hidden above 16,384). ``out`` is r, or (r, h), to write into: any row stride, x or
    y themselves are allowed."""
    ldx, S, hidden, device = _bf16_rows(x)
    ldy = _norm_rows("y", y, S, hidden, device)
    starts, n = (None, 1) if segments is None else _segments(segments)
    gate, ld_gate = _norm_table("gate", gate, n, hidden, device)
    post = _norm_gamma("post_gamma", post_gamma, hidden, device)
    norm = h = None
    ldh = hidden
    if next_norm is not None:
        wrong = set(next_norm) - {"gamma", "scale", "shift"}
        if wrong:
            raise ValueError(f"next_norm takes gamma, scale and shift, got {sorted(wrong)}")
        norm = _norm_c(next_norm.get("gamma"), next_norm.get("scale"), next_norm.get("shift"), n,
                       hidden, device)
    if out is None:
        r, ldr = _empty(S, hidden, dtype=_BF16, device=device), hidden
        if norm is not None:
            h = _empty(S, hidden, dtype=_BF16, device=device)
    else:
        r, h = out if norm is not None else (out, None)
        ldr = _norm_rows("out", r, S, hidden, device)
        if h is not None:
            ldh = _norm_rows("out[1]", h, S, hidden, device)
    rc = _run(L.lib().h3hip_gated_residual, device, x.data_ptr(), ldx, y.data_ptr(), ldy, S, hidden,
              gate, ld_gate, post, residual_scale, norm, eps, starts, n, r.data_ptr(), ldr,
              None if h is None else h.data_ptr(), ldh)
    if rc == L.DECLINED:
        return None
    return r if norm is None else (r, h)


# -------------------------------------------------------------------- attention

def _head_major_qkv(plan: TilePlan, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor):
    """q, k, v must be contiguous bf16 GPU tensors of one shape [H, seq_pad, D]:
    the kernel reads all H heads x D columns x seq_len rows of each. Returns (H, D).
    (A head count or head_dim the library does not take is declined by the library
    before anything is read.)"""
    for name, t in (("q", q), ("k", k), ("v", v)):
        if not t.is_contiguous() or t.dim() != 3 or t.shape[1] != plan.seq_pad:
            raise ValueError(f"{name} must be contiguous [heads, {plan.seq_pad}, head_dim], "
                             f"got shape {tuple(t.shape)}")
    if k.shape != q.shape or v.shape != q.shape:
        raise ValueError(f"q, k and v must have one shape, got {tuple(q.shape)}, "
                         f"{tuple(k.shape)}, {tuple(v.shape)}")
    for name, t in (("q", q), ("k", k), ("v", v)):
        _require_gpu_bf16(name, t)
    return q.shape[0], q.shape[2]


def _require_out(out: torch.Tensor, shape, device):
    if (not isinstance(out, torch.Tensor) or out.dtype != torch.bfloat16 or out.device != device
            or not out.is_contiguous() or tuple(out.shape) != tuple(shape)):
        raise ValueError(f"out must be a contiguous bf16 tensor of shape {tuple(shape)} on "
                         f"{device}, got {getattr(out, 'shape', None)}")


def bsattn_fwd(plan: TilePlan, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
               scale: float | None = None, out_layout: int = L.OUT_HEAD_MAJOR,
               out: torch.Tensor | None = None):
    """Block-sparse attention over the plan's tiles; q/k/v [H, seq_pad, D] bf16.

    Returns the output tensor, or None when the call is declined."""
    H, D = _head_major_qkv(plan, q, k, v)
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    if out_layout not in (L.OUT_HEAD_MAJOR, L.OUT_TOKEN_MAJOR):
        raise ValueError(f"unknown out_layout {out_layout}")
    shape = (H, plan.seq_pad, D) if out_layout == L.OUT_HEAD_MAJOR else (plan.seq_pad, H * D)
    if out is None:
        out = torch.empty(shape, dtype=torch.bfloat16, device=q.device)
    else:
        _require_out(out, shape, q.device)
    rc = L.lib().h3hip_bsattn_fwd(plan.handle, _ptr(q), _ptr(k), _ptr(v), H, D, scale,
                                  _ptr(out), out_layout, _stream(q))
    if L.check(rc, allow_declined=True) == L.DECLINED:
        return None
    return out


def _views(q, k, v, out, S):
    """[heads, rows, head_dim] tensors -> h3hip_views (strides in elements). The
    kernel touches every head and all head_dim columns of rows < S of each, so
    every view must hold q's head count and head_dim and at least S rows."""
    if q.dim() != 3:
        raise ValueError(f"q must be a [heads, rows, head_dim] view, got shape {tuple(q.shape)}")
    H, _, D = q.shape
    named = (("q", q), ("k", k), ("v", v), ("out", out))
    for name, t in named:
        if (t.dim() != 3 or t.stride(2) != 1 or t.shape[0] != H or t.shape[2] != D
                or t.shape[1] < S):
            raise ValueError(f"{name} must be a [{H}, >= {S}, {D}] view with unit stride along "
                             f"head_dim, got shape {tuple(t.shape)} strides {t.stride()}")
    for name, t in named:
        _require_gpu_bf16(name, t)
    return [L.ViewC(t.data_ptr(), t.stride(0), t.stride(1)) for _, t in named]


def bsattn_fwd_strided(plan: TilePlan, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                       scale: float | None = None, out: torch.Tensor | None = None):
    """Block-sparse attention on strided [heads, rows, head_dim] views.

    q, k, v may be views straight into a fused token-major projection (e.g.
    ``qkv.view(S, 3, H, D)[:, 2].transpose(0, 1)`` for V); only rows < S are
    read. ``out`` is a [heads, >= S, head_dim] view to write rows < S into;
    by default a token-major [S, heads*head_dim] tensor is allocated and
    returned. Returns None when the call is declined."""
    S = plan.seq_len
    if q.dim() != 3:
        raise ValueError(f"q must be a [heads, rows, head_dim] view, got shape {tuple(q.shape)}")
    H, _, D = q.shape
    ret = None
    if out is None:
        ret = torch.empty((S, H * D), dtype=torch.bfloat16, device=q.device)
        out = ret.view(S, H, D).transpose(0, 1)
    views = _views(q, k, v, out, S)
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    rc = L.lib().h3hip_bsattn_fwd_strided(plan.handle, ctypes.byref(views[0]),
                                          ctypes.byref(views[1]), ctypes.byref(views[2]), H, D,
                                          scale, ctypes.byref(views[3]), _stream(q))
    if L.check(rc, allow_declined=True) == L.DECLINED:
        return None
    return ret if ret is not None else out


def attend_strided(plan: TilePlan, context, q: torch.Tensor, k: torch.Tensor,
                   v: torch.Tensor, scale: float, out: torch.Tensor | None = None):
    """h3hip_attend_strided: policy + geometry checks, then the sparse kernel
    on [heads, rows, head_dim] views (rows >= S; unit stride along head_dim).

    ``out`` is a [heads, >= S, head_dim] view; by default a token-major
    [S, heads*head_dim] buffer is allocated and its [heads, S, head_dim] view
    returned. Returns None when the call is declined."""
    S = plan.seq_len
    if q.dim() != 3:
        raise ValueError(f"q must be a [heads, rows, head_dim] view, got shape {tuple(q.shape)}")
    H, _, D = q.shape
    if out is None:
        out = torch.empty((S, H * D), dtype=torch.bfloat16, device=q.device)
        out = out.view(S, H, D).transpose(0, 1)
    views = _views(q, k, v, out, S)
    cctx = None if context is None else ctypes.byref(context.to_c())
    rc = L.lib().h3hip_attend_strided(plan.handle, cctx, ctypes.byref(views[0]),
                                      ctypes.byref(views[1]), ctypes.byref(views[2]), H, D,
                                      scale, ctypes.byref(views[3]), _stream(q))
    if L.check(rc, allow_declined=True) == L.DECLINED:
        return None
    return out


def attend(plan: TilePlan, context, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
           scale: float, out: torch.Tensor | None = None):
    """h3hip_attend: policy + geometry checks, then the sparse kernel.

    ``context`` is an AttentionContext (or None, which declines). q, k, v are
    contiguous [heads, seq_pad, head_dim] like bsattn_fwd's; a given ``out``
    must be contiguous [heads, seq_pad, head_dim] bf16."""
    H, D = _head_major_qkv(plan, q, k, v)
    if out is None:
        out = torch.empty((H, plan.seq_pad, D), dtype=torch.bfloat16, device=q.device)
    else:
        _require_out(out, (H, plan.seq_pad, D), q.device)
    cctx = None if context is None else ctypes.byref(context.to_c())
    rc = L.lib().h3hip_attend(plan.handle, cctx, _ptr(q), _ptr(k), _ptr(v), H, D, scale,
                              _ptr(out), _stream(q))
    if L.check(rc, allow_declined=True) == L.DECLINED:
        return None
    return out
