"""AttentionLayer of the DiT block on MI355X (Sources/H3Modules/DiTBlock.swift).

Mirrors ``AttentionLayer.callAsFunction(_:ropeTable:context:)`` (:336-359):

    qkv = matmul(x, qkvWeight.T); q, k, v = split(qkv)          (:338-344)
    q = qNorm(q); k = kNorm(k)                                   (:346-347)
    if ropeTable: q, k = SplitHalfRoPE.apply(q/k, ropeTable)     (:348-351)
    merged = sdpa(q, k, v, context)                              (:356-357)
    return matmul(merged, outWeight.T)                           (:358)

with the projection and the norm/RoPE either fused in one kernel
(h3hip_qkv_proj) or run as hipBLASLt's GEMM followed by the prologue kernel
(h3hip_qk_norm_rope), the attention through the backend seam (block-sparse
kernel with a context, the reference's dense SDPA otherwise), and the
out-projection -- a plain GEMM -- on the projection kernel's main loop
(h3hip_out_proj), or on hipBLASLt when that kernel declines the shape. Q and K
come out head-major and V is read in place, so no relayout copy runs between
the stages.

With ``projection="int8"`` both projections run on int8 operands with scales for
each token and output channel (h3hip_quant_rows, h3hip_qkv_proj_i8,
h3hip_proj_i8): the weights are rounded once, the activations in every call. A
RopeState of ROUND_ONCE keeps Q and K in fp32 from that product to their store.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from . import _lib as L
from . import ops
from .backend import AttentionContext, H3AttentionBackend


@dataclass
class RopeState:
    """The render's rotation state (H3Transformer.swift:263-276, built once per
    render): the rotation table H3RoPE.rotationTable -- the ``ropeTable`` every
    layer takes -- and the (positions, pair) tables it comes from. The fused
    projection rotates with the table, the prologue kernel re-evaluates the same
    entries from the pair tables; both give the same bits."""
    pos: torch.Tensor          # [S, 3] fp32 (t, h, w)
    pair_axis: torch.Tensor    # [rot/2] int32
    pair_inv: torch.Tensor     # [rot/2] fp32
    rot: int
    rounding: int
    table: torch.Tensor        # [S, rot/2, 2, 2], bf16 (REFERENCE) or fp32

    @classmethod
    def build(cls, pos, pair_axis, pair_inv, rot: int | None = None,
              rounding: int = L.ROUND_REFERENCE) -> "RopeState":
        rot = rot if rot is not None else 2 * pair_axis.numel()
        table = ops.rope_table(pos, pair_axis, pair_inv, rot=rot, rounding=rounding)
        return cls(pos, pair_axis, pair_inv, rot, rounding, table)

    @classmethod
    def identity(cls, seq_len: int, head_dim: int, device,
                 rounding: int = L.ROUND_REFERENCE) -> "RopeState":
        """Position 0 everywhere: the rotation is the identity, bit for bit in
        both rounding modes -- the layer without a ropeTable."""
        pos = torch.zeros((seq_len, 3), dtype=torch.float32, device=device)
        half = head_dim // 2
        axis = torch.zeros(half, dtype=torch.int32, device=device)
        inv = torch.ones(half, dtype=torch.float32, device=device)
        return cls.build(pos, axis, inv, head_dim, rounding)


@dataclass
class Int8Weight:
    """A projection's weight rounded to int8 once: [out, in padded to a multiple of 128]
    int8 rows with an fp32 scale each."""
    values: torch.Tensor
    scale: torch.Tensor
    in_features: int

    @classmethod
    def round(cls, weight: torch.Tensor) -> "Int8Weight":
        """weight: [out, in] bf16 on the GPU."""
        return cls(*ops.quant_rows(weight), weight.shape[1])

    @property
    def shape(self):
        return self.values.shape[0], self.in_features


class AttentionLayer:
    """One DiT attention layer (DiTBlock.swift:262-359).

    qkv_weight: [3*heads*head_dim, hidden] bf16 (Q | K | V rows, as stored);
    out_weight: [hidden, heads*head_dim] bf16; q_gamma, k_gamma: [head_dim] bf16
    (qNorm, kNorm). ``projection`` picks the QKV path: "fused" (h3hip_qkv_proj)
    or "hipblaslt" (GEMM + h3hip_qk_norm_rope); either falls back to the other
    when its kernel declines the geometry. "int8" runs both projections on int8
    operands (qkv_weight and out_weight are rounded here, or given as Int8Weight;
    the bf16 ones are not kept, so nothing is fallen back to), of at most
    ops.INT8_MAX_REDUCTION in features, padded to a multiple of 128."""

    def __init__(self, qkv_weight, out_weight, q_gamma, k_gamma, *, heads: int,
                 head_dim: int = 128, eps: float = 1e-5, backend: H3AttentionBackend | None = None,
                 projection: str = "hipblaslt"):
        if projection not in ("fused", "hipblaslt", "int8"):
            raise ValueError("projection must be 'fused', 'hipblaslt' or 'int8', got "
                             f"{projection!r}")
        inner = heads * head_dim
        if qkv_weight.shape[0] != 3 * inner or out_weight.shape[1] != inner:
            raise ValueError("weights do not match heads * head_dim")
        if projection == "int8":
            for name, w in (("qkv_weight", qkv_weight), ("out_weight", out_weight)):
                if (w.shape[1] + 127) // 128 * 128 > ops.INT8_MAX_REDUCTION:
                    raise NotImplementedError(
                        f"no int8 kernel takes {name}'s {w.shape[1]} in features (at most "
                        f"{ops.INT8_MAX_REDUCTION}, padded to a multiple of 128)")
            qkv_weight, out_weight = (w if isinstance(w, Int8Weight) else Int8Weight.round(w)
                                      for w in (qkv_weight, out_weight))
        elif isinstance(qkv_weight, Int8Weight) or isinstance(out_weight, Int8Weight):
            raise ValueError("an Int8Weight needs projection='int8'")
        self.qkv_weight, self.out_weight = qkv_weight, out_weight
        self.q_gamma, self.k_gamma = q_gamma, k_gamma
        self.heads, self.head_dim, self.eps = heads, head_dim, eps
        self.backend, self.projection = backend, projection

    # ---------------------------------------------------------------- stages

    def _project_fused(self, x, rope: RopeState, seq_pad: int):
        r = ops.qkv_proj(x, self.qkv_weight, self.q_gamma, self.k_gamma, rope.table,
                         heads=self.heads, head_dim=self.head_dim, eps=self.eps,
                         seq_pad=seq_pad, rounding=rope.rounding)
        if r is None:
            return None
        q, k, v = r
        S = x.shape[0]
        return q[:, :S], k[:, :S], v[:, :S]

    def _project_hipblaslt(self, x, rope: RopeState, seq_pad: int):
        S, inner = x.shape[0], self.heads * self.head_dim
        qkv = torch.mm(x, self.qkv_weight.t())
        r = ops.qk_norm_rope(qkv[:, :inner], qkv[:, inner:2 * inner], self.q_gamma,
                             self.k_gamma, rope.pos, rope.pair_axis, rope.pair_inv,
                             heads=self.heads, head_dim=self.head_dim, eps=self.eps, rot=rope.rot,
                             seq_pad=seq_pad, rounding=rope.rounding)
        if r is None:
            return None
        v = qkv[:, 2 * inner:].view(S, self.heads, self.head_dim).transpose(0, 1)
        return r[0][:, :S], r[1][:, :S], v

    def _project_int8(self, x, rope: RopeState, seq_pad: int):
        w, S = self.qkv_weight, x.shape[0]
        r = ops.qkv_proj_i8(*ops.quant_rows(x), w.values, w.scale, self.q_gamma, self.k_gamma,
                            rope.table, heads=self.heads, head_dim=self.head_dim, eps=self.eps,
                            seq_pad=seq_pad, rounding=rope.rounding)
        return None if r is None else tuple(t[:, :S] for t in r)

    def _attend(self, q, k, v, context: AttentionContext | None):
        """AttentionLayer.sdpa (DiTBlock.swift:280-328) on [H, S, D] views:
        the backend only with a context; a decline runs dense SDPA."""
        H, S, D = q.shape
        scale = 1.0 / math.sqrt(D)
        if self.backend is not None and context is not None:
            o = self.backend.attend(q, k, v, scale, None, context)
            if o is not None:
                return o.transpose(0, 1).reshape(S, H * D)
        # Dense: computed in fp32 one head at a time (at least as accurate as
        # a bf16 SDPA, which accumulates in fp32; keeps torch off its bf16
        # batched-product path; one [S, S] score matrix at a time), rounded to
        # the input dtype as the reference's sdpa returns it.
        out = torch.empty((S, H, D), dtype=q.dtype, device=q.device)
        for h in range(H):
            o = torch.nn.functional.scaled_dot_product_attention(
                q[h][None].float(), k[h][None].float(), v[h][None].float(), scale=scale)
            out[:, h] = o[0].to(q.dtype)
        return out.reshape(S, H * D)

    # ------------------------------------------------------------------ call

    def __call__(self, x: torch.Tensor, rope: RopeState | None,
                 context: AttentionContext | None = None) -> torch.Tensor:
        """x: [S, hidden] bf16 -> [S, hidden] bf16."""
        if x.dim() != 2 or x.shape[1] != self.qkv_weight.shape[1]:
            raise ValueError(f"x must be [S, {self.qkv_weight.shape[1]}] (the packed-row layout), "
                             f"got {tuple(x.shape)}")
        S = x.shape[0]
        if rope is not None and rope.rounding == L.ROUND_ONCE and self.projection != "int8":
            raise ValueError("ROUND_ONCE needs projection='int8'")
        if rope is None:
            rope = RopeState.identity(S, self.head_dim, x.device)
        seq_pad = ((S + L.TILE - 1) // L.TILE) * L.TILE
        paths = {"fused": (self._project_fused, self._project_hipblaslt),
                 "hipblaslt": (self._project_hipblaslt, self._project_fused),
                 "int8": (self._project_int8,)}[self.projection]
        qkv = None
        for project in paths:
            qkv = qkv or project(x, rope, seq_pad)
        if qkv is None:
            raise NotImplementedError(
                f"no kernel takes head_dim {self.head_dim} / rot {rope.rot} / heads {self.heads}")
        merged = self._attend(*qkv, context)
        if self.projection == "int8":
            return ops.proj_i8(*ops.quant_rows(merged), self.out_weight.values,
                               self.out_weight.scale)
        y = ops.out_proj(merged, self.out_weight)
        if y is None:       # a width the kernel declines: hipBLASLt's GEMM
            y = torch.mm(merged, self.out_weight.t())
        return y
