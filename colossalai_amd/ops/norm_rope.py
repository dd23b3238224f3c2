"""Normed and rotated query and key heads of a packed projection (``csrc/norm_rope.hip``).

``qkv_norm_rope`` splits ``[q | k | v]``, divides each query and key head by its root mean square, multiplies it by a
weight that the heads share and rotates it by its position (pairs ``(i, i + D / 2)``, the tables of ``build_rope_table``), in one
pass over the data; the values are copied. Its backward is one pass too and leaves the projection's gradient packed, with
the weights' gradients beside it. Statistics, angles and sums are float32, and a result is rounded to its type once; the
separate operators (``rms_norm``, then ``apply_rope``) round between them as well.
"""

from typing import Optional, Tuple

import torch

from ._kernels import kernels, native_function, use_hip

__all__ = ["qkv_norm_rope", "qkv_norm_rope_ref", "norm_rope_ref"]

_TYPES = (torch.bfloat16, torch.float16, torch.float32)


def norm_rope_ref(x: torch.Tensor, weight: Optional[torch.Tensor], table: torch.Tensor, positions: torch.Tensor, eps: float,
                  dtype=torch.float32) -> torch.Tensor:
    """x [.., H, D] with positions [..]: normed if there is a weight, and rotated, in ``dtype``. A position that the table does not have
    gives NaN."""
    y = x.to(dtype)
    if weight is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps) * weight.to(dtype)
    here = (positions >= 0) & (positions < table.shape[0])
    if table.shape[0] == 0:
        table = table.new_zeros(1, table.shape[1])
    rows = table.to(dtype)[torch.where(here, positions, 0).long()].masked_fill(~here.unsqueeze(-1), float("nan"))
    cos, sin = rows.unsqueeze(-2).chunk(2, -1)
    lo, hi = y.chunk(2, -1)
    return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)


def qkv_norm_rope_ref(qkv, q_weight, k_weight, table, num_heads, num_kv_heads, positions=None, eps=1e-6):
    B, S, _ = qkv.shape
    heads = qkv.reshape(B, S, num_heads + 2 * num_kv_heads, q_weight.numel())
    q, k, v = heads.split([num_heads, num_kv_heads, num_kv_heads], 2)
    at = torch.arange(S, device=qkv.device).expand(B, S) if positions is None else positions.reshape(B, S)
    return (norm_rope_ref(q, q_weight, table, at, eps).to(qkv.dtype), norm_rope_ref(k, k_weight, table, at, eps).to(qkv.dtype),
            v.contiguous())


class _NormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, q_weight, k_weight, table, num_heads, num_kv_heads, positions, eps):
        ctx.save_for_backward(qkv, q_weight, k_weight, table, positions)
        ctx.rest = num_heads, num_kv_heads, eps
        return tuple(kernels().norm_rope_fwd(qkv, q_weight, k_weight, table, positions, num_heads, num_kv_heads, eps))

    @staticmethod
    def backward(ctx, dq, dk, dv):
        qkv, q_weight, k_weight, table, positions = ctx.saved_tensors
        num_heads, num_kv_heads, eps = ctx.rest
        if torch.is_grad_enabled():  # the gradient is part of a graph itself: the kernel's result would end it
            of = [qkv, q_weight, k_weight]
            to = [t for t in of if t.requires_grad]
            pairs = [(y, g) for y, g in zip(qkv_norm_rope_ref(qkv, q_weight, k_weight, table, num_heads, num_kv_heads, positions, eps),
                                            (dq, dk, dv)) if y.requires_grad]
            got = iter(torch.autograd.grad([y for y, _ in pairs], to, [g for _, g in pairs], create_graph=True, allow_unused=True))
            return tuple(next(got) if t.requires_grad else None for t in of) + (None,) * 5
        return tuple(kernels().norm_rope_bwd(dq, dk, dv, qkv, q_weight, k_weight, table, positions, num_heads, num_kv_heads, eps)) + (None,) * 5


def qkv_norm_rope(
    qkv: torch.Tensor,
    q_weight: torch.Tensor,
    k_weight: torch.Tensor,
    table: torch.Tensor,
    num_heads: int,
    num_kv_heads: int,
    positions: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """qkv [B, S, (num_heads + 2 num_kv_heads) D] in bfloat16, float16 or float32 (dense channels, batch and token strides free);
    both weights [D], of the same type or float32; table [positions, D] float32; D a multiple of 16 up to 512. ``positions``: int32, one a token
    (any shape of B * S), or None for 0 .. S - 1 in each sequence; one that the table does not have gives NaN. Returns contiguous
    q [B, S, num_heads, D], k and v [B, S, num_kv_heads, D] in qkv's type."""
    if qkv.dim() != 3 or qkv.dtype not in _TYPES:
        raise ValueError(f"qkv must be [B, S, channels] in bfloat16, float16 or float32, got {qkv.dtype} {tuple(qkv.shape)}")
    D = q_weight.numel()
    if q_weight.dim() != 1 or q_weight.shape != k_weight.shape or D % 16 or not 16 <= D <= 512:
        raise ValueError(f"both weights must be [D], D a multiple of 16 up to 512, got {tuple(q_weight.shape)} and {tuple(k_weight.shape)}")
    if q_weight.dtype != k_weight.dtype or q_weight.dtype not in (qkv.dtype, torch.float32):
        raise ValueError(f"both weights must be of qkv's type or float32, got {q_weight.dtype} and {k_weight.dtype}")
    if num_heads < 1 or num_kv_heads < 1 or qkv.shape[2] != (num_heads + 2 * num_kv_heads) * D:
        raise ValueError(f"{num_heads} + 2 * {num_kv_heads} heads of {D} channels are not qkv's {qkv.shape[2]}")
    if table.dim() != 2 or table.shape[1] != D or table.dtype != torch.float32:
        raise ValueError(f"table must be float32 [positions, {D}], got {table.dtype} {tuple(table.shape)}")
    if positions is None:
        if qkv.shape[1] > table.shape[0]:
            raise ValueError(f"{qkv.shape[1]} positions, the table has {table.shape[0]}")
    elif positions.dtype != torch.int32 or positions.numel() != qkv.shape[0] * qkv.shape[1]:
        raise ValueError(f"positions must be int32, one a token, got {positions.dtype} {tuple(positions.shape)}")
    else:
        positions = positions.contiguous()
    if not use_hip(qkv):
        return qkv_norm_rope_ref(qkv, q_weight, k_weight, table, num_heads, num_kv_heads, positions, eps)
    q_weight, k_weight, table = q_weight.contiguous(), k_weight.contiguous(), table.contiguous()
    native = native_function("native_norm_rope", qkv)
    out = native(qkv, q_weight, k_weight, table, positions, num_heads, num_kv_heads, eps) if native else None
    return _NormRope.apply(qkv, q_weight, k_weight, table, num_heads, num_kv_heads, positions, eps) if out is None else out
