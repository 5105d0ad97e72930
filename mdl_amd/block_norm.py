"""The norms around a block, fused with its gate and residual scale.

A block's output is normalised, gated and scaled, added to the residual
stream, and the sum is normalised for the next block: one operator,
``mdl_hip::gated_residual_norm`` (differentiable) over ``block_norm_forward``
and ``block_norm_backward``, instead of about ten passes over the rows.  ROCm
kernels in ``libmdl_torch.so`` over the C ABI; CPU and fake kernels here.

Sums, statistics and the value between the two norms are fp32; outputs are
rounded once.
"""

from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor

from . import library  # noqa: F401  (loads libmdl_torch.so and its schemas)
from .library import _cpu_kernel, _fake_kernel

_NORM = torch.ops.mdl_hip.gated_residual_norm.default  # looked up once


def _check(x, block_out, post_weight, next_weight, gate, residual_scale, eps) -> None:
    if x.ndim < 1 or x.size(-1) < 1:
        raise ValueError("block norm input needs a last dimension")
    if x.dtype not in (torch.float32, torch.bfloat16) or next_weight.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError("unsupported block norm dtype; expected float32 or bfloat16")
    if eps < 0:
        raise ValueError("block norm eps must not be negative")
    if block_out is None and not (post_weight is None and gate is None and residual_scale is None):
        raise ValueError("gate, residual_scale and post_weight belong to a block's output")
    for name, t in (("block_out", block_out), ("gate", gate)):
        if t is not None and t.shape != x.shape:
            raise ValueError(f"{name} must have the input's shape")
        if t is not None and t.dtype != x.dtype:
            raise TypeError(f"{name} must have the input's dtype")
    for name, t in (("next_weight", next_weight), ("post_weight", post_weight), ("residual_scale", residual_scale)):
        if t is not None and t.shape != (x.size(-1),):
            raise ValueError(f"{name} must be [{x.size(-1)}]")
        if t is not None and t.dtype != next_weight.dtype:
            raise TypeError("block norm weights must have one dtype")


def _parts_cpu(x, block_out, post_weight, gate, residual_scale, eps):
    """fp32 (y, 1 / rms of o, normalised o, gate, post * scale, post, scale)."""

    y = x.float()
    if block_out is None:
        return y, None, None, None, None, None, None
    o = block_out.float()
    inv = torch.rsqrt(o.square().mean(-1, keepdim=True) + eps)
    one = torch.ones(x.size(-1))
    post = one if post_weight is None else post_weight.float()
    scale = one if residual_scale is None else residual_scale.float()
    g = torch.ones_like(o) if gate is None else torch.sigmoid(gate.float())
    return y + o * inv * (post * scale) * g, inv, o * inv, g, post * scale, post, scale


@_cpu_kernel("block_norm_forward")
def _forward_cpu(x, block_out, post_weight, next_weight, gate, residual_scale, eps):
    _check(x, block_out, post_weight, next_weight, gate, residual_scale, eps)
    y, inv_o = _parts_cpu(x, block_out, post_weight, gate, residual_scale, eps)[:2]
    inv_y = torch.rsqrt(y.square().mean(-1, keepdim=True) + eps)
    rstd = torch.zeros(2, x.numel() // x.size(-1))
    if inv_o is not None:
        rstd[0] = inv_o.flatten()
    rstd[1] = inv_y.flatten()
    h = (y * inv_y * next_weight.float()).to(x.dtype)
    return x.new_empty(0) if block_out is None else y.to(x.dtype), h, rstd


@_fake_kernel("block_norm_forward")
def _forward_fake(x, block_out, post_weight, next_weight, gate, residual_scale, eps):
    y = x.new_empty(0) if block_out is None else x.new_empty(x.shape)
    return y, x.new_empty(x.shape), x.new_empty((2, x.numel() // x.size(-1)), dtype=torch.float32)


@_cpu_kernel("block_norm_backward")
def _backward_cpu(grad_y, grad_h, x, block_out, post_weight, next_weight, gate, residual_scale, rstd, eps, needs):
    y, inv_o, n_o, g, both, post, scale = _parts_cpu(x, block_out, post_weight, gate, residual_scale, eps)
    over = tuple(range(x.ndim - 1))
    wdtype = next_weight.dtype
    none = x.new_empty(0)
    d_scale = d_post = d_next = next_weight.new_empty(0)
    dx = torch.zeros_like(y) if grad_y is None else grad_y.float()
    if needs & 4:
        d_next = next_weight.new_zeros(x.size(-1))
    if grad_h is not None:
        inv_y = torch.rsqrt(y.square().mean(-1, keepdim=True) + eps)
        n_y, dh = y * inv_y, grad_h.float()
        if needs & 4:
            d_next = (dh * n_y).sum(over).to(wdtype)
        a = dh * next_weight.float()
        dx = dx + inv_y * (a - n_y * (a * n_y).mean(-1, keepdim=True))
    if block_out is None:
        return dx.to(x.dtype), none, none.clone(), d_scale.clone(), d_post.clone(), d_next
    t = dx * g * n_o
    if needs & 1 and residual_scale is not None:
        d_scale = (t * post).sum(over).to(wdtype)
    if needs & 2 and post_weight is not None:
        d_post = (t * scale).sum(over).to(wdtype)
    d_gate = none if gate is None else (dx * n_o * both * g * (1 - g)).to(x.dtype)
    b = dx * g * both
    d_o = inv_o * (b - n_o * (b * n_o).mean(-1, keepdim=True))
    return dx.to(x.dtype), d_o.to(x.dtype), d_gate, d_scale.clone(), d_post.clone(), d_next


@_fake_kernel("block_norm_backward")
def _backward_fake(grad_y, grad_h, x, block_out, post_weight, next_weight, gate, residual_scale, rstd, eps, needs):
    def rows(t):
        return x.new_empty(0 if t is None else x.shape)

    def weight(t, bit):
        return next_weight.new_empty(next_weight.shape if t is not None and needs & bit else 0)

    return (x.new_empty(x.shape), rows(block_out), rows(gate), weight(residual_scale, 1), weight(post_weight, 2),
            weight(next_weight, 4))


def gated_residual_norm(
    x: Tensor,
    block_out: Optional[Tensor],
    post_weight: Optional[Tensor],
    next_weight: Tensor,
    *,
    gate: Optional[Tensor] = None,
    residual_scale: Optional[Tensor] = None,
    eps: float = 1e-6,
) -> tuple[Tensor, Tensor]:
    """``(y, h)``: the residual stream past a block, and the next block's input.

    ``y = x + sigmoid(gate) * residual_scale * rms_norm(block_out) * post_weight``
    and ``h = rms_norm(y) * next_weight`` over the last dimension (mean square
    plus ``eps``).  ``block_out`` and ``gate`` have ``x``'s shape and dtype (fp32
    or bf16), the weights the last dimension's size and one dtype of their
    own; ``gate``, ``residual_scale`` and ``post_weight`` may be left out.
    Without ``block_out`` (before the first block) ``y`` is ``x``.  Rows of at
    most 8192 (bf16) or 4096 (fp32) elements.
    """

    return _NORM(x, block_out, post_weight, next_weight, gate, residual_scale, float(eps))
