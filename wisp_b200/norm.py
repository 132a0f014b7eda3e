"""The norms around a block: post-norm, gate and residual of its output, and the norm before
the next block, in one launch (wisp_b200_block_norm in include/wisp_b200.h)."""
from __future__ import annotations

import ctypes as C

import torch

from . import abi
from .fp4 import dtype_code, invalid, on_device, row_stride, same_device, stream_of


def _weight(w: torch.Tensor | None, hidden: int, what: str) -> None:
    if w is not None and (w.shape != (hidden,) or not w.is_contiguous()):
        raise invalid(f"{what}: a contiguous vector of {hidden}")


def block_norm(x: torch.Tensor, y: torch.Tensor | None = None, *,
               gate: torch.Tensor | None = None, residual_scale: float = 1.0,
               post_weight: torch.Tensor | None = None, pre_weight: torch.Tensor | None = None,
               post: bool = True, pre: bool = True, eps: float = 1e-6,
               weight_offset: float = 0.0, dtype: torch.dtype = torch.bfloat16,
               x_out: torch.Tensor | None = None, n_out: torch.Tensor | None = None):
    """(x', n) of rows x and a block's output rows y:

        x' = residual_scale * x + gate * post_norm(y)     (x itself without y)
        n  = pre_norm(x')

    with post_norm(v) = v / sqrt(mean(v^2) + eps) * (weight_offset + post_weight) (v itself with
    post=False) and pre_norm alike. gate: [hidden], [tokens, 1] or [tokens, hidden]; the two
    weights share a dtype. x' has x's dtype (x_out may be x itself), n has ``dtype``; n is None
    with pre=False."""
    T, M = x.shape if x.dim() == 2 else (0, 0)
    c = abi.WispBlockNorm()
    c.tokens, c.hidden = T, M
    c.ld_x = row_stride(x, "x")
    c.x_type = dtype_code(x.dtype, "x")
    c.eps, c.residual_scale, c.weight_offset = eps, residual_scale, weight_offset
    if y is None:
        if gate is not None or post_weight is not None or x_out is not None:
            raise invalid("gate, post_weight and x_out need y")
        if not pre:
            raise invalid("nothing to compute")
    else:
        if y.shape != x.shape:
            raise invalid(f"y {tuple(y.shape)}, x {tuple(x.shape)}")
        c.ld_y = row_stride(y, "y")
        c.y_type = dtype_code(y.dtype, "y")
        c.post_norm = 1 if post else 0
        if post_weight is not None and not post:
            raise invalid("post_weight without post")
    if pre_weight is not None and not pre:
        raise invalid("pre_weight without pre")
    if n_out is not None and not pre:
        raise invalid("n_out without pre")
    _weight(post_weight, M, "post_weight")
    _weight(pre_weight, M, "pre_weight")
    w = pre_weight if pre_weight is not None else post_weight
    if w is not None:
        c.w_type = dtype_code(w.dtype, "weight")
        if post_weight is not None and post_weight.dtype != w.dtype:
            raise invalid("post_weight and pre_weight differ in dtype")
    if gate is not None:
        c.gate_type = dtype_code(gate.dtype, "gate")
        if gate.shape == (M,) and gate.is_contiguous():
            c.gate_kind = abi.WISP_GATE_CHANNEL
        elif gate.shape == (T, 1) and gate.is_contiguous():
            c.gate_kind = abi.WISP_GATE_TOKEN
        elif gate.shape == (T, M):
            c.gate_kind = abi.WISP_GATE_ELEMENT
            c.ld_gate = row_stride(gate, "gate")
        else:
            raise invalid(f"gate {tuple(gate.shape)}: [{M}], [{T}, 1] or [{T}, {M}]")
    same_device(x, y=y, gate=gate, post_weight=post_weight, pre_weight=pre_weight, x_out=x_out,
                n_out=n_out)
    with on_device(x):
        if y is None:
            x_new, xo = x, None
        else:
            if x_out is None:
                x_out = torch.empty((T, M), dtype=x.dtype, device=x.device)
            elif x_out.shape != x.shape or x_out.dtype != x.dtype:
                raise invalid("x_out differs from x in shape or dtype")
            c.ld_x_out = row_stride(x_out, "x_out")
            x_new, xo = x_out, x_out.data_ptr()
        if pre:
            if n_out is None:
                n_out = torch.empty((T, M), dtype=dtype, device=x.device)
            elif n_out.shape != x.shape:
                raise invalid("n_out differs from x in shape")
            c.n_type = dtype_code(n_out.dtype, "n")
            c.ld_n = row_stride(n_out, "n_out")
        abi.call("wisp_b200_block_norm", C.byref(c), x.data_ptr(),
                 None if y is None else y.data_ptr(), None if gate is None else gate.data_ptr(),
                 None if post_weight is None else post_weight.data_ptr(),
                 None if pre_weight is None else pre_weight.data_ptr(), xo,
                 n_out.data_ptr() if pre else None, stream_of(x))
    return x_new, n_out if pre else None
