"""The norms around a block: post-norm, gate and residual of its output, and the norm before
the next block, in one launch (wisp_b200_block_norm in include/wisp_b200.h)."""
from __future__ import annotations

import ctypes as C

import torch

from . import abi
from .fp4 import dtype_code, elsewhere, invalid, row_stride, stream_of


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
    ld_x = row_stride(x, "x")
    T, M = x.shape
    x_type = dtype_code(x.dtype, "x")
    ld_y = y_type = ld_gate = gate_type = gate_kind = w_type = ld_xo = n_type = ld_n = 0
    xp, yp, gp, pp, qp, xop, nop = x.data_ptr(), None, None, None, None, None, None
    dev = x.get_device()
    same = True       # all tensors on x's device
    if y is None:
        if gate is not None or post_weight is not None or x_out is not None:
            raise invalid("gate, post_weight and x_out need y")
        if not pre:
            raise invalid("nothing to compute")
        post = False
    else:
        if y.shape != x.shape:
            raise invalid(f"y {tuple(y.shape)}, x {tuple(x.shape)}")
        ld_y = row_stride(y, "y")
        y_type = dtype_code(y.dtype, "y")
        yp = y.data_ptr()
        same = y.get_device() == dev
    if post_weight is not None:
        if not post:
            raise invalid("post_weight without post")
        _weight(post_weight, M, "post_weight")
        w_type = dtype_code(post_weight.dtype, "post_weight")
        pp = post_weight.data_ptr()
        same = same and post_weight.get_device() == dev
    if pre_weight is not None:
        if not pre:
            raise invalid("pre_weight without pre")
        _weight(pre_weight, M, "pre_weight")
        if pp is not None and pre_weight.dtype != post_weight.dtype:
            raise invalid("post_weight and pre_weight differ in dtype")
        w_type = dtype_code(pre_weight.dtype, "pre_weight")
        qp = pre_weight.data_ptr()
        same = same and pre_weight.get_device() == dev
    if gate is not None:
        gate_type = dtype_code(gate.dtype, "gate")
        shape = gate.shape
        if shape == (M,) and gate.is_contiguous():
            gate_kind = abi.WISP_GATE_CHANNEL
        elif shape == (T, 1) and gate.is_contiguous():
            gate_kind = abi.WISP_GATE_TOKEN
        elif shape == (T, M):
            gate_kind = abi.WISP_GATE_ELEMENT
            ld_gate = row_stride(gate, "gate")
        else:
            raise invalid(f"gate {tuple(shape)}: [{M}], [{T}, 1] or [{T}, {M}]")
        gp = gate.data_ptr()
        same = same and gate.get_device() == dev
    if n_out is not None and not pre:
        raise invalid("n_out without pre")
    for out in (x_out, n_out):
        if out is not None:
            if out.shape != x.shape:
                raise invalid(f"an output is {tuple(out.shape)}, x {tuple(x.shape)}")
            same = same and out.get_device() == dev
    if not same:
        raise invalid(f"a tensor is not on {x.device} like x")
    other = elsewhere(x)
    if other is not None:
        with other:
            return block_norm(x, y, gate=gate, residual_scale=residual_scale,
                              post_weight=post_weight, pre_weight=pre_weight, post=post, pre=pre,
                              eps=eps, weight_offset=weight_offset, dtype=dtype, x_out=x_out,
                              n_out=n_out)
    if y is not None:
        if x_out is None:
            x_out, ld_xo = x.new_empty((T, M)), M
        else:
            if x_out.dtype != x.dtype:
                raise invalid("x_out differs from x in dtype")
            ld_xo = row_stride(x_out, "x_out")
        xop = x_out.data_ptr()
    if pre:
        if n_out is None:
            n_out, ld_n = x.new_empty((T, M), dtype=dtype), M
        else:
            ld_n, dtype = row_stride(n_out, "n_out"), n_out.dtype
        n_type = dtype_code(dtype, "n")
        nop = n_out.data_ptr()
    c = abi.WispBlockNorm(T, M, x_type, y_type, w_type, gate_type, n_type, 1 if post else 0,
                          gate_kind, residual_scale, eps, weight_offset, ld_x, ld_y, ld_gate,
                          ld_xo, ld_n)
    abi.call("wisp_b200_block_norm", C.byref(c), xp, yp, gp, pp, qp, xop, nop, stream_of(x))
    return x if y is None else x_out, n_out
