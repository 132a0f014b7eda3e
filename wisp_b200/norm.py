"""The norms around a block: post-norm, gate and residual of its output, and the norm before
the next block, in one launch (wisp_b200_block_norm in include/wisp_b200.h)."""
from __future__ import annotations

import ctypes as C

import torch

from . import abi
from .fp4 import DTYPES, elsewhere, invalid, refuse_grad, row_stride, stream_of, wants_grad


class _ErrorWord:
    """The current device's error word of wisp_b200_block_norm, as torch.as_tensor takes it."""

    def __init__(self):
        ptr = abi.lib().wisp_b200_block_norm_error_word()
        if not ptr:
            raise RuntimeError("wisp engine error: no CUDA device")
        self.__cuda_array_interface__ = {"shape": (1,), "typestr": "<i4", "data": (ptr, False),
                                         "version": 2}


def error_word(device: torch.device | int | None = None) -> torch.Tensor:
    """The device's error word (int32 [1], the library's own memory; default: the current
    device)."""
    with torch.cuda.device(device):
        return torch.as_tensor(_ErrorWord(), device="cuda")


def check(device: torch.device | int | None = None) -> None:
    """Raise if a block_norm on the device (default: the current one) gave up waiting for a row
    since the last check that raised; that row and some after it are NaN. Waits for the device's
    current stream; calls on its other streams should have finished."""
    with torch.cuda.device(device):
        word = error_word()
        try:
            abi.call("wisp_b200_check_error_flag", word.data_ptr(), stream_of(word))
        except RuntimeError:
            word.zero_()
            raise


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
    with pre=False. There is no gradient: under grad mode tensors that require one (parameters
    among them) are refused."""
    # (One pass over the arguments: at a few rows this function takes longer than its kernel.)
    if wants_grad(x, y, gate, post_weight, pre_weight, x_out, n_out):
        refuse_grad()
    ld_x = row_stride(x, "x")
    shape = x.shape
    T, M = shape
    vector = (M,)
    dev = x.get_device()
    same = True       # all tensors on x's device
    ld_y = y_type = ld_gate = gate_type = gate_kind = w_type = ld_xo = n_type = ld_n = 0
    yp = gp = pp = qp = xop = nop = None
    try:
        x_type = DTYPES[x.dtype]
        if y is not None:
            if y.shape != shape:
                raise invalid(f"y {tuple(y.shape)}, x {tuple(shape)}")
            ld_y = row_stride(y, "y")
            y_type, yp = DTYPES[y.dtype], y.data_ptr()
            same = y.get_device() == dev
        elif gate is not None or post_weight is not None or x_out is not None:
            raise invalid("gate, post_weight and x_out need y")
        elif not pre:
            raise invalid("nothing to compute")
        else:
            post = False
        if post_weight is not None:
            if not post:
                raise invalid("post_weight without post")
            if post_weight.shape != vector or not post_weight.is_contiguous():
                raise invalid(f"post_weight: a contiguous vector of {M}")
            w_type, pp = DTYPES[post_weight.dtype], post_weight.data_ptr()
            same = same and post_weight.get_device() == dev
        if pre_weight is not None:
            if not pre:
                raise invalid("pre_weight without pre")
            if pre_weight.shape != vector or not pre_weight.is_contiguous():
                raise invalid(f"pre_weight: a contiguous vector of {M}")
            t = DTYPES[pre_weight.dtype]
            if pp is not None and t != w_type:
                raise invalid("post_weight and pre_weight differ in dtype")
            w_type, qp = t, pre_weight.data_ptr()
            same = same and pre_weight.get_device() == dev
        if gate is not None:
            gshape = gate.shape
            if gshape == vector and gate.is_contiguous():
                gate_kind = abi.WISP_GATE_CHANNEL
            elif gshape == (T, 1) and gate.is_contiguous():
                gate_kind = abi.WISP_GATE_TOKEN
            elif gshape == shape:
                gate_kind = abi.WISP_GATE_ELEMENT
                ld_gate = row_stride(gate, "gate")
            else:
                raise invalid(f"gate {tuple(gshape)}: [{M}], [{T}, 1] or [{T}, {M}]")
            gate_type, gp = DTYPES[gate.dtype], gate.data_ptr()
            same = same and gate.get_device() == dev
        if x_out is not None:
            if x_out.shape != shape or x_out.dtype != x.dtype:
                raise invalid("x_out differs from x in shape or dtype")
            ld_xo, xop = row_stride(x_out, "x_out"), x_out.data_ptr()
            same = same and x_out.get_device() == dev
        if n_out is not None:
            if not pre:
                raise invalid("n_out without pre")
            if n_out.shape != shape:
                raise invalid(f"n_out {tuple(n_out.shape)}, x {tuple(shape)}")
            ld_n, nop, dtype = row_stride(n_out, "n_out"), n_out.data_ptr(), n_out.dtype
            same = same and n_out.get_device() == dev
        if pre:
            n_type = DTYPES[dtype]
    except KeyError as e:
        raise invalid(f"{e.args[0]} (float32, bfloat16 or float16)") from None
    if not same:
        raise invalid(f"a tensor is not on {x.device} like x")
    other = elsewhere(x)
    if other is not None:
        with other:
            return block_norm(x, y, gate=gate, residual_scale=residual_scale,
                              post_weight=post_weight, pre_weight=pre_weight, post=post, pre=pre,
                              eps=eps, weight_offset=weight_offset, dtype=dtype, x_out=x_out,
                              n_out=n_out)
    if y is not None and xop is None:
        x_out = torch.empty_like(x) if ld_x == M else x.new_empty(shape)
        ld_xo, xop = M, x_out.data_ptr()
    if pre and nop is None:
        n_out = x.new_empty(shape, dtype=dtype)
        ld_n, nop = M, n_out.data_ptr()
    c = abi.WispBlockNorm(T, M, x_type, y_type, w_type, gate_type, n_type, 1 if post else 0,
                          gate_kind, residual_scale, eps, weight_offset, ld_x, ld_y, ld_gate,
                          ld_xo, ld_n)
    abi.call("wisp_b200_block_norm", C.byref(c), x.data_ptr(), yp, gp, pp, qp, xop, nop,
             stream_of(x))
    return x if y is None else x_out, n_out
