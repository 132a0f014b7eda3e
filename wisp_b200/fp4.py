"""4-bit block-scaled (MXFP4 / NVFP4) rows, expert matrices and MoE layer.

Thin wrappers over the C ABI (include/wisp_b200.h): tensors are PyTorch CUDA
tensors used as device memory; every launch goes on the current torch stream
of the tensors' device. The work itself runs in libwisp_b200.so. For serving: no
operator has a gradient, and tensors that require one are refused where autograd
would record the call.

    q = quantize(x, abi.WISP_FP4_MX)                # rows -> codes and scales
    w = Fp4Weights(abi.WISP_FP4_MX, codes, scales)  # [V, n, k/2], [V, n, k/32]
    y = product(q, w, segments)                     # rows by their experts' matrices
"""
from __future__ import annotations

import contextlib
import ctypes as C

import torch

from . import abi

BLOCK = {abi.WISP_FP4_MX: 32, abi.WISP_FP4_NV: 16}
INT_MAX = 0x7FFFFFFF     # the ABI's counts are 32-bit; ctypes cuts larger ones off without a word
DTYPES = {torch.float32: abi.WISP_DT_F32, torch.bfloat16: abi.WISP_DT_BF16,
          torch.float16: abi.WISP_DT_F16}


def invalid(msg: str) -> RuntimeError:
    return RuntimeError(f"wisp engine error [{abi.WISP_ERR_INVALID_ARG}]: {msg}")


def elsewhere(t: torch.Tensor):
    """None when t is on the current CUDA device (the usual case, kept cheap), else the context
    in which launches go to t's device."""
    dev = t.get_device()
    if dev < 0:
        raise invalid(f"tensor on {t.device}: the kernels have no CPU path")
    if dev == torch._C._cuda_getDevice():
        return None
    return torch.cuda.device(dev)


def stream_of(t: torch.Tensor) -> int:
    return torch._C._cuda_getCurrentRawStream(t.get_device())


def ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def dtype_code(dtype: torch.dtype, what: str) -> int:
    code = DTYPES.get(dtype)
    if code is None:
        raise invalid(f"{what}: {dtype} (float32, bfloat16 or float16)")
    return code


def wants_grad(*tensors: torch.Tensor | None) -> bool:
    """Whether autograd would expect a gradient for one of the tensors."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def refuse_grad() -> None:
    raise invalid("a tensor requires a gradient, and this operator has none (torch.no_grad() or "
                  "detach() for serving)")


def row_stride(t: torch.Tensor, what: str) -> int:
    """Elements between the rows of a 2D tensor whose rows are contiguous."""
    shape, stride = t.shape, t.stride()
    if len(shape) != 2 or (shape[1] > 1 and stride[1] != 1):
        raise invalid(f"{what}: a 2D tensor with contiguous rows is needed")
    if shape[0] > INT_MAX or shape[1] > INT_MAX:
        raise invalid(f"{what}: {tuple(shape)}, more than 2^31 - 1 rows or columns")
    return stride[0] if shape[0] > 1 else shape[1]


def same_device(ref: torch.Tensor, **tensors) -> None:
    dev = ref.get_device()
    for name, t in tensors.items():
        if t is not None and t.get_device() != dev:
            raise invalid(f"{name} is on {t.device}, not on {ref.device}")


def _check_scale(ts: torch.Tensor | None, n: int, what: str) -> None:
    if ts is not None and (ts.dtype != torch.float32 or ts.numel() != n or not ts.is_contiguous()):
        raise invalid(f"{what}: {n} contiguous float32 needed")


def _check_codes(fmt: int, codes: torch.Tensor, scales: torch.Tensor) -> int:
    """Checks a codes/scales pair; returns the row length."""
    if fmt not in BLOCK:
        raise invalid(f"unknown format {fmt}")
    if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
        raise invalid("codes and scales are uint8")
    if not codes.is_contiguous() or not scales.is_contiguous():
        raise invalid("codes and scales must be contiguous")
    k = codes.shape[-1] * 2
    if max(k, *codes.shape) > INT_MAX:
        raise invalid(f"codes {tuple(codes.shape)}: more than 2^31 - 1 entries, rows or columns")
    if codes.shape[:-1] != scales.shape[:-1] or k % BLOCK[fmt] or \
            scales.shape[-1] != k // BLOCK[fmt]:
        raise invalid(f"codes {tuple(codes.shape)} and scales {tuple(scales.shape)} disagree "
                      f"(blocks of {BLOCK[fmt]})")
    same_device(codes, scales=scales)
    return k


class Fp4Rows:
    """Quantised rows: codes [rows, cols/2], scales [rows, cols/block], one tensor scale (NV; None
    stands for 1)."""

    def __init__(self, fmt: int, codes: torch.Tensor, scales: torch.Tensor,
                 tensor_scale: torch.Tensor | None = None):
        if codes.dim() != 2:
            raise invalid("rows are 2D")
        self.cols = _check_codes(fmt, codes, scales)
        if fmt == abi.WISP_FP4_MX and tensor_scale is not None:
            raise invalid("MX rows have no tensor scale")
        _check_scale(tensor_scale, 1, "tensor_scale")
        same_device(codes, tensor_scale=tensor_scale)
        self.fmt, self.tensor_scale, self.rows = fmt, tensor_scale, codes.shape[0]
        self._views = (codes, scales)
        self._buf = codes
        self._codes, self._scales = codes.data_ptr(), scales.data_ptr()
        self._ts = ptr(tensor_scale)

    @classmethod
    def _empty(cls, x: torch.Tensor, fmt: int, rows: int, cols: int,
               tensor_scale: torch.Tensor | None) -> "Fp4Rows":
        """Rows to be written, in one allocation on x's device; the codes and scales tensors
        are made when someone asks for them (they cost more than the launch)."""
        q = cls.__new__(cls)
        split = (rows * cols // 2 + 31) & ~31
        q._buf = buf = x.new_empty(split + rows * cols // BLOCK[fmt], dtype=torch.uint8)
        q._views = None
        q._codes = buf.data_ptr()
        q._scales = q._codes + split
        q.fmt, q.tensor_scale, q.rows, q.cols = fmt, tensor_scale, rows, cols
        q._ts = None if tensor_scale is None else tensor_scale.data_ptr()
        return q

    def record_stream(self, stream: torch.cuda.Stream) -> None:
        """As torch.Tensor.record_stream: the rows are in use on `stream` too."""
        for t in (self._buf, *(self._views or ()), self.tensor_scale):
            if t is not None:
                t.record_stream(stream)

    def _split(self) -> tuple[torch.Tensor, torch.Tensor]:
        if self._views is None:
            n, m = self.rows * self.cols // 2, self.rows * self.cols // BLOCK[self.fmt]
            at = self._scales - self._codes
            self._views = (self._buf[:n].view(self.rows, self.cols // 2),
                           self._buf[at:at + m].view(self.rows, self.cols // BLOCK[self.fmt]))
        return self._views

    @property
    def codes(self) -> torch.Tensor:
        return self._split()[0]

    @property
    def scales(self) -> torch.Tensor:
        return self._split()[1]


def tensor_scale(x: torch.Tensor) -> torch.Tensor:
    """The NV tensor scale that lets the largest block scale reach 448: max|x| / 2688
    (1 for an all-zero tensor)."""
    s = x.detach().abs().amax().float() / (6.0 * 448.0)
    return torch.where(s > 0, s, torch.ones_like(s)).reshape(1)


def quantize(x: torch.Tensor, fmt: int, tensor_scale: torch.Tensor | None = None,
             rows: torch.Tensor | None = None) -> Fp4Rows:
    """Rows of x (float32, bfloat16 or float16) as 4-bit codes; rows (int32): row p of the
    result is row rows[p] of x, a row of zeros where rows[p] is outside x. tensor_scale: needed
    for NV, not used for MX."""
    block = BLOCK.get(fmt)
    if block is None:
        raise invalid(f"unknown format {fmt}")
    if wants_grad(x, tensor_scale):
        refuse_grad()
    ld = row_stride(x, "x")
    n, cols = x.shape
    if cols % block or cols == 0:
        raise invalid(f"row length {cols} is no multiple of {block}")
    if fmt == abi.WISP_FP4_NV:
        if tensor_scale is None:
            raise invalid("NV rows need a tensor scale")
        _check_scale(tensor_scale, 1, "tensor_scale")
    else:
        tensor_scale = None
    r = n
    if rows is not None:
        if rows.dtype != torch.int32 or rows.dim() != 1 or not rows.is_contiguous():
            raise invalid("rows: a contiguous 1D int32 tensor")
        if rows.shape[0] > INT_MAX:
            raise invalid(f"rows: {rows.shape[0]} indices, more than 2^31 - 1")
        r = rows.shape[0]
    dt = dtype_code(x.dtype, "x")
    other = elsewhere(x)
    if other is not None:
        with other:
            return quantize(x, fmt, tensor_scale, rows)
    if tensor_scale is not None or rows is not None:
        same_device(x, tensor_scale=tensor_scale, rows=rows)
    q = Fp4Rows._empty(x, fmt, r, cols, tensor_scale)
    abi.call("wisp_b200_fp4_quantize", x.data_ptr(), dt, ld, n,
             None if rows is None else rows.data_ptr(), r, cols, fmt, q._ts, q._codes, q._scales,
             stream_of(x))
    return q


def dequantize(q: Fp4Rows, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values of quantised rows."""
    dt = dtype_code(dtype, "dtype")
    buf = q._buf
    other = elsewhere(buf)
    if other is not None:
        with other:
            return dequantize(q, dtype)
    cols = q.cols
    out = buf.new_empty((q.rows, cols), dtype=dtype)
    abi.call("wisp_b200_fp4_dequantize", q._codes, q._scales, q.rows, cols, q.fmt, q._ts,
             out.data_ptr(), dt, cols, stream_of(buf))
    return out


class Fp4Weights:
    """V matrices [n, k] (one per expert) laid out once for the product; with ``up`` = (codes,
    scales[, scale]), V pairs for silu(gate x) * up x. codes [V, n, k/2] stay in use where
    they are; scales [V, n, k/block] are laid out into a buffer of the object and no longer
    needed; scale: fp32 [V] tensor scales or None."""

    def __init__(self, fmt: int, codes: torch.Tensor, scales: torch.Tensor,
                 scale: torch.Tensor | None = None, up: tuple | None = None):
        if codes.dim() != 3:
            raise invalid("weight codes are [entries, n, k/2]")
        self.fmt = fmt
        self.k = _check_codes(fmt, codes, scales)
        self.entries, self.n = codes.shape[:2]
        if self.k % 32:
            raise invalid(f"k={self.k} is no multiple of 32")
        mats = [(codes, scales, scale)]
        if up is not None:
            if len(up) not in (2, 3):
                raise invalid("up: (codes, scales) or (codes, scales, scale)")
            mats.append(tuple(up) if len(up) == 3 else (*up, None))
        self.cfg = abi.WispFp4Config(fmt, self.entries, self.n, self.k, len(mats) - 1,
                                     abi.WISP_DT_F32)
        self._keep, structs = [], []
        with elsewhere(codes) or contextlib.nullcontext():
            nbytes = abi.lib().wisp_b200_fp4_prepared_bytes(C.byref(self.cfg))
            if nbytes == 0:
                raise invalid(f"weights [{self.entries}, {self.n}, {self.k}] are not supported")
            for c, s, ts in mats:
                if c.shape != codes.shape:
                    raise invalid("gate and up differ in shape")
                _check_codes(fmt, c, s)
                _check_scale(ts, self.entries, "scale")
                same_device(codes, codes=c, scales=s, scale=ts)
                prepared = torch.empty(nbytes, dtype=torch.uint8, device=codes.device)
                abi.call("wisp_b200_fp4_prepare", C.byref(self.cfg), s.data_ptr(),
                         prepared.data_ptr(), nbytes, stream_of(codes))
                self._keep.append((c, prepared, ts))
                structs.append(abi.WispFp4Mats(c.data_ptr(), prepared.data_ptr(), ptr(ts)))
            self.error_word = torch.zeros(1, dtype=torch.int32, device=codes.device)
            # laid out once: any stream may use the object from here on
            torch.cuda.current_stream(codes.device).synchronize()
        self.mats = structs[0]
        self.up_mats = structs[1] if len(structs) == 2 else None
        # what a product passes, by output type
        self._cfgs = {dt: C.byref(abi.WispFp4Config(fmt, self.entries, self.n, self.k,
                                                    len(mats) - 1, code))
                      for dt, code in DTYPES.items()}
        self._mats = C.byref(self.mats)
        self._up_mats = None if self.up_mats is None else C.byref(self.up_mats)
        self._error = self.error_word.data_ptr()

    @classmethod
    def from_values(cls, fmt: int, w: torch.Tensor, up: torch.Tensor | None = None) -> "Fp4Weights":
        """Quantises matrices w [V, n, k] (and up), one tensor scale per matrix for NV. The set
        holds constants: parameters may be given, and get no gradient from it."""
        sets = []
        for m in [w] if up is None else [w, up]:
            if m.dim() != 3:
                raise invalid("weights are [entries, n, k]")
            m = m.detach()
            ts = None
            if fmt == abi.WISP_FP4_NV:
                ts = torch.cat([tensor_scale(e) for e in m])
            qs = [quantize(e, fmt, None if ts is None else ts[i:i + 1]) for i, e in enumerate(m)]
            sets.append((torch.stack([q.codes for q in qs]), torch.stack([q.scales for q in qs]),
                         ts))
        return cls(fmt, *sets[0], up=sets[1] if len(sets) == 2 else None)

    @property
    def device(self) -> torch.device:
        return self.error_word.device

    def check(self) -> None:
        """Raise if a product with these weights gave up waiting or skipped a bad segment since
        the last check that raised (which clears what it reports; products on other streams than
        the current one should have finished). Waits for the current stream."""
        with elsewhere(self.error_word) or contextlib.nullcontext():
            try:
                abi.call("wisp_b200_check_error_flag", self.error_word.data_ptr(),
                         stream_of(self.error_word))
            except RuntimeError:
                self.error_word.zero_()
                raise


def product(q: Fp4Rows, w: Fp4Weights, segments: torch.Tensor | None = None,
            out: torch.Tensor | None = None, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """out[p] = w_e q[p] (silu(gate q) * up q for paired weights) for the rows p of each
    segment. segments: int32 [S, 4] (expert, first row, rows, 0) on the device, as
    wisp_b200_dispatch_plan writes them; None: all rows through entry 0. Rows in no segment are
    left as they are (out given) or undefined (out allocated here)."""
    if q.fmt != w.fmt or q.cols != w.k:
        raise invalid(f"rows (format {q.fmt}, k={q.cols}) do not fit the weights (format "
                      f"{w.fmt}, k={w.k})")
    if wants_grad(out, q.tensor_scale):
        refuse_grad()
    n_segs = 0
    if segments is not None:
        if segments.dtype != torch.int32 or segments.dim() != 2 or segments.shape[1] != 4 or \
                not segments.is_contiguous():
            raise invalid("segments: a contiguous int32 [S, 4] tensor")
        n_segs = min(segments.shape[0], INT_MAX)     # (1025 at most, which the call checks)
    buf = q._buf
    other = elsewhere(buf)
    if other is not None:
        with other:
            return product(q, w, segments, out, dtype)
    same_device(buf, weights=w.error_word, segments=segments, out=out)
    rows = q.rows
    if out is None:
        dtype_code(dtype, "dtype")
        out = buf.new_empty((rows, w.n), dtype=dtype)
        ld = w.n
    else:
        if out.shape != (rows, w.n):
            raise invalid(f"out {tuple(out.shape)}, not {(rows, w.n)}")
        dtype = out.dtype
        dtype_code(dtype, "out")
        ld = row_stride(out, "out")
    if segments is not None and n_segs == 0:
        return out          # (an empty tensor has no address, which would mean "all rows")
    x = abi.WispFp4Rows(q._codes, q._scales, q._ts, rows)
    abi.call("wisp_b200_fp4_product", w._cfgs[dtype], w._mats, w._up_mats, C.byref(x),
             None if segments is None else segments.data_ptr(), n_segs, out.data_ptr(), ld,
             w._error, stream_of(buf))
    return out


class Fp4MoeLayer:
    """One routed-expert MoE layer over fp4 weights (the counterpart of moe.MoeLayer): router,
    dispatch, quantised rows, gate/up + SwiGLU, quantised rows, down, fixed-order combine."""

    def __init__(self, spec, router_w: torch.Tensor, router_bias: torch.Tensor | None,
                 gate_up: Fp4Weights, down: Fp4Weights, tokens: int,
                 x_scale: torch.Tensor | None = None, h_scale: torch.Tensor | None = None):
        """spec: a synth.MoeSpec (its group_size is not used). x_scale, h_scale: the NV tensor
        scales of the layer's input and of the SwiGLU output."""
        V = spec.n_virtual
        if (gate_up.entries, gate_up.n, gate_up.k) != (V, spec.inter, spec.hidden) or \
                gate_up.up_mats is None:
            raise invalid("gate_up does not fit the layer")
        if (down.entries, down.n, down.k) != (V, spec.hidden, spec.inter) or \
                down.up_mats is not None or down.fmt != gate_up.fmt:
            raise invalid("down does not fit the layer")
        if gate_up.fmt == abi.WISP_FP4_NV and (x_scale is None or h_scale is None):
            raise invalid("NV layers need x_scale and h_scale")
        if router_w.dtype not in (torch.bfloat16, torch.float16) or \
                router_w.shape != (spec.n_experts, spec.hidden) or not router_w.is_contiguous():
            raise invalid("router_w: contiguous bfloat16 or float16 [experts, hidden]")
        if router_bias is not None and (router_bias.dtype != torch.float32 or
                                        router_bias.shape != (spec.n_experts,) or
                                        not router_bias.is_contiguous()):
            raise invalid("router_bias: contiguous float32 [experts]")
        _check_scale(x_scale, 1, "x_scale")
        _check_scale(h_scale, 1, "h_scale")
        same_device(gate_up.error_word, router_w=router_w, router_bias=router_bias,
                    down=down.error_word, x_scale=x_scale, h_scale=h_scale)
        self.spec, self.gate_up, self.down = spec, gate_up, down
        self.cfg = spec.cfg(tokens)
        self.cfg.router_fp16 = 1 if router_w.dtype == torch.float16 else 0
        self._keep = (router_w, router_bias, x_scale, h_scale)
        w = self._w = abi.WispFp4MoeWeights()
        w.router_w = router_w.data_ptr()
        w.router_bias = None if router_bias is None else router_bias.data_ptr()
        w.gate, w.up, w.down = gate_up.mats, gate_up.up_mats, down.mats
        w.x_scale = None if x_scale is None else x_scale.data_ptr()
        w.h_scale = None if h_scale is None else h_scale.data_ptr()
        w.format = gate_up.fmt
        nbytes = abi.lib().wisp_b200_fp4_moe_workspace_bytes(C.byref(self.cfg), gate_up.fmt)
        if nbytes == 0:
            raise invalid("invalid MoE config")
        dev = gate_up.device
        self.workspace = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        self.idx = torch.empty((tokens, spec.top_k), dtype=torch.int32, device=dev)
        self.wt = torch.empty((tokens, spec.top_k), dtype=torch.float32, device=dev)

    def forward(self, x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
        """x bf16 [tokens, hidden] -> fp32 [tokens, hidden]. One call at a time per layer."""
        shape = (self.cfg.tokens, self.spec.hidden)
        if x.dtype != torch.bfloat16 or not x.is_contiguous() or x.shape != shape:
            raise invalid(f"x: contiguous bfloat16 {shape}")
        if wants_grad(x, out):
            refuse_grad()
        same_device(self.workspace, x=x, out=out)
        other = elsewhere(x)
        if other is not None:
            with other:
                return self.forward(x, out)
        if out is None:
            out = torch.empty(shape, dtype=torch.float32, device=x.device)
        elif out.dtype != torch.float32 or out.shape != shape or not out.is_contiguous():
            raise invalid(f"out: contiguous float32 {shape}")
        abi.call("wisp_b200_fp4_moe_forward", C.byref(self.cfg), C.byref(self._w), x.data_ptr(),
                 out.data_ptr(), self.idx.data_ptr(), self.wt.data_ptr(),
                 self.workspace.data_ptr(), self.workspace.numel(),
                 self.gate_up.error_word.data_ptr(), stream_of(x))
        return out

    def check(self) -> None:
        """Raise if a forward of this layer, or another product with its gate and up weights,
        gave up waiting since the last check that raised."""
        self.gate_up.check()
