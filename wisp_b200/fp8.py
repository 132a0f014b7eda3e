"""8-bit block-scaled (e4m3, fp32 scales) rows, expert matrices and MoE layer.

Thin wrappers over the C ABI (include/wisp_b200.h): tensors are PyTorch CUDA
tensors used as device memory; every launch goes on the current torch stream
of the tensors' device. The work itself runs in libwisp_b200.so. For serving: no
operator has a gradient or a tangent, and tensors that require or carry one are refused
where autograd would follow the call.

    q = quantize(x)                       # rows -> codes, a scale per 128 values
    q = gather(q, rows)                   # the rows of each expert's tokens
    w = Fp8Weights(codes, scales)         # [V, n, k], [V, n/128, k/128]
    y = product(q, w, segments)           # rows by their experts' matrices
"""
from __future__ import annotations

import contextlib
import ctypes as C

import torch

from . import abi
from .fp4 import DTYPES, INT_MAX, dtype_code, elsewhere, invalid, refuse_grad, row_stride, \
    same_device, stream_of, wants_grad
from .routing import check_bias

BLOCK = 128
CODES = torch.float8_e4m3fn


def _blocks(n: int) -> int:
    return (n + BLOCK - 1) // BLOCK


def _as_codes(codes: torch.Tensor, what: str) -> torch.Tensor:
    if codes.dtype == torch.uint8:
        codes = codes.view(CODES)
    if codes.dtype != CODES:
        raise invalid(f"{what}: {codes.dtype} (float8_e4m3fn, or its bytes as uint8)")
    if not codes.is_contiguous():
        raise invalid(f"{what} must be contiguous")
    k = codes.shape[-1]
    if k == 0 or k % 16:
        raise invalid(f"{what}: row length {k} is no multiple of 16")
    if max(codes.shape) > INT_MAX:
        raise invalid(f"{what} {tuple(codes.shape)}: more than 2^31 - 1 entries, rows or columns")
    return codes


class Fp8Rows:
    """Quantised rows: codes [rows, cols] (float8_e4m3fn), scales float32 [rows, ceil(cols/128)]
    of any strides (quantize stores them block by block, as the product reads them)."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        if codes.dim() != 2:
            raise invalid("rows are 2D")
        codes = _as_codes(codes, "codes")
        self.rows, self.cols = codes.shape
        if scales.dtype != torch.float32 or scales.shape != (self.rows, _blocks(self.cols)):
            raise invalid(f"scales: float32 {(self.rows, _blocks(self.cols))}, not {scales.dtype} "
                          f"{tuple(scales.shape)}")
        if wants_grad(codes, scales):
            refuse_grad()
        same_device(codes, scales=scales)
        self._buf = self._codes_view = codes
        self._scales_view = scales
        self._codes, self._scales = codes.data_ptr(), scales.data_ptr()
        self._row, self._block = scales.stride()

    @classmethod
    def _empty(cls, x: torch.Tensor, rows: int, cols: int) -> "Fp8Rows":
        """Rows to be written, in one allocation on x's device; the codes and scales tensors
        are made when someone asks for them."""
        q = cls.__new__(cls)
        n = rows * cols             # (a multiple of 16)
        q._buf = buf = x.new_empty(n // 4 + rows * ((cols + BLOCK - 1) // BLOCK),
                                   dtype=torch.float32)
        q._codes_view = q._scales_view = None
        q._codes = at = buf.data_ptr()
        q._scales = at + n
        q._row, q._block = 1, rows or 1
        q.rows, q.cols = rows, cols
        return q

    def __reduce__(self):
        # (copies and pickles are made anew from their own tensors: the addresses are of these)
        return Fp8Rows, (self.codes.view(torch.uint8), self.scales)

    def record_stream(self, stream: torch.cuda.Stream) -> None:
        """As torch.Tensor.record_stream: the rows are in use on `stream` too."""
        for t in (self._buf, self._codes_view, self._scales_view):
            if t is not None:
                t.record_stream(stream)

    @property
    def codes(self) -> torch.Tensor:
        if self._codes_view is None:
            self._codes_view = self._buf.view(CODES).as_strided((self.rows, self.cols),
                                                                (self.cols, 1))
        return self._codes_view

    @property
    def scales(self) -> torch.Tensor:
        if self._scales_view is None:
            self._scales_view = self._buf.as_strided((self.rows, _blocks(self.cols)),
                                                     (1, self._block), self.rows * self.cols // 4)
        return self._scales_view


def _indices(rows: torch.Tensor) -> int:
    if rows.dtype != torch.int32 or rows.dim() != 1 or not rows.is_contiguous():
        raise invalid("rows: a contiguous 1D int32 tensor")
    if rows.shape[0] > INT_MAX:
        raise invalid(f"rows: {rows.shape[0]} indices, more than 2^31 - 1")
    return rows.shape[0]


def quantize(x: torch.Tensor, rows: torch.Tensor | None = None, pow2: bool = False) -> Fp8Rows:
    """Rows of x (float32, bfloat16 or float16) as e4m3 codes, with one scale max|x| / 448 per
    128 values (pow2: the least power of two that is not below it); rows (int32): row p of the
    result is row rows[p] of x, a row of zeros where rows[p] is outside x."""
    if wants_grad(x):
        refuse_grad()
    ld = row_stride(x, "x")
    n, cols = x.shape
    if cols % 16 or cols == 0:
        raise invalid(f"row length {cols} is no multiple of 16")
    r = n if rows is None else _indices(rows)
    dt = dtype_code(x.dtype, "x")
    other = elsewhere(x)
    if other is not None:
        with other:
            return quantize(x, rows, pow2)
    if rows is not None:
        same_device(x, rows=rows)
        # Every row of x once and copies, where rows are wanted several times and there is
        # enough to do: 4096 bf16 rows of 7168 to 32,768 142 -> 77 us, 1024 to 8192 42 -> 27; 256
        # to 2048 16.4 against 17.4, 4096 to 8192 43 against 42. (A second call from here costs
        # the host 7 to 10 us; the layer, whose launches do not, copies from fewer rows on.)
        if r >= 4 * n and r * cols >= 1 << 25:
            return gather(quantize(x, pow2=pow2), rows)
    q = Fp8Rows._empty(x, r, cols)
    abi.call("wisp_b200_fp8_quantize", x.data_ptr(), dt, ld, n,
             None if rows is None else rows.data_ptr(), r, cols, 1 if pow2 else 0, q._codes,
             q._scales, 1, q._block, stream_of(x))
    return q


def gather(q: Fp8Rows, rows: torch.Tensor) -> Fp8Rows:
    """Rows of q, codes and scales as they are: row p of the result is row rows[p] (int32) of q, a
    row of zeros where rows[p] is outside q."""
    r, buf, cols = _indices(rows), q._buf, q.cols
    other = elsewhere(buf)
    if other is not None:
        with other:
            return gather(q, rows)
    same_device(buf, rows=rows)
    out = Fp8Rows._empty(buf, r, cols)
    x = abi.WispFp8Rows(q._codes, q._scales, q._row, q._block, q.rows)
    abi.call("wisp_b200_fp8_gather", C.byref(x), rows.data_ptr(), r, cols, out._codes, out._scales,
             1, out._block, stream_of(buf))
    return out


def dequantize(q: Fp8Rows, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values of quantised rows."""
    dt = dtype_code(dtype, "dtype")
    buf = q._buf
    other = elsewhere(buf)
    if other is not None:
        with other:
            return dequantize(q, dtype)
    cols = q.cols
    out = buf.new_empty((q.rows, cols), dtype=dtype)
    abi.call("wisp_b200_fp8_dequantize", q._codes, q._scales, q._row, q._block, q.rows, cols,
             out.data_ptr(), dt, cols, stream_of(buf))
    return out


class Fp8Weights:
    """V matrices [n, k] (one per expert) for the product; with ``up`` = (codes, scales), V pairs
    for silu(gate x) * up x. codes [V, n, k] (float8_e4m3fn) and scales float32 [V, ceil(n/128),
    ceil(k/128)] stay in use where they are."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, up: tuple | None = None):
        if codes.dim() != 3:
            raise invalid("weight codes are [entries, n, k]")
        mats = [(codes, scales)]
        if up is not None:
            if len(up) != 2:
                raise invalid("up: (codes, scales)")
            mats.append(tuple(up))
        self.entries, self.n, self.k = codes.shape
        self._keep, structs = [], []
        for c, s in mats:
            c = _as_codes(c, "weight codes")
            if c.shape != codes.shape:
                raise invalid("gate and up differ in shape")
            want = (self.entries, _blocks(self.n), _blocks(self.k))
            if s.dtype != torch.float32 or s.shape != want or not s.is_contiguous():
                raise invalid(f"weight scales: contiguous float32 {want}")
            if wants_grad(c, s):
                refuse_grad()
            same_device(codes, codes=c, scales=s)
            self._keep.append((c, s))
            structs.append(abi.WispFp8Mats(c.data_ptr(), s.data_ptr()))
        with elsewhere(codes) or contextlib.nullcontext():
            with torch.inference_mode(False):        # (check clears it in either mode)
                self.error_word = torch.zeros(1, dtype=torch.int32, device=codes.device)
            # any stream may use the object from here on
            torch.cuda.current_stream(codes.device).synchronize()
        self.mats = structs[0]
        self.up_mats = structs[1] if len(structs) == 2 else None
        # what a product passes, by output type
        self._cfgs = {dt: C.byref(abi.WispFp8Config(self.entries, self.n, self.k, len(mats) - 1,
                                                    code))
                      for dt, code in DTYPES.items()}
        self._mats = C.byref(self.mats)
        self._up_mats = None if self.up_mats is None else C.byref(self.up_mats)
        self._error = self.error_word.data_ptr()

    @classmethod
    def from_values(cls, w: torch.Tensor, up: torch.Tensor | None = None) -> "Fp8Weights":
        """Quantises matrices w [V, n, k] (and up) by blocks of 128 x 128. The set holds
        constants: parameters may be given, and get no gradient from it."""
        sets = [quantize_weights(m) for m in ([w] if up is None else [w, up])]
        return cls(*sets[0], up=sets[1] if len(sets) == 2 else None)

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


def quantize_weights(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of matrices w [V, n, k], one scale max|w| / 448 per block of 128 x 128.
    The codes are constants: a parameter gets no gradient from them."""
    if w.dim() != 3:
        raise invalid("weights are [entries, n, k]")
    w = w.detach().contiguous()
    V, n, k = w.shape
    if k == 0 or k % 16:
        raise invalid(f"k={k} is no multiple of 16")
    if max(w.shape) > INT_MAX:
        raise invalid(f"weights {tuple(w.shape)}: more than 2^31 - 1 entries, rows or columns")
    dt = dtype_code(w.dtype, "weights")
    other = elsewhere(w)
    if other is not None:
        with other:
            return quantize_weights(w)
    codes = torch.empty((V, n, k), dtype=CODES, device=w.device)
    scales = torch.empty((V, _blocks(n), _blocks(k)), dtype=torch.float32, device=w.device)
    abi.call("wisp_b200_fp8_quantize_weights", w.data_ptr(), dt, V, n, k, codes.data_ptr(),
             scales.data_ptr(), stream_of(w))
    return codes, scales


def product(q: Fp8Rows, w: Fp8Weights, segments: torch.Tensor | None = None,
            out: torch.Tensor | None = None, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """out[p] = w_e q[p] (silu(gate q) * up q for paired weights) for the rows p of each
    segment. segments: int32 [S, 4] (expert, first row, rows, 0) on the device, as
    wisp_b200_dispatch_plan writes them; None: all rows through entry 0. Rows in no segment are
    left as they are (out given) or undefined (out allocated here)."""
    if q.cols != w.k:
        raise invalid(f"rows of {q.cols} values do not fit the weights (k={w.k})")
    if wants_grad(out):
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
    x = abi.WispFp8Rows(q._codes, q._scales, q._row, q._block, rows)
    abi.call("wisp_b200_fp8_product", w._cfgs[dtype], w._mats, w._up_mats, C.byref(x),
             None if segments is None else segments.data_ptr(), n_segs, out.data_ptr(), ld,
             w._error, stream_of(buf))
    return out


class Fp8MoeLayer:
    """One routed-expert MoE layer over fp8 weights (the counterpart of moe.MoeLayer): router,
    dispatch, quantised rows, gate/up + SwiGLU, quantised rows, down, fixed-order combine."""

    def __init__(self, spec, router_w: torch.Tensor, router_bias: torch.Tensor | None,
                 gate_up: Fp8Weights, down: Fp8Weights, tokens: int,
                 routing: abi.WispRouting | None = None, score_bias: torch.Tensor | None = None,
                 pow2: bool = False):
        """spec: a synth.MoeSpec (its group_size is not used). routing: a routing.policy, in place
        of the spec's scoring, groups and scaling; score_bias: its balance bias, which chooses and
        does not weigh. pow2: the quantised rows' scales are powers of two."""
        V = spec.n_virtual
        if (gate_up.entries, gate_up.n, gate_up.k) != (V, spec.inter, spec.hidden) or \
                gate_up.up_mats is None:
            raise invalid("gate_up does not fit the layer")
        if (down.entries, down.n, down.k) != (V, spec.hidden, spec.inter) or \
                down.up_mats is not None:
            raise invalid("down does not fit the layer")
        if router_w.dtype not in (torch.bfloat16, torch.float16) or \
                router_w.shape != (spec.n_experts, spec.hidden) or not router_w.is_contiguous():
            raise invalid("router_w: contiguous bfloat16 or float16 [experts, hidden]")
        check_bias(router_bias, spec.n_experts, "router_bias")
        check_bias(score_bias, spec.n_experts, "score_bias")
        if score_bias is not None and routing is None:
            raise invalid("score_bias without a routing")
        same_device(gate_up.error_word, router_w=router_w, router_bias=router_bias,
                    down=down.error_word, score_bias=score_bias)
        if wants_grad(router_w, router_bias, score_bias):
            refuse_grad()
        if not 0 < tokens <= INT_MAX:
            raise invalid(f"tokens={tokens}")
        self.spec, self.gate_up, self.down, self.routing = spec, gate_up, down, routing
        self.cfg = spec.cfg(tokens)
        self.cfg.router_fp16 = 1 if router_w.dtype == torch.float16 else 0
        self._routing = None if routing is None else C.byref(routing)
        self._keep = (router_w, router_bias, score_bias)
        w = self._w = abi.WispFp8MoeWeights()
        w.router_w = router_w.data_ptr()
        w.router_bias = None if router_bias is None else router_bias.data_ptr()
        w.score_bias = None if score_bias is None else score_bias.data_ptr()
        w.gate, w.up, w.down = gate_up.mats, gate_up.up_mats, down.mats
        w.pow2 = 1 if pow2 else 0
        nbytes = abi.lib().wisp_b200_fp8_moe_workspace_bytes(C.byref(self.cfg), self._routing)
        if nbytes == 0:
            raise invalid("invalid MoE config or routing")
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
        abi.call("wisp_b200_fp8_moe_forward", C.byref(self.cfg), self._routing, C.byref(self._w),
                 x.data_ptr(), out.data_ptr(), self.idx.data_ptr(), self.wt.data_ptr(),
                 self.workspace.data_ptr(), self.workspace.numel(),
                 self.gate_up.error_word.data_ptr(), stream_of(x))
        return out

    def check(self) -> None:
        """Raise if a forward of this layer, or another product with its gate and up weights,
        gave up waiting since the last check that raised."""
        self.gate_up.check()
