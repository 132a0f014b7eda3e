"""4-bit block-scaled rows, products and the MoE layer over them, against the formats'
definitions in 64 bits; refusals on the CPU."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

import fp4_ref as ref
from fp4_ref import MX, NV
from wisp_b200 import abi, fp4, norm, synth

P = 1 << 20   # a non-null aligned stand-in pointer; never dereferenced here
DEV = "cuda"
FMTS = pytest.mark.parametrize("fmt", [MX, NV], ids=["mx", "nv"])
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------------------
# Refusals (no GPU)
# ---------------------------------------------------------------------------
def _refused(name, *args, match=""):
    with pytest.raises(RuntimeError, match=r"wisp engine error \[4\].*" + match):
        abi.call(name, *args)


@pytest.mark.parametrize("kw,match", [
    (dict(fmt=2), "format"), (dict(dt=3), "x_type"), (dict(cols=48), "cols"), (dict(cols=0), "cols"),
    (dict(ld=32), "ld"), (dict(rows=-1), "rows"), (dict(rows=5), "d_src"), (dict(x=None), "null"),
    (dict(codes=P + 4), "aligned"), (dict(x=P + 1), "aligned"), (dict(fmt=NV, ts=None), "null"),
    (dict(scales=None), "null"),
])
def test_quantize_refuses(kw, match):
    a = dict(x=P, dt=1, ld=64, x_rows=4, src=None, rows=4, cols=64, fmt=MX, ts=P, codes=P, scales=P)
    a.update(kw)
    _refused("wisp_b200_fp4_quantize", a["x"], a["dt"], a["ld"], a["x_rows"], a["src"], a["rows"],
             a["cols"], a["fmt"], a["ts"], a["codes"], a["scales"], None, match=match)


@pytest.mark.parametrize("kw,match", [
    (dict(fmt=-1), "format"), (dict(dt=9), "out_type"), (dict(cols=24, fmt=NV), "cols"),
    (dict(ld=63), "ld"), (dict(out=None), "null"), (dict(out=P + 2, dt=0), "aligned"),
    (dict(codes=P + 2), "aligned"),
])
def test_dequantize_refuses(kw, match):
    a = dict(codes=P, scales=P, rows=4, cols=64, fmt=MX, out=P, dt=1, ld=64)
    a.update(kw)
    _refused("wisp_b200_fp4_dequantize", a["codes"], a["scales"], a["rows"], a["cols"], a["fmt"],
             P, a["out"], a["dt"], a["ld"], None, match=match)


def test_calls_without_rows_launch_nothing():
    abi.call("wisp_b200_fp4_quantize", None, 1, 64, 0, None, 0, 64, MX, None, None, None, None)
    abi.call("wisp_b200_fp4_dequantize", None, None, 0, 64, MX, None, None, 1, 64, None)
    cfg = abi.WispFp4Config(MX, 2, 64, 64, 0, 1)
    m = abi.WispFp4Mats(P, P, None)
    x = abi.WispFp4Rows(None, None, None, 0)
    abi.call("wisp_b200_fp4_product", C.byref(cfg), C.byref(m), None, C.byref(x), None, 0, None, 64,
             None, None)


@pytest.mark.parametrize("kw,match", [
    (dict(format=2), "format"), (dict(k=48), "k=48"), (dict(n=0), "n=0"), (dict(n_entries=0), "n_entries"),
    (dict(n_entries=1 << 16, n=1 << 16), "2\\^31"), (dict(out_type=3), "out_type"),
    (dict(swiglu=1), "up weights"), (dict(up=True), "without swiglu"), (dict(codes=P + 8), "aligned"),
    (dict(prepared=P + 128), "aligned"), (dict(xcodes=P + 8), "aligned"), (dict(out=None), "null"),
    (dict(ld=63), "ld"), (dict(n_segs=1026), "n_segs"), (dict(n_segs=-1), "n_segs"),
    (dict(segs=None, n_segs=1), "n_segs"), (dict(rows=-1), "rows"), (dict(codes=None), "null"),
])
def test_product_refuses(kw, match):
    a = dict(format=MX, n_entries=2, n=64, k=64, swiglu=0, out_type=1, codes=P, prepared=P, up=False,
             xcodes=P, rows=3, segs=P, n_segs=2, out=P, ld=64)
    a.update(kw)
    cfg = abi.WispFp4Config(*[a[f] for f in ("format", "n_entries", "n", "k", "swiglu", "out_type")])
    m = abi.WispFp4Mats(a["codes"], a["prepared"], None)
    x = abi.WispFp4Rows(a["xcodes"], P, None, a["rows"])
    _refused("wisp_b200_fp4_product", C.byref(cfg), C.byref(m), C.byref(m) if a["up"] else None,
             C.byref(x), a["segs"], a["n_segs"], a["out"], a["ld"], None, None, match=match)


def test_mx_rows_have_no_tensor_scale():
    """Refused wherever rows are used, so that their values and their products cannot differ by
    a scale that only one of the two knows."""
    why = "MX rows have no tensor scale"
    _refused("wisp_b200_fp4_dequantize", P, P, 4, 64, MX, P, P, 1, 64, None, match=why)
    cfg = abi.WispFp4Config(MX, 2, 64, 64, 0, 1)
    m, x = abi.WispFp4Mats(P, P, P), abi.WispFp4Rows(P, P, P, 3)
    _refused("wisp_b200_fp4_product", C.byref(cfg), C.byref(m), None, C.byref(x), P, 2, P, 64, None,
             None, match=why)
    with pytest.raises(RuntimeError, match=rf"wisp engine error \[4\].*{why}"):
        fp4.Fp4Rows(MX, torch.zeros(2, 32, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.uint8),
                    torch.ones(1))


def test_prepare_sizes_and_refusals():
    cfg = abi.WispFp4Config(MX, 3, 130, 288, 0, 1)
    n = abi.lib().wisp_b200_fp4_prepared_bytes(C.byref(cfg))
    assert n == 3 * 2 * 2 * 1024      # entries x feature tiles x 256-k stages x 2 words of 512
    cfg.format = NV
    assert abi.lib().wisp_b200_fp4_prepared_bytes(C.byref(cfg)) == 2 * n
    _refused("wisp_b200_fp4_prepare", C.byref(cfg), P, P, 2 * n - 1, None, match="required")
    _refused("wisp_b200_fp4_prepare", C.byref(cfg), P, P + 16, 2 * n, None, match="256-byte")
    _refused("wisp_b200_fp4_prepare", C.byref(cfg), None, P, 2 * n, None, match="null")
    cfg.k = 40
    assert abi.lib().wisp_b200_fp4_prepared_bytes(C.byref(cfg)) == 0


def test_moe_refusals():
    cfg = abi.WispMoeConfig()
    cfg.tokens, cfg.hidden, cfg.inter, cfg.n_experts, cfg.top_k = 4, 256, 128, 8, 2
    L = abi.lib()
    need = L.wisp_b200_fp4_moe_workspace_bytes(C.byref(cfg), MX)    # group_size 0: not used
    assert need > 0 and L.wisp_b200_fp4_moe_workspace_bytes(C.byref(cfg), 7) == 0
    w = abi.WispFp4MoeWeights()
    w.router_w, w.format = P, NV
    call = lambda ws: ("wisp_b200_fp4_moe_forward", C.byref(cfg), C.byref(w), P, P, None, None, P, ws,
                       None, None)
    _refused(*call(need * 4), match="x_scale")
    w.format = MX
    _refused(*call(need - 1), match="workspace")
    cfg.top_k = 9
    _refused(*call(need), match="top_k")
    assert L.wisp_b200_fp4_moe_workspace_bytes(C.byref(cfg), MX) == 0


def test_python_refusals():
    x = torch.zeros(2, 64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        fp4.quantize(x, MX)
    for bad in (lambda: fp4.quantize(x, 5), lambda: fp4.quantize(x[:, :40], MX),
                lambda: fp4.quantize(x.t(), MX), lambda: fp4.quantize(x, NV),
                lambda: fp4.quantize(x.double(), MX),
                lambda: fp4.quantize(x, MX, rows=torch.zeros(2, dtype=torch.int64)),
                lambda: fp4.Fp4Rows(MX, torch.zeros(2, 32, dtype=torch.uint8),
                                    torch.zeros(2, 4, dtype=torch.uint8)),
                lambda: fp4.Fp4Weights(MX, torch.zeros(2, 32, dtype=torch.uint8),
                                       torch.zeros(2, 2, dtype=torch.uint8)),
                lambda: fp4.Fp4Weights(MX, torch.zeros(1, 2, 32, dtype=torch.uint8),
                                       torch.zeros(1, 2, 2, dtype=torch.uint8), up=(x,)),
                lambda: norm.block_norm(x, pre=False), lambda: norm.block_norm(x, gate=x),
                lambda: norm.block_norm(x, x, gate=x[:, :3]),
                lambda: norm.block_norm(x, x, post=False, post_weight=x[0]),
                lambda: norm.block_norm(x, x.t())):
        with pytest.raises(RuntimeError, match=r"wisp engine error \[4\]"):
            bad()


def test_counts_past_32_bits_are_refused():
    """The ABI's counts are 32-bit ints: larger ones are refused, not cut off, and so are those
    that a kernel would round up past 2^31."""
    most, over = 0x7FFFFF00, 0x7FFFFF01
    _refused("wisp_b200_fp4_quantize", P, 1, 16, 4, P, over, 16, NV, P, P, P, None, match="2\\^31")
    _refused("wisp_b200_fp4_dequantize", P, P, over, 32, MX, None, P, 1, 32, None, match="2\\^31")
    cfg, m = abi.WispFp4Config(MX, 1, 1, 32, 0, 1), abi.WispFp4Mats(P, P, None)
    for rows, why in ((over, "2\\^31"), (most, "null")):
        x = abi.WispFp4Rows(P, P, None, rows)
        _refused("wisp_b200_fp4_product", C.byref(cfg), C.byref(m), None, C.byref(x), None, 0, None, 1,
                 None, None, match=why)
    c = abi.WispBlockNorm(tokens=over, hidden=1, ld_x=1, ld_n=1, n_type=1, x_type=1)
    _refused("wisp_b200_block_norm", C.byref(c), P, None, None, None, None, None, P, None,
             match="2\\^31")
    big = lambda *s, dtype=torch.bfloat16: torch.empty(s, dtype=dtype, device="meta")
    u8, n = torch.uint8, 2 ** 32 + 4
    for call in (lambda: fp4.quantize(big(n, 32), MX),
                 lambda: fp4.quantize(big(4, 32), MX, rows=big(n, dtype=torch.int32)),
                 lambda: fp4.Fp4Rows(MX, big(n, 16, dtype=u8), big(n, 1, dtype=u8)),
                 lambda: fp4.Fp4Weights(MX, big(n, 1, 16, dtype=u8), big(n, 1, 1, dtype=u8)),
                 lambda: norm.block_norm(big(n, 1)), lambda: norm.block_norm(big(4, n))):
        with pytest.raises(RuntimeError, match=r"wisp engine error \[4\].*2\^31"):
            call()


def test_quantize_has_no_gradient():
    x, ts = torch.zeros(2, 64), torch.ones(1)
    for a, b in ((x.clone().requires_grad_(), ts), (x, ts.clone().requires_grad_())):
        with pytest.raises(RuntimeError, match=r"wisp engine error \[4\].*gradient"):
            fp4.quantize(a, NV, b)
        with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU path"):
            fp4.quantize(a, NV, b)


# ---------------------------------------------------------------------------
# Quantisation
# ---------------------------------------------------------------------------
def _ts(v):
    return torch.tensor([v], dtype=torch.float32, device=DEV)


def _check_quantize(x, fmt, ts=None, rows=None, src=None):
    q = fp4.quantize(x, fmt, ts, rows=rows)
    c, sb = ref.quantize(x if src is None else src, fmt, ts)
    assert torch.equal(q.scales, sb)
    assert torch.equal(q.codes, c)
    return q


@pytest.mark.gpu
@FMTS
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("rows,cols", [(1, 32), (1, 7168), (3, 2080), (37, 96), (128, 4128)])
def test_quantize_and_back(fmt, dtype, rows, cols):
    g = torch.Generator(device=DEV).manual_seed(rows * cols)
    x = torch.randn((rows, cols), generator=g, device=DEV)
    x = (x * torch.exp2(torch.randint(-9, 10, (rows, 1), generator=g, device=DEV).float())).to(DT[dtype])
    ts = fp4.tensor_scale(x) if fmt == NV else None
    q = _check_quantize(x, fmt, ts)
    want = ref.values(q.codes, q.scales, fmt, ts)
    for out in DT.values():
        got = fp4.dequantize(q, out)
        # NV multiplies the exact code * scale by the tensor scale in fp32: 2^-24 more
        ref.check_rounded(got, want, want.abs() * (2.0 ** -24 if fmt == NV else 0.0))


@pytest.mark.gpu
def test_nv_values_next_to_borders():
    """Every border between two codes times every kind of scale, and its two fp32 neighbours:
    the decisions of exact arithmetic, where x times a reciprocal would miss some."""
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64)
    for g in (1.0, 0.1, 3.3e-5, 1.0 / 2688, 7.7e3):
        ts = _ts(g)
        gd = ts.double().item()
        top = torch.tensor([6.0 * s for s in (448, 416, 15, 1.125, 0.875, 2.0 ** -9)],
                           dtype=torch.float64) * gd
        rows = []
        for t in top:
            s = (t / 6).item()
            mid = (borders * s).float()
            for k in (-1, 0, 1):
                v = mid if k == 0 else torch.nextafter(mid, torch.full_like(mid, k * 3e38))
                rows.append(torch.cat([t.float().reshape(1), v, -v, torch.zeros(1)]))
        x = torch.stack(rows).to(DEV)
        _check_quantize(x, NV, ts)


@pytest.mark.gpu
def test_nv_scale_next_to_borders():
    """Block maxima at the midpoints of neighbouring e4m3 scales and their neighbours."""
    tab = ref.scale_values(torch.arange(0x7F), NV)
    mid = (tab[1:] + tab[:-1]) / 2
    for g in (1.0, 0.1, 3.3e-5):
        ts = _ts(g)
        top = (mid * 6 * ts.double().item()).float()
        top = torch.cat([top, torch.nextafter(top, torch.zeros_like(top)),
                         torch.nextafter(top, torch.full_like(top, 3e38)),
                         torch.tensor([0.0, 1e-30, 3e4, 3e38])])
        x = torch.zeros((top.numel(), 16))
        x[:, 3] = -top
        x[:, 9] = top * 0.3
        _check_quantize(x.to(DEV), NV, ts)


@pytest.mark.gpu
@FMTS
def test_quantize_extreme_blocks(fmt):
    """Zeros, signed zeros, subnormals, the largest values; infinities and NaN only spoil the
    block that they are in."""
    x = torch.zeros((9, 64))
    x[1, ::2] = -0.0
    x[2] = torch.linspace(-1, 1, 64) * 2.0 ** -140
    x[3] = torch.linspace(-1, 1, 64) * 3.4e38
    x[4, 5] = 2.0 ** -149
    x[5] = torch.arange(64) - 31.5
    x[5, 40] = float("inf")
    x[6] = torch.arange(64) - 31.5
    x[6, 3] = float("nan")
    x[7, 33] = float("-inf")
    x[8] = 2.0 ** -126
    for ts in [None] if fmt == MX else [_ts(1.0), _ts(1e-30), _ts(2.0 ** -149), _ts(1e36)]:
        q = _check_quantize(x.to(DEV), fmt, ts)
        v = fp4.dequantize(q)
        bad = torch.isnan(v)
        n = ref.BLOCK[fmt]
        want = torch.zeros_like(bad)
        for r, c in ((5, 40), (6, 3), (7, 33)):
            want[r, c // n * n:(c // n + 1) * n] = True
        assert torch.equal(bad, want)


@pytest.mark.gpu
@pytest.mark.parametrize("g", [0.0, -1.0, float("nan"), float("inf")])
def test_nv_unusable_tensor_scale(g):
    q = fp4.quantize(torch.ones((2, 32), device=DEV), NV, _ts(g))
    assert (q.scales == 0x7F).all() and (q.codes == 0).all()


@pytest.mark.gpu
@FMTS
def test_quantize_gathered_strided_and_unaligned(fmt):
    g = torch.Generator(device=DEV).manual_seed(3)
    big = torch.randn((40, 333), generator=g, device=DEV).to(torch.bfloat16)
    x = big[:, 5:5 + 96]                          # rows 666 bytes apart, 10 bytes off
    ts = _ts(0.002) if fmt == NV else None
    src = torch.tensor([3, 39, 0, 3, -1, 40, 1 << 30, 7], dtype=torch.int32, device=DEV)
    ok = (src >= 0) & (src < 40)
    want = torch.where(ok[:, None], x[src.clamp(0, 39).long()], torch.zeros_like(x[:1]))
    _check_quantize(x, fmt, ts, rows=src, src=want)
    _check_quantize(x, fmt, ts)
    wide = big[:, 8:8 + 96].float()               # aligned rows of another type
    _check_quantize(wide, fmt, ts)
    assert fp4.quantize(x, fmt, ts, rows=src[:0]).codes.shape == (0, 48)
    empty = fp4.quantize(x[:0], fmt, ts, rows=src)
    assert (empty.codes == 0).all() and (empty.scales == 0).all()


@pytest.mark.gpu
@FMTS
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("rows", [4737, 4738, 9475])     # 1, 2 and 3 left of fours, 1 of twos
@pytest.mark.parametrize("cols", [96, 2080])
def test_quantize_and_back_many_rows(fmt, dtype, rows, cols):
    """Enough rows that a thread takes several of them: as they lie, gathered (indices outside the
    input among them), and from rows that start anywhere."""
    g = torch.Generator(device=DEV).manual_seed(rows + cols)
    big = torch.randn((rows, cols + 13), generator=g, device=DEV)
    big *= torch.exp2(torch.randint(-9, 10, (rows, 1), generator=g, device=DEV).float())
    big = big.to(DT[dtype])
    x = big[:, :cols].contiguous()
    ts = fp4.tensor_scale(x) if fmt == NV else None
    q = _check_quantize(x, fmt, ts)
    want = ref.values(q.codes, q.scales, fmt, ts)
    for out in DT.values():
        ref.check_rounded(fp4.dequantize(q, out), want,
                          want.abs() * (2.0 ** -24 if fmt == NV else 0.0))
    apart = big[:, 5:5 + cols]
    _check_quantize(apart, fmt, ts)
    src = torch.randint(0, rows, (rows,), generator=g, device=DEV, dtype=torch.int32)
    src[::7], src[3::11], src[-1] = -1, rows, 1 << 30
    ok = (src >= 0) & (src < rows)
    for v in (x, apart):
        picked = torch.where(ok[:, None], v[src.clamp(0, rows - 1).long()], torch.zeros_like(v[:1]))
        _check_quantize(v, fmt, ts, rows=src, src=picked)


@pytest.mark.gpu
@FMTS
def test_quantize_past_32_bit_offsets(fmt):
    rows, cols = 301_000, 7168                    # 2.16e9 values
    x = torch.zeros((rows, cols), dtype=torch.bfloat16, device=DEV)
    x[-1] = torch.randn(cols, device=DEV).to(torch.bfloat16)
    ts = fp4.tensor_scale(x[-1:]) if fmt == NV else None
    q = fp4.quantize(x, fmt, ts)
    c, sb = ref.quantize(x[-1:], fmt, ts)
    assert torch.equal(q.codes[-1:], c) and torch.equal(q.scales[-1:], sb)
    assert not q.codes[:-1].any()
    tail = fp4.dequantize(q, torch.bfloat16)[-1:]
    v = ref.values(c, sb, fmt, ts)
    ref.check_rounded(tail, v, v.abs() * 2.0 ** -24)


# ---------------------------------------------------------------------------
# Product
# ---------------------------------------------------------------------------
def _mats(g, fmt, V, n, k):
    """Random codes of every kind, scales over a few binades, tensor scales."""
    codes = torch.randint(0, 256, (V, n, k // 2), generator=g, device=DEV, dtype=torch.uint8)
    lo, hi = (120, 130) if fmt == MX else (0x08, 0x7F)
    scales = torch.randint(lo, hi, (V, n, k // ref.BLOCK[fmt]), generator=g, device=DEV,
                           dtype=torch.uint8)
    ts = torch.rand((V,), generator=g, device=DEV) * 1e-3 + 1e-4 if fmt == NV else None
    return codes, scales, ts


def _rows(g, fmt, rows, k):
    x = torch.randn((rows, k), generator=g, device=DEV)
    return fp4.quantize(x, fmt, _ts(0.0015) if fmt == NV else None)


def _segs(counts, experts=None, start=0):
    at, out = start, []
    for i, r in enumerate(counts):
        out.append((i if experts is None else experts[i], at, r))
        at += r
    return out, torch.tensor([(*s, 0) for s in out], dtype=torch.int32, device=DEV)


def _run_product(fmt, swiglu, dtype, n, k, counts, V=None, experts=None, seed=1, extra=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    V = V or len(counts)
    mats = [_mats(g, fmt, V, n, k) for _ in range(2 if swiglu else 1)]
    if swiglu:   # gates of a few units, so that the sigmoid is not all 0 and 1
        mats[0] = (mats[0][0], (mats[0][1] - 6 if fmt == MX else mats[0][1] // 2), mats[0][2])
    q = _rows(g, fmt, sum(counts) + extra, k)
    w = fp4.Fp4Weights(fmt, *mats[0], up=mats[1] if swiglu else None)
    segs, dev = _segs(counts, experts)
    out = fp4.product(q, w, dev, dtype=dtype)
    w.check()
    ref.check_product(out, q, mats, segs, k)
    return q, w, mats, segs, dev, out


@pytest.mark.gpu
@FMTS
@pytest.mark.parametrize("swiglu", [False, True], ids=["plain", "swiglu"])
@pytest.mark.parametrize("n,k,counts", [
    (128, 256, [1]),                       # one stage, one tile
    (64, 32, [1, 0, 2]),                   # one block or two of K
    (1, 64, [5]),                          # one feature
    (257, 2080, [0, 7, 0, 0, 33, 1, 0]),   # ragged everything, empty experts
    (384, 1056, [16, 17, 31, 32, 33]),     # around the MMA's row granularity
    (130, 512, [191, 192, 193, 224, 225]),  # around the tile's row limits
    (200, 768, [700, 3, 1000]),            # several tiles a segment
    (128, 7168, [1, 1, 1, 1]),             # long sums
])
def test_product(fmt, swiglu, n, k, counts):
    for dtype in (torch.float32, torch.bfloat16):
        _run_product(fmt, swiglu, dtype, n, k, counts)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("k,rows", [(32, 1), (32, 200), (2048, 1), (2048, 40)])   # K whole, and split
def test_swiglu_of_large_gates(dtype, k, rows):
    """Gates at which exp(-g) is near the end of fp32's range or past it, and silu(g) is small but
    not 0, times an up value that brings it back. The gates are sums of few multiples of 1/2, so
    exact; a row of ones by 4-bit values."""
    gates = [0.0, 0.5, 20.0, 88.0, 100.0, -20.0, -86.5, -87.5, -88.0, -88.5, -89.0, -90.5, -95.0,
             -100.0, -103.0]
    codes = torch.zeros((1, len(gates), k), dtype=torch.uint8)
    for i, v in enumerate(gates):
        left, j = abs(v), 0
        while left:
            c = max(c for c in range(8) if ref.GRID[c] <= left)
            codes[0, i, j] = c + 8 * (v < 0)
            left, j = left - ref.GRID[c].item(), j + 1
        assert j <= 32
    pack = lambda c: (c[..., 0::2] | c[..., 1::2] << 4).contiguous().to(DEV)
    sc = lambda n, b: torch.full((n, len(gates), k // 32), b, dtype=torch.uint8, device=DEV)
    one = torch.zeros((1, len(gates), k), dtype=torch.uint8)
    one[..., 0] = 2
    w = fp4.Fp4Weights(MX, pack(codes), sc(1, 127), up=(pack(one), sc(1, 127 + 90)))
    x = torch.zeros((rows, k), dtype=torch.uint8)
    x[:, :32] = 2
    q = fp4.Fp4Rows(MX, pack(x), torch.full((rows, k // 32), 127, dtype=torch.uint8, device=DEV))
    out = fp4.product(q, w, dtype=DT[dtype]).double().cpu()
    g, u = torch.tensor(gates, dtype=torch.float64), 2.0 ** 90
    want = g * torch.sigmoid(g) * u
    # the exponential of half the gate (1 ulp, and twice for its square), two products, a sum, a
    # quotient (2 ulp) and the product with u: 8 times 2^-23. Below fp32's normal range the
    # products and the quotient round by half of 2^-149 each. A 16-bit output: half a step, and the
    # fast exponential's argument, |g| / 2 * log2(e) rounded to fp32, twice over: |g| 2^-23, with
    # a factor 2 for the instruction.
    tol = 8 * 2.0 ** -23 * want.abs() + 3 * 2.0 ** -150 * u
    if dtype == "bf16":
        tol = tol + (ref.half_step(torch.bfloat16) + g.abs() * 2.0 ** -22) * want.abs() * 1.001
    assert ((out - want).abs() <= tol).all()


@pytest.mark.gpu
@FMTS
def test_product_more_tiles_than_ctas(fmt):
    _run_product(fmt, False, torch.float16, 2200, 288, [1, 40, 260, 9] * 8)
    _run_product(fmt, True, torch.bfloat16, 2200, 288, [1, 40, 260, 9] * 8)


@pytest.mark.gpu
@FMTS
@pytest.mark.parametrize("k", [2080, 4128, 7168])
def test_product_long_rows_in_short_rings(fmt, k):
    """Tiles of many rows leave room for few stages of K, so that a warp's next turn at the row
    scales may lie two rounds of the ring ahead; repeated runs give the same bits."""
    for swiglu, n, counts in ((True, 1000, [510, 8, 0, 79, 333]), (False, 300, [450]), (True, 64, [190])):
        q, w, mats, segs, dev, out = _run_product(fmt, swiglu, torch.float32, n, k, counts)
        for _ in range(10):
            assert torch.equal(fp4.product(q, w, dev, dtype=torch.float32), out)
        w.check()


@pytest.mark.gpu
@FMTS
@pytest.mark.parametrize("swiglu", [False, True], ids=["plain", "swiglu"])
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("n,k,counts", [
    (3840, 2048, [1]),              # 30 feature tiles: K split by 2, four stages each
    (1000, 2080, [40, 3, 0, 9]),    # the same over ragged segments, nine stages as 4 and 5
    (6900, 1824, [17]),             # 54 feature tiles, the last of 116 features
    (200, 2080, [33, 7, 20]),       # by 4, several rounds of 16 rows
])
def test_product_split_over_k(fmt, swiglu, dtype, n, k, counts):
    _run_product(fmt, swiglu, DT[dtype], n, k, counts)


@pytest.mark.gpu
@FMTS
def test_product_many_segments_same_expert(fmt):
    """1025 segments, experts out of order and repeated."""
    counts = [(i * 7) % 4 for i in range(1025)]
    _run_product(fmt, False, torch.float32, 136, 160, counts, V=5,
                 experts=[(i * 3) % 5 for i in range(1025)])


@pytest.mark.gpu
@FMTS
def test_product_dense_is_one_segment(fmt):
    g = torch.Generator(device=DEV).manual_seed(2)
    mats = _mats(g, fmt, 1, 200, 544)
    w = fp4.Fp4Weights(fmt, *mats)
    for rows in (1, 2, 100, 500):
        q = _rows(g, fmt, rows, 544)
        out = fp4.product(q, w, dtype=torch.float32)
        ref.check_product(out, q, [mats], [(0, 0, rows)], 544)
    q = fp4.Fp4Rows(fmt, q.codes[:0], q.scales[:0], q.tensor_scale)
    assert fp4.product(q, w).shape == (0, 200)


@pytest.mark.gpu
@FMTS
def test_product_leaves_other_rows_and_columns(fmt):
    """Rows in no segment and the columns beside a strided output stay as they were."""
    g = torch.Generator(device=DEV).manual_seed(4)
    mats = _mats(g, fmt, 3, 100, 160)
    w = fp4.Fp4Weights(fmt, *mats)
    q = _rows(g, fmt, 60, 160)
    big = torch.full((60, 333), 7.0, device=DEV)
    segs = [(2, 3, 10), (0, 20, 0), (1, 30, 25)]
    fp4.product(q, w, torch.tensor([(*s, 0) for s in segs], dtype=torch.int32, device=DEV),
                out=big[:, 9:109])
    ref.check_product(big[:, 9:109], q, [mats], segs, 160)
    touched = torch.zeros_like(big, dtype=torch.bool)
    for _, r0, r in segs:
        touched[r0:r0 + r, 9:109] = True
    assert (big[~touched] == 7.0).all()


@pytest.mark.gpu
@FMTS
def test_product_of_no_segments(fmt):
    g = torch.Generator(device=DEV).manual_seed(14)
    w = fp4.Fp4Weights(fmt, *_mats(g, fmt, 2, 64, 64))
    out = torch.full((20, 64), 7.0, device=DEV)
    none = torch.empty((0, 4), dtype=torch.int32, device=DEV)
    for segs in (none, torch.zeros((3, 4), dtype=torch.int32, device=DEV)):
        fp4.product(_rows(g, fmt, 20, 64), w, segs, out=out)
        assert (out == 7.0).all()
    w.check()


@pytest.mark.gpu
@FMTS
def test_product_skips_bad_segments(fmt):
    g = torch.Generator(device=DEV).manual_seed(5)
    mats = _mats(g, fmt, 2, 64, 64)
    w = fp4.Fp4Weights(fmt, *mats)
    q = _rows(g, fmt, 20, 64)
    for bad in ((2, 0, 4), (-1, 0, 4), (0, 17, 4), (0, -1, 4), (1, 0, -3), (0, 2 ** 31 - 1, 2)):
        out = torch.full((20, 64), 7.0, device=DEV)
        segs = torch.tensor([(*bad, 0), (1, 8, 5, 0)], dtype=torch.int32, device=DEV)
        fp4.product(q, w, segs, out=out)
        ref.check_product(out, q, [mats], [(1, 8, 5)], 64)
        assert (out[:8] == 7.0).all() and (out[13:] == 7.0).all()
        with pytest.raises(RuntimeError, match=r"wisp engine error \[4\].*segment"):
            w.check()
        w.error_word.zero_()


@pytest.mark.gpu
def test_error_word_keeps_both_states():
    """A segment skipped (2) does not hide a wait that was given up (1), in whichever order they
    came; the wait is what a check reports of the two."""
    word = torch.zeros(1, dtype=torch.int32, device=DEV)
    check = lambda: abi.call("wisp_b200_check_error_flag", word.data_ptr(),
                             torch.cuda.current_stream().cuda_stream)
    check()
    for v, code, text in ((1, 7, "waiting"), (2, 4, "segment"), (3, 7, "waiting.*segment")):
        word.fill_(v)
        with pytest.raises(RuntimeError, match=rf"wisp engine error \[{code}\].*{text}"):
            check()
    g = torch.Generator(device=DEV).manual_seed(15)
    w = fp4.Fp4Weights(MX, *_mats(g, MX, 2, 64, 64))
    bad = torch.tensor([(2, 0, 4, 0)], dtype=torch.int32, device=DEV)
    for before, after in ((0, 2), (1, 3), (2, 2), (3, 3)):
        w.error_word.fill_(before)
        fp4.product(_rows(g, MX, 20, 64), w, bad)
        assert w.error_word.item() == after


@pytest.mark.gpu
def test_check_reports_once():
    """A check that raised clears what it reported: the products after it are judged by
    themselves."""
    g = torch.Generator(device=DEV).manual_seed(16)
    w = fp4.Fp4Weights(MX, *_mats(g, MX, 2, 64, 64))
    q = _rows(g, MX, 20, 64)
    good, bad = (torch.tensor([(e, 0, 4, 0)], dtype=torch.int32, device=DEV) for e in (1, 2))
    for _ in range(2):
        fp4.product(q, w, bad)
        with pytest.raises(RuntimeError, match=r"wisp engine error \[4\].*segment"):
            w.check()
        fp4.product(q, w, good)
        w.check()


@pytest.mark.gpu
@FMTS
def test_product_of_nonfinite_blocks(fmt):
    """A NaN scale spoils its row's or its feature's products only."""
    g = torch.Generator(device=DEV).manual_seed(6)
    codes, scales, ts = _mats(g, fmt, 1, 140, 96)
    scales[0, 133, 1] = 255 if fmt == MX else 0x7F
    w = fp4.Fp4Weights(fmt, codes, scales, ts)
    x = torch.randn((9, 96), generator=g, device=DEV)
    x[4, 70] = float("inf")
    q = fp4.quantize(x, fmt, _ts(0.002) if fmt == NV else None)
    bad = torch.isnan(fp4.product(q, w, dtype=torch.float32))
    want = torch.zeros_like(bad)
    want[4] = True
    want[:, 133] = True
    assert torch.equal(bad, want)


@pytest.mark.gpu
@FMTS
def test_product_on_streams_and_in_graphs(fmt):
    """Two streams at once, and two captured graphs that share the weights, give the bits of a
    call alone."""
    g = torch.Generator(device=DEV).manual_seed(7)
    mats = _mats(g, fmt, 4, 300, 544)
    w = fp4.Fp4Weights(fmt, *mats)
    _, segs = _segs([40, 0, 3, 200])
    qs = [_rows(g, fmt, 243, 544) for _ in range(2)]
    want = [fp4.product(q, w, segs, dtype=torch.float32) for q in qs]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        own = fp4.dequantize(qs[0])
    qs[0].record_stream(side)
    side.synchronize()
    assert torch.equal(own, fp4.dequantize(qs[0]))
    outs = [torch.zeros_like(want[0]) for _ in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    for _ in range(5):
        for q, o, s in zip(qs, outs, streams):
            with torch.cuda.stream(s):
                fp4.product(q, w, segs, out=o)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    graphs = []
    for q, o in zip(qs, outs):
        o.zero_()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            fp4.product(q, w, segs, out=o)
        graphs.append(gr)
    for _ in range(2):
        for o in outs:
            o.zero_()
        for gr, s in zip(graphs, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
    w.check()


@pytest.mark.gpu
@FMTS
def test_product_past_32_bit_offsets(fmt):
    """An output of more than 2^31 values."""
    g = torch.Generator(device=DEV).manual_seed(8)
    mats = _mats(g, fmt, 1, 4096, 32)
    w = fp4.Fp4Weights(fmt, *mats)
    rows = 530_000
    q = _rows(g, fmt, rows, 32)
    out = fp4.product(q, w, dtype=torch.bfloat16)
    w.check()
    for r0 in (0, 524_280, rows - 40):
        part = fp4.Fp4Rows(fmt, q.codes[r0:r0 + 40], q.scales[r0:r0 + 40], q.tensor_scale)
        ref.check_product(out[r0:r0 + 40], part, [mats], [(0, 0, 40)], 32)


@pytest.mark.gpu
def test_product_of_the_most_rows():
    """2^31 - 256 rows in one segment (34 GB of codes)."""
    rows = 0x7FFFFF00
    g = torch.Generator(device=DEV).manual_seed(18)
    mats = _mats(g, MX, 1, 1, 32)
    w = fp4.Fp4Weights(MX, *mats)
    codes = torch.zeros((rows, 16), dtype=torch.uint8, device=DEV)
    scales = torch.full((rows, 1), 127, dtype=torch.uint8, device=DEV)
    spots = (0, rows // 2, rows - 50)
    for r0 in spots:
        codes[r0:r0 + 50] = torch.randint(0, 256, (50, 16), generator=g, device=DEV, dtype=torch.uint8)
    out = fp4.product(fp4.Fp4Rows(MX, codes, scales), w, dtype=torch.bfloat16)
    w.check()
    for r0 in spots:
        part = fp4.Fp4Rows(MX, codes[r0:r0 + 50], scales[r0:r0 + 50])
        ref.check_product(out[r0:r0 + 50], part, [mats], [(0, 0, 50)], 32)
    assert int((out != 0).sum()) <= 150


@pytest.mark.gpu
@FMTS
def test_weights_from_values(fmt):
    g = torch.Generator(device=DEV).manual_seed(9)
    wv = torch.randn((3, 70, 96), generator=g, device=DEV).to(torch.bfloat16) * 0.02
    w = fp4.Fp4Weights.from_values(fmt, wv)
    q = _rows(g, fmt, 30, 96)
    segs, dev = _segs([10, 5, 15])
    out = fp4.product(q, w, dev, dtype=torch.float32)
    mats = []
    for e in range(3):
        ts = fp4.tensor_scale(wv[e]) if fmt == NV else None
        mats.append((*ref.quantize(wv[e], fmt, ts), ts))
    codes, scales = (torch.stack([m[i] for m in mats]) for i in (0, 1))
    ts = torch.cat([m[2] for m in mats]) if fmt == NV else None
    ref.check_product(out, q, [(codes, scales, ts)], segs, 96)


@pytest.mark.gpu
@FMTS
def test_products_have_no_gradient(fmt):
    """An output or an input that requires a gradient is refused under grad mode; weights are
    constants, laid out from parameters too."""
    g = torch.Generator(device=DEV).manual_seed(17)
    wv = torch.randn((2, 64, 96), generator=g, device=DEV)
    w = fp4.Fp4Weights.from_values(fmt, torch.nn.Parameter(wv))
    q, (_, segs) = _rows(g, fmt, 9, 96), _segs([4, 5])
    want = fp4.product(q, fp4.Fp4Weights.from_values(fmt, wv), segs, dtype=torch.float32)
    assert torch.equal(fp4.product(q, w, segs, dtype=torch.float32), want)
    out = torch.zeros((9, 64), device=DEV, requires_grad=True)
    why = r"wisp engine error \[4\].*gradient"
    with pytest.raises(RuntimeError, match=why):
        fp4.product(q, w, segs, out=out)
    with torch.no_grad():
        fp4.product(q, w, segs, out=out)
    assert torch.equal(out.detach(), want)
    layer = _layer(fmt, synth.MoeSpec("soft", 512, 256, 16, 4), 3)
    x = torch.randn((3, 512), device=DEV).to(torch.bfloat16).requires_grad_()
    with pytest.raises(RuntimeError, match=why):
        layer.forward(x)
    with torch.no_grad():
        y = layer.forward(x)
    assert torch.equal(y, layer.forward(x.detach()))


@pytest.mark.gpu
@FMTS
def test_up_without_tensor_scales(fmt):
    g = torch.Generator(device=DEV).manual_seed(10)
    (gc, gs, _), (uc, us, _) = _mats(g, fmt, 2, 64, 96), _mats(g, fmt, 2, 64, 96)
    q = _rows(g, fmt, 9, 96)
    segs, dev = _segs([4, 5])
    out, same = (fp4.product(q, fp4.Fp4Weights(fmt, gc, gs, up=up), dev, dtype=torch.float32)
                 for up in ((uc, us), (uc, us, None)))
    assert torch.equal(out.view(torch.int32), same.view(torch.int32))


# ---------------------------------------------------------------------------
# The MoE layer, and the block it stands in
# ---------------------------------------------------------------------------
def _layer(fmt, spec, tokens, seed=11):
    g = torch.Generator(device=DEV).manual_seed(seed)
    V = spec.n_virtual
    router = (torch.randn((spec.n_experts, spec.hidden), generator=g, device=DEV) * 0.05).to(torch.bfloat16)
    rnd = lambda n, k: torch.randn((V, n, k), generator=g, device=DEV) / k ** 0.5
    gu = fp4.Fp4Weights.from_values(fmt, rnd(spec.inter, spec.hidden), up=rnd(spec.inter, spec.hidden))
    dn = fp4.Fp4Weights.from_values(fmt, rnd(spec.hidden, spec.inter))
    xs, hs = (_ts(5.0 / 2688), _ts(6.0 / 2688)) if fmt == NV else (None, None)
    return fp4.Fp4MoeLayer(spec, router, None, gu, dn, tokens, x_scale=xs, h_scale=hs)


def _check_layer(layer, x, out, keep=slice(None)):
    """The layer's output against its own stages, each of which the tests above hold to 64 bits:
    the rows each token was routed to, quantised, multiplied, quantised, multiplied, and summed
    with the routing weights in 64 bits."""
    spec, T = layer.spec, x.shape[0]
    idx, wt = layer.idx.cpu().long(), layer.wt.double().cpu()
    rows = [[t for t in range(T) if (idx[t] == e).any()] for e in range(spec.n_experts)]
    if spec.has_shared:
        rows.append(list(range(T)))
    _, segs = _segs([len(r) for r in rows])
    tok = torch.tensor([t for r in rows for t in r], dtype=torch.int32, device=DEV)
    fmt = layer.gate_up.fmt
    xs, hs = layer._keep[2:]
    h = fp4.product(fp4.quantize(x, fmt, xs, rows=tok), layer.gate_up, segs, dtype=torch.bfloat16)
    y = fp4.product(fp4.quantize(h, fmt, hs), layer.down, segs, dtype=torch.bfloat16).double()
    wrow = torch.tensor([1.0 if e == spec.n_experts else wt[t][(idx[t] == e)].item()
                         for e, r in enumerate(rows) for t in r], dtype=torch.float64, device=DEV)
    want = torch.zeros((T, spec.hidden), dtype=torch.float64, device=DEV)
    mag = torch.zeros_like(want)
    want.index_add_(0, tok.long(), y * wrow[:, None])
    mag.index_add_(0, tok.long(), (y * wrow[:, None]).abs())
    # one fused multiply-add per row
    bound = (spec.top_k + 2) * 2.0 ** -24 * mag + 1e-30
    assert ((out.double() - want).abs() <= bound)[keep].all()


@pytest.mark.gpu
@FMTS
@pytest.mark.parametrize("tokens", [5, 700])   # rows quantised singly, and gathered
@pytest.mark.parametrize("shared", [False, True])
def test_moe_layer_nan_tokens_stay_apart(fmt, tokens, shared):
    """A token of NaN has no expert under softmax scores: the plan fills fewer rows, and what the
    workspace holds behind them is not followed."""
    spec = synth.MoeSpec("nan", 512, 256, 16, 4, has_shared=shared)
    layer = _layer(fmt, spec, tokens)
    layer.workspace.fill_(0x7f)
    x = torch.randn((tokens, spec.hidden), device=DEV).to(torch.bfloat16)
    bad = torch.zeros(tokens, dtype=torch.bool, device=DEV)
    bad[1::3] = True
    x[bad] = float("nan")
    out = layer.forward(x)
    layer.check()
    assert (layer.idx[bad] == -1).all() and (layer.idx[~bad] >= 0).all()
    _check_layer(layer, x, out, ~bad)
    assert out[bad].isnan().all() if shared else (out[bad] == 0).all()


@pytest.mark.gpu
@FMTS
@pytest.mark.parametrize("tokens", [1, 3, 64, 210, 300, 700])
def test_moe_layer(fmt, tokens):
    for spec in (synth.MoeSpec("soft", 512, 256, 16, 4, has_shared=True),
                 synth.MoeSpec("sig", 384, 128, 32, 4, scoring=abi.WISP_SCORE_SIGMOID_GROUPED,
                               n_groups=4, topk_groups=2, routed_scaling=2.5)):
        layer = _layer(fmt, spec, tokens)
        x = torch.randn((tokens, spec.hidden), device=DEV).to(torch.bfloat16)
        out = layer.forward(x)
        layer.check()
        _check_layer(layer, x, out)
        assert torch.equal(layer.forward(x), out)


@pytest.mark.gpu
@FMTS
@pytest.mark.parametrize("tokens", [1, 40, 1100])
def test_moe_layer_of_several_k_stages(fmt, tokens):
    """Row lengths of nine and five 256-k stages: K split for one token, a ring that goes round
    for the others."""
    layer = _layer(fmt, synth.MoeSpec("deep", 2304, 1152, 8, 2, has_shared=True), tokens)
    x = torch.randn((tokens, 2304), device=DEV).to(torch.bfloat16)
    out = layer.forward(x)
    layer.check()
    _check_layer(layer, x, out)
    assert torch.equal(layer.forward(x), out)


@pytest.mark.gpu
@FMTS
def test_blocks_of_norms_and_layers(fmt):
    """Two blocks as a model runs them (norm, MoE layer, norm of its output with gate and
    residual, next norm), eager and as one replayed graph, checked stage by stage."""
    spec = synth.MoeSpec("blk", 512, 256, 16, 4, has_shared=True)
    T, M = 24, spec.hidden
    layers = [_layer(fmt, spec, T, seed=s) for s in (21, 22)]
    g = torch.Generator(device=DEV).manual_seed(23)
    pre = [(1 + 0.1 * torch.randn(M, generator=g, device=DEV)).to(torch.bfloat16) for _ in range(3)]
    post = [(1 + 0.1 * torch.randn(M, generator=g, device=DEV)).to(torch.bfloat16) for _ in range(2)]
    gates = [torch.rand(M, generator=g, device=DEV) for _ in range(2)]

    def model(x, check=False):
        _, n = norm.block_norm(x, pre_weight=pre[0])
        for i, layer in enumerate(layers):
            y = layer.forward(n)
            if check:
                layer.check()
                _check_layer(layer, n, y)
            x2, n2 = norm.block_norm(x, y, gate=gates[i], residual_scale=0.9, post_weight=post[i],
                                     pre_weight=pre[i + 1])
            if check:
                xr, dx, nr, dn = ref.block_norm(x, y, gates[i], 0.9, post[i], pre[i + 1], True, True,
                                                1e-6, 0.0)
                ref.check_rounded(x2, xr, dx)
                ref.check_rounded(n2, nr, dn)
            x, n = x2, n2
        return x, n

    x0 = torch.randn((T, M), generator=g, device=DEV).to(torch.bfloat16)
    x, n = model(x0, check=True)
    static = torch.zeros_like(x0)
    gr = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(gr):
        gx, gn = model(static)
    for _ in range(2):
        static.copy_(x0)
        gr.replay()
        assert torch.equal(gx, x) and torch.equal(gn, n)
