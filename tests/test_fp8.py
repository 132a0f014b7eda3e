"""8-bit block-scaled rows, products and the MoE layer over them, against the format's
definition in 64 bits; refusals on the CPU."""
from __future__ import annotations

import ctypes as C
import os
import subprocess
import sys

import pytest
import torch

import fp4_ref
import fp8_ref as ref
from wisp_b200 import abi, fp4, fp8, norm, routing, synth

P = 1 << 20   # a non-null aligned stand-in pointer; never dereferenced here
DEV = "cuda"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
POW2 = pytest.mark.parametrize("pow2", [False, True], ids=["fp32", "pow2"])
SWIGLU = pytest.mark.parametrize("swiglu", [False, True], ids=["plain", "swiglu"])


# ---------------------------------------------------------------------------
# Refusals (no GPU)
# ---------------------------------------------------------------------------
def _refused(name, *args, match=""):
    with pytest.raises(RuntimeError, match=r"wisp engine error \[4\].*" + match):
        abi.call(name, *args)


@pytest.mark.parametrize("kw,match", [
    (dict(dt=3), "x_type"), (dict(cols=40), "cols"), (dict(cols=0), "cols"), (dict(ld=32), "ld"),
    (dict(cols=(1 << 27) + 16, ld=1 << 28), "2\\^27"), (dict(rows=-1), "rows"),
    (dict(rows=5), "d_src"), (dict(x=None), "null"), (dict(codes=P + 8), "aligned"),
    (dict(x=P + 1), "aligned"), (dict(scales=None), "null"), (dict(scales=P + 2), "aligned"),
    (dict(src=P + 2), "aligned"), (dict(srow=0), "strides"), (dict(sblock=0), "strides"),
    (dict(rows=0x7FFFFF01, src=P), "2\\^31"),
])
def test_quantize_refuses(kw, match):
    a = dict(x=P, dt=1, ld=64, x_rows=4, src=None, rows=4, cols=64, codes=P, scales=P, srow=1, sblock=4)
    a.update(kw)
    _refused("wisp_b200_fp8_quantize", a["x"], a["dt"], a["ld"], a["x_rows"], a["src"], a["rows"],
             a["cols"], 0, a["codes"], a["scales"], a["srow"], a["sblock"], None, match=match)


@pytest.mark.parametrize("kw,match", [
    (dict(dt=9), "out_type"), (dict(cols=24), "cols"), (dict(ld=63), "ld"), (dict(out=None), "null"),
    (dict(out=P + 2, dt=0), "aligned"), (dict(codes=P + 8), "aligned"),
    (dict(scales=P + 1), "aligned"), (dict(rows=0x7FFFFF01), "2\\^31"),
])
def test_dequantize_refuses(kw, match):
    a = dict(codes=P, scales=P, rows=4, cols=64, out=P, dt=1, ld=64)
    a.update(kw)
    _refused("wisp_b200_fp8_dequantize", a["codes"], a["scales"], 1, 4, a["rows"], a["cols"],
             a["out"], a["dt"], a["ld"], None, match=match)


@pytest.mark.parametrize("kw,match", [
    (dict(cols=24), "cols"), (dict(cols=0), "cols"), (dict(cols=(1 << 27) + 16), "2\\^27"),
    (dict(rows=-1), "rows"), (dict(rows=0x7FFFFF01), "2\\^31"), (dict(x_rows=-1), "x="),
    (dict(codes=None), "null"), (dict(scales=None), "null"), (dict(src=None), "null"),
    (dict(out=None), "null"), (dict(out_scales=None), "null"), (dict(codes=P + 8), "aligned"),
    (dict(scales=P + 2), "aligned"), (dict(src=P + 2), "aligned"), (dict(out=P + 8), "aligned"),
    (dict(out_scales=P + 1), "aligned"), (dict(srow=0), "strides"), (dict(sblock=0), "strides"),
])
def test_gather_refuses(kw, match):
    a = dict(codes=P, scales=P, x_rows=4, src=P, rows=4, cols=64, out=P, out_scales=P, srow=1, sblock=4)
    a.update(kw)
    x = abi.WispFp8Rows(a["codes"], a["scales"], 1, 4, a["x_rows"])
    _refused("wisp_b200_fp8_gather", C.byref(x), a["src"], a["rows"], a["cols"], a["out"],
             a["out_scales"], a["srow"], a["sblock"], None, match=match)


@pytest.mark.parametrize("kw,match", [
    (dict(dt=4), "out_type"), (dict(V=0), "n_entries"), (dict(n=0), "n=0"), (dict(k=24), "k=24"),
    (dict(V=65536), "65535"), (dict(n=65535 * 128 + 1), "65535"), (dict(w=None), "null"),
    (dict(codes=P + 4), "aligned"), (dict(w=P + 2, dt=0), "aligned"),
])
def test_quantize_weights_refuses(kw, match):
    a = dict(w=P, dt=1, V=2, n=64, k=64, codes=P, scales=P)
    a.update(kw)
    _refused("wisp_b200_fp8_quantize_weights", a["w"], a["dt"], a["V"], a["n"], a["k"], a["codes"],
             a["scales"], None, match=match)


def test_calls_without_rows_launch_nothing():
    abi.call("wisp_b200_fp8_quantize", None, 1, 64, 0, None, 0, 64, 0, None, None, 1, 1, None)
    abi.call("wisp_b200_fp8_dequantize", None, None, 1, 1, 0, 64, None, 1, 64, None)
    cfg = abi.WispFp8Config(2, 64, 64, 0, 1)
    m = abi.WispFp8Mats(P, P)
    x = abi.WispFp8Rows(None, None, 1, 1, 0)
    abi.call("wisp_b200_fp8_gather", C.byref(x), None, 0, 64, None, None, 1, 1, None)
    abi.call("wisp_b200_fp8_product", C.byref(cfg), C.byref(m), None, C.byref(x), None, 0, None, 64,
             None, None)


@pytest.mark.parametrize("kw,match", [
    (dict(k=24), "k=24"), (dict(k=(1 << 27) + 16), "2\\^27"), (dict(n=0), "n=0"),
    (dict(n_entries=0), "n_entries"), (dict(n_entries=1 << 16, n=1 << 16), "2\\^31"),
    (dict(out_type=3), "out_type"), (dict(swiglu=1), "up weights"), (dict(up=True), "without swiglu"),
    (dict(codes=P + 8), "aligned"), (dict(scales=P + 2), "aligned"), (dict(xcodes=P + 8), "aligned"),
    (dict(xscales=P + 1), "aligned"), (dict(xscales=None), "null"), (dict(out=None), "null"),
    (dict(out=P + 1), "aligned"), (dict(ld=63), "ld"), (dict(n_segs=1026), "n_segs"),
    (dict(n_segs=-1), "n_segs"), (dict(segs=None, n_segs=1), "n_segs"), (dict(rows=-1), "rows"),
    (dict(rows=0x7FFFFF01), "2\\^31"), (dict(codes=None), "null"), (dict(scales=None), "null"),
    (dict(segs=P + 2), "aligned"),
])
def test_product_refuses(kw, match):
    a = dict(n_entries=2, n=64, k=64, swiglu=0, out_type=1, codes=P, scales=P, up=False, xcodes=P,
             xscales=P, rows=3, segs=P, n_segs=2, out=P, ld=64)
    a.update(kw)
    cfg = abi.WispFp8Config(*[a[f] for f in ("n_entries", "n", "k", "swiglu", "out_type")])
    m = abi.WispFp8Mats(a["codes"], a["scales"])
    x = abi.WispFp8Rows(a["xcodes"], a["xscales"], 1, 4, a["rows"])
    _refused("wisp_b200_fp8_product", C.byref(cfg), C.byref(m), C.byref(m) if a["up"] else None,
             C.byref(x), a["segs"], a["n_segs"], a["out"], a["ld"], None, None, match=match)


def test_products_refuse_an_error_word_off_its_alignment():
    m8, m4 = abi.WispFp8Mats(P, P), abi.WispFp4Mats(P, P, None)
    for flag in (P + 1, P + 2):
        _refused("wisp_b200_fp8_product", C.byref(abi.WispFp8Config(2, 64, 64, 0, 1)), C.byref(m8), None,
                 C.byref(abi.WispFp8Rows(P, P, 1, 4, 3)), P, 2, P, 64, flag, None, match="aligned")
        _refused("wisp_b200_fp4_product",
                 C.byref(abi.WispFp4Config(abi.WISP_FP4_MX, 2, 64, 64, 0, 1)), C.byref(m4), None,
                 C.byref(abi.WispFp4Rows(P, P, None, 3)), P, 2, P, 64, flag, None, match="aligned")


def test_moe_refusals():
    cfg = abi.WispMoeConfig()
    cfg.tokens, cfg.hidden, cfg.inter, cfg.n_experts, cfg.top_k = 4, 256, 128, 8, 2
    r = routing.policy(n_groups=4, topk_groups=2)
    L = abi.lib()
    need = L.wisp_b200_fp8_moe_workspace_bytes(C.byref(cfg), C.byref(r))    # group_size 0: not used
    assert need > 0 and need == L.wisp_b200_fp8_moe_workspace_bytes(C.byref(cfg), None)
    w = abi.WispFp8MoeWeights()
    w.router_w = P

    def call(ws, rt=r, out=P, match=""):
        _refused("wisp_b200_fp8_moe_forward", C.byref(cfg), None if rt is None else C.byref(rt),
                 C.byref(w), P, out, None, None, P, ws, None, None, match=match)

    call(need - 1, match="workspace")
    call(need, out=P + 8, match="aligned")
    call(need, out=None, match="null")
    w.score_bias = P
    call(need, rt=None, match="score_bias")
    cfg.scoring = 5              # not used with a routing of its own
    assert L.wisp_b200_fp8_moe_workspace_bytes(C.byref(cfg), C.byref(r)) == need
    assert L.wisp_b200_fp8_moe_workspace_bytes(C.byref(cfg), None) == 0
    r.n_groups = 3
    call(need, match="n_groups")
    r.n_groups, cfg.top_k = 4, 9
    call(need, match="top_k")
    cfg.top_k, cfg.tokens = 2, 0x7FFFFFFF
    call(need, match="2\\^31")


@pytest.mark.parametrize("kw,match", [
    (dict(router_bias=P + 2), "router_bias"), (dict(score_bias=P + 1), "score_bias"),
    (dict(idx=P + 2), "topk_idx"), (dict(wt=P + 1), "topk_w"), (dict(flag=P + 2), "error word"),
    (dict(gate=(None, P)), "null pointer argument \\(gate"), (dict(up=(P, None)), "null.*\\(up"),
    (dict(down=(None, None)), "null.*\\(down"), (dict(gate=(P + 8, P)), "gate codes.*aligned"),
    (dict(up=(P, P + 2)), "up codes.*aligned"), (dict(down=(P + 4, P)), "down codes.*aligned"),
])
def test_moe_refuses_before_it_launches(kw, match):
    """What one of the layer's later steps would refuse, or a kernel would stumble over."""
    a = dict(router_bias=None, score_bias=None, idx=None, wt=None, flag=None, gate=(P, P), up=(P, P),
             down=(P, P))
    a.update(kw)
    cfg = abi.WispMoeConfig()
    cfg.tokens, cfg.hidden, cfg.inter, cfg.n_experts, cfg.top_k = 4, 256, 128, 8, 2
    r = routing.policy()
    w = abi.WispFp8MoeWeights()
    w.router_w, w.router_bias, w.score_bias = P, a["router_bias"], a["score_bias"]
    for name in ("gate", "up", "down"):
        setattr(w, name, abi.WispFp8Mats(*a[name]))
    _refused("wisp_b200_fp8_moe_forward", C.byref(cfg), C.byref(r), C.byref(w), P, P, a["idx"], a["wt"],
             P, 1 << 40, a["flag"], None, match=match)


def test_moe_workspace_of_sizes_past_the_products():
    cfg = abi.WispMoeConfig()
    cfg.tokens, cfg.n_experts, cfg.top_k = 1, 8, 2
    size = lambda: abi.lib().wisp_b200_fp8_moe_workspace_bytes(C.byref(cfg), None)
    for h, i, ok in ((1 << 27, 128, True), ((1 << 27) + 128, 128, False), (128, (1 << 27) + 128, False),
                     (1 << 26, 1 << 20, True)):
        cfg.hidden, cfg.inter = h, i
        assert (size() > 0) == ok
    cfg.n_experts, cfg.hidden, cfg.inter = 1024, 128, 1 << 21     # 2^31 rows of gate
    assert size() == 0


def test_moe_workspace_holds_copied_tokens_only_where_rows_are_copied():
    """A layer that quantises every row has no use for its tokens' codes, however many rows it has."""
    cfg = abi.WispMoeConfig()
    cfg.hidden, cfg.inter, cfg.n_experts = 2048, 128, 8

    def size(tokens):
        cfg.tokens = tokens
        return abi.lib().wisp_b200_fp8_moe_workspace_bytes(C.byref(cfg), None)

    # one token more: what it needs, and slack for parts that are rounded up to 256 bytes and for
    # the plan's counters; its codes and those of all before it would be 4 MB and more
    for top_k, shared in ((1, 0), (2, 0), (1, 1), (2, 1)):
        cfg.top_k, cfg.has_shared = top_k, shared
        for tokens in (1023, 2047, 4095, 8191):
            assert size(tokens + 1) - size(tokens) < 1 << 20
    cfg.top_k, cfg.has_shared = 4, 0               # 2^23 values of four rows a token: from 1024 on
    assert size(1024) - size(1023) > 1024 * 2048
    cfg.top_k, cfg.has_shared = 3, 1
    assert size(1024) - size(1023) > 1024 * 2048


def test_python_refusals():
    x = torch.zeros(2, 64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        fp8.quantize(x)
    u8, f8 = torch.uint8, torch.float8_e4m3fn
    z = lambda *s, dtype=torch.float32: torch.zeros(s, dtype=dtype)
    big = lambda *s, dtype=torch.bfloat16: torch.empty(s, dtype=dtype, device="meta")
    n = 2 ** 32 + 4
    for bad in (lambda: fp8.quantize(x[:, :40]), lambda: fp8.quantize(x.t()),
                lambda: fp8.quantize(x.double()),
                lambda: fp8.quantize(x, rows=torch.zeros(2, dtype=torch.int64)),
                lambda: fp8.quantize(x.clone().requires_grad_()),
                lambda: fp8.Fp8Rows(z(2, 32, dtype=u8), z(2, 2)),
                lambda: fp8.Fp8Rows(z(2, 32, dtype=u8), z(2, 1).double()),
                lambda: fp8.Fp8Rows(z(2, 24, dtype=u8), z(2, 1)),
                lambda: fp8.Fp8Rows(z(2, 32), z(2, 1)),
                lambda: fp8.Fp8Rows(z(32, 2, dtype=f8).t(), z(2, 1)),
                lambda: fp8.Fp8Weights(z(2, 32, dtype=f8), z(1, 1)),
                lambda: fp8.Fp8Weights(z(1, 200, 32, dtype=f8), z(1, 1, 1)),
                lambda: fp8.Fp8Weights(z(1, 64, 32, dtype=f8), z(1, 1, 1), up=(x,)),
                lambda: fp8.Fp8Weights(z(1, 64, 32, dtype=f8), z(1, 1, 1),
                                       up=(z(1, 64, 48, dtype=f8), z(1, 1, 1))),
                lambda: fp8.quantize_weights(x), lambda: fp8.quantize_weights(z(1, 2, 40)),
                lambda: fp8.quantize(big(n, 32)),
                lambda: fp8.quantize(big(4, 32), rows=big(n, dtype=torch.int32)),
                lambda: fp8.Fp8Rows(big(n, 32, dtype=u8), big(n, 1, dtype=torch.float32)),
                lambda: fp8.Fp8Weights(big(n, 1, 16, dtype=u8), big(n, 1, 1, dtype=torch.float32))):
        with pytest.raises(RuntimeError, match=r"wisp engine error \[4\]"):
            bad()
    with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU path"):
        fp8.quantize(x.clone().requires_grad_())


def test_scales_that_require_a_gradient_are_refused():
    codes = torch.zeros((2, 32), dtype=torch.uint8)
    for make in (lambda s: fp8.Fp8Rows(codes, s), lambda s: fp8.Fp8Weights(codes[None], s[None, :1])):
        with pytest.raises(RuntimeError, match=r"wisp engine error \[4\].*gradient"):
            make(torch.ones((2, 1), requires_grad=True))
    with torch.no_grad():
        assert fp8.Fp8Rows(codes, torch.ones((2, 1), requires_grad=True)).rows == 2


def test_codes_that_require_a_gradient_are_refused():
    codes = torch.zeros((2, 32), dtype=torch.float8_e4m3fn, requires_grad=True)
    plain, s = codes.detach(), torch.ones((2, 1))
    for make in (lambda c: fp8.Fp8Rows(c, s), lambda c: fp8.Fp8Weights(c[None], s[None, :1]),
                 lambda c: fp8.Fp8Weights(plain[None], s[None, :1], up=(c[None], s[None, :1]))):
        with pytest.raises(RuntimeError, match=r"wisp engine error \[4\].*gradient"):
            make(codes)
    with torch.no_grad():
        assert fp8.Fp8Rows(codes, s).rows == 2


# ---------------------------------------------------------------------------
# Quantisation
# ---------------------------------------------------------------------------
def _same_scales(got, want):
    assert torch.equal(torch.nan_to_num(got.double(), -1.0), torch.nan_to_num(want, -1.0))


def _check_quantize(x, pow2=False, rows=None, src=None):
    q = fp8.quantize(x, rows=rows, pow2=pow2)
    c, s = ref.quantize(x if src is None else src, pow2)
    _same_scales(q.scales, s)
    assert torch.equal(ref.unsigned_zeros(q.codes), c)
    return q


def _check_back(q):
    want = ref.row_values(q.codes, q.scales)
    for out in DT.values():
        # the product of code and scale is rounded to fp32 first
        first = 0.0 if out == torch.float32 else 2.0 ** -24
        fp4_ref.check_rounded(fp8.dequantize(q, out), want, want.abs() * first)


@pytest.mark.gpu
@POW2
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("rows,cols", [(1, 16), (1, 7168), (3, 2064), (37, 112), (128, 4112), (5, 128),
                                       (2, 240)])
def test_quantize_and_back(pow2, dtype, rows, cols):
    g = torch.Generator(device=DEV).manual_seed(rows * cols)
    x = torch.randn((rows, cols), generator=g, device=DEV)
    x = (x * torch.exp2(torch.randint(-9, 6, (rows, 1), generator=g, device=DEV).float())).to(DT[dtype])
    q = _check_quantize(x, pow2)
    assert torch.isfinite(q.scales).all()
    _check_back(q)


@pytest.mark.gpu
def test_values_next_to_borders():
    """Every border between two codes times scales of many mantissas, and its two fp32 neighbours:
    the decisions of exact arithmetic, where x times a reciprocal would miss some."""
    g = torch.Generator(device=DEV).manual_seed(1)
    grid = ref.grid("cpu")
    mid = (grid[1:] + grid[:-1]) / 2
    tops = torch.cat([torch.rand(60, generator=g, device=DEV).cpu() * 3 + 0.2,
                      torch.tensor([448.0, 1.0, 2.0 ** -100, 2.0 ** -117, 2.0 ** -125, 2.0 ** -130,
                                    3.3e38, 7.0 * 2.0 ** -140])])
    rows = []
    for top in tops:
        s = (top.double() / 448).float().double()
        v = (mid * s).float()
        for k in (-1, 0, 1):
            w = v if k == 0 else torch.nextafter(v, torch.full_like(v, k * 3.4e38))
            w = w.clamp(max=top.item())
            rows.append(torch.cat([top.reshape(1), w[:126], -top.reshape(1)]))
            rows.append(-rows[-1])
    x = torch.stack(rows).to(DEV)
    _check_quantize(x)
    _check_quantize(x, True)


@pytest.mark.gpu
def test_pow2_scales_next_to_borders():
    """Block maxima at 448 * 2^e, next to it and far from it, down to subnormals."""
    t = torch.cat([448.0 * torch.exp2(torch.arange(-160, 119).double()),
                   torch.exp2(torch.arange(-149, 128).double())])
    t = t[t > 0].float()
    t = torch.cat([t, torch.nextafter(t, torch.zeros_like(t)),
                   torch.nextafter(t, torch.full_like(t, 3.4e38)), torch.zeros(1)])
    t = t[torch.isfinite(t)]
    x = torch.zeros((t.numel(), 32))
    x[:, 3] = -t
    x[:, 9] = t * 0.3
    _check_quantize(x.to(DEV), True)
    _check_quantize(x.to(DEV), False)


@pytest.mark.gpu
@POW2
def test_quantize_extreme_blocks(pow2):
    """Zeros, signed zeros, subnormals, the largest values; infinities and NaN only spoil the
    block that they are in."""
    x = torch.zeros((9, 272))
    x[1, ::2] = -0.0
    x[2] = torch.linspace(-1, 1, 272) * 2.0 ** -140
    x[3] = torch.linspace(-1, 1, 272) * 3.4e38
    x[4, 5] = 2.0 ** -149
    x[5] = torch.arange(272) - 31.5
    x[5, 140] = float("inf")
    x[6] = torch.arange(272) - 31.5
    x[6, 3] = float("nan")
    x[7, 260] = float("-inf")
    x[8] = 2.0 ** -126
    q = _check_quantize(x.to(DEV), pow2)
    bad = torch.isnan(fp8.dequantize(q))
    want = torch.zeros_like(bad)
    for r, c in ((5, 140), (6, 3), (7, 260)):
        want[r, c // 128 * 128:(c // 128 + 1) * 128] = True
    assert torch.equal(bad, want)


@pytest.mark.gpu
def test_quantize_gathered_strided_and_unaligned():
    g = torch.Generator(device=DEV).manual_seed(3)
    big = torch.randn((40, 333), generator=g, device=DEV).to(torch.bfloat16)
    x = big[:, 5:5 + 144]                         # rows 666 bytes apart, 10 bytes off
    src = torch.tensor([3, 39, 0, 3, -1, 40, 1 << 30, 7], dtype=torch.int32, device=DEV)
    ok = (src >= 0) & (src < 40)
    want = torch.where(ok[:, None], x[src.clamp(0, 39).long()], torch.zeros_like(x[:1]))
    _check_quantize(x, rows=src, src=want)
    _check_quantize(x)
    wide = big[:, 8:8 + 144].float()              # aligned rows of another type
    _check_quantize(wide, True)
    none = fp8.quantize(x, rows=src[:0])
    assert none.codes.shape == (0, 144) and none.scales.shape == (0, 2)
    assert fp8.dequantize(none).shape == (0, 144)
    empty = fp8.quantize(x[:0], rows=src)
    assert not empty.codes.view(torch.uint8).any() and (empty.scales == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("rows", [4737, 4738, 9475])     # 1, 2 and 3 left of fours, 1 of twos
@pytest.mark.parametrize("cols", [112, 2064])
def test_quantize_and_back_many_rows(dtype, rows, cols):
    """Enough rows that a thread takes several of them: as they lie, gathered (indices outside the
    input among them), and from rows that start anywhere."""
    g = torch.Generator(device=DEV).manual_seed(rows + cols)
    big = torch.randn((rows, cols + 13), generator=g, device=DEV)
    big *= torch.exp2(torch.randint(-9, 10, (rows, 1), generator=g, device=DEV).float())
    big = big.to(DT[dtype])
    x = big[:, :cols].contiguous()
    q = _check_quantize(x)
    _check_back(q)
    _check_quantize(x, True)
    apart = big[:, 5:5 + cols]
    _check_quantize(apart)
    src = torch.randint(0, rows, (rows,), generator=g, device=DEV, dtype=torch.int32)
    src[::7], src[3::11], src[-1] = -1, rows, 1 << 30
    ok = (src >= 0) & (src < rows)
    for v in (x, apart):
        picked = torch.where(ok[:, None], v[src.clamp(0, rows - 1).long()], torch.zeros_like(v[:1]))
        _check_quantize(v, rows=src, src=picked)


@pytest.mark.gpu
@POW2
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("rows,cols", [(80_003, 16), (75_777, 144), (30_011, 272), (9_473, 1024),
                                       (5_000, 2048)])
def test_short_rows_several_to_a_block(pow2, dtype, rows, cols):
    g = torch.Generator(device=DEV).manual_seed(rows)
    x = torch.randn((rows, cols), generator=g, device=DEV).to(DT[dtype])
    q = _check_quantize(x, pow2)
    assert torch.equal(fp8.dequantize(q, DT[dtype]).double(),
                       ref.row_values(q.codes, q.scales).float().to(DT[dtype]).double())
    src = torch.randint(0, rows, (rows,), generator=g, device=DEV, dtype=torch.int32)
    got = fp8.gather(q, src)
    assert torch.equal(got.codes.view(torch.uint8), q.codes.view(torch.uint8)[src.long()])
    assert torch.equal(got.scales, q.scales[src.long()])


@pytest.mark.gpu
def test_dequantize_scales_of_any_strides():
    g = torch.Generator(device=DEV).manual_seed(20)
    for rows in (7, 3000):
        q = fp8.quantize(torch.randn((rows, 400), generator=g, device=DEV))
        want = fp8.dequantize(q)
        for s in (q.scales.contiguous(), torch.stack([q.scales, q.scales * 0], 2)[:, :, 0]):
            assert torch.equal(fp8.dequantize(fp8.Fp8Rows(q.codes, s)), want)


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [16, 112, 2064])
@pytest.mark.parametrize("rows", [0, 1, 9473, 9479])     # 1 and 7 left of eights
def test_gather(cols, rows):
    g = torch.Generator(device=DEV).manual_seed(rows + cols)
    n = 300
    codes = torch.randint(0, 256, (n, cols), generator=g, device=DEV, dtype=torch.uint8)
    wide = torch.rand((n, 2 * ref.blocks(cols) + 1), generator=g, device=DEV)
    scales = wide[:, 1::2]
    scales[3] = float("nan")
    src = torch.randint(-2, n + 2, (rows,), generator=g, device=DEV, dtype=torch.int32)
    if rows:
        src[0], src[-1] = 3, 2 ** 31 - 1
        src[rows // 2] = -2 ** 31
    got = fp8.gather(fp8.Fp8Rows(codes, scales), src)
    inside = ((src >= 0) & (src < n))[:, None]
    at = src.clamp(0, n - 1).long()
    assert torch.equal(got.codes.view(torch.uint8), torch.where(inside, codes[at], 0))
    _same_scales(got.scales, torch.where(inside, scales[at], 0.0).double())


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [70_001, 1_050_001], ids=["past the L2 cache", "past 32-bit offsets"])
def test_gather_of_large_results(rows):
    g = torch.Generator(device=DEV).manual_seed(28)
    q = fp8.quantize(torch.randn((700, 2064), generator=g, device=DEV))
    src = torch.randint(0, 702, (rows,), generator=g, device=DEV, dtype=torch.int32)
    got = fp8.gather(q, src)
    for r0 in (0, rows // 2, rows - 5000):
        at, s = slice(r0, r0 + 5000), src[r0:r0 + 5000].long()
        inside = (s < 700)[:, None]
        s = s.clamp(max=699)
        assert torch.equal(got.codes.view(torch.uint8)[at],
                           torch.where(inside, q.codes.view(torch.uint8)[s], 0))
        assert torch.equal(got.scales[at], torch.where(inside, q.scales[s], 0.0))


@pytest.mark.gpu
def test_gather_of_no_rows_gives_zeros():
    q = fp8.quantize(torch.ones((0, 64), device=DEV))
    for m in (5, 2 ** 19):             # (the second as a quantise of many rows does it)
        rows = torch.arange(m, device=DEV, dtype=torch.int32)
        for got in (fp8.gather(q, rows), fp8.quantize(torch.ones((0, 64), device=DEV), rows)):
            assert got.rows == m and not got.codes.view(torch.uint8).any() and not got.scales.any()


@pytest.mark.gpu
@POW2
@pytest.mark.parametrize("dtype", list(DT))
def test_quantize_of_rows_wanted_often(pow2, dtype):
    # 16,300 x 2064 values are enough for every row of x to be quantised once and copied
    g = torch.Generator(device=DEV).manual_seed(8)
    x = torch.randn((1100, 2064), generator=g, device=DEV).to(DT[dtype])[:1000]
    x[5, 7], x[6] = float("inf"), 0
    src = torch.randint(-3, 1003, (16300,), generator=g, device=DEV, dtype=torch.int32)
    src[:2] = torch.tensor([5, 6], device=DEV, dtype=torch.int32)
    many = fp8.quantize(x, src, pow2=pow2)
    for a in range(0, 16300, 3000):    # too few at a time for that
        few = fp8.quantize(x, src[a:a + 3000].clone(), pow2=pow2)
        assert torch.equal(many.codes.view(torch.uint8)[a:a + 3000], few.codes.view(torch.uint8))
        _same_scales(many.scales[a:a + 3000], few.scales.double())


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [900, 16300], ids=["singly", "copied"])
def test_quantize_on_streams_and_in_graphs(rows):
    """Two streams at once, and a graph that is replayed over other values, other indices and
    another graph's replays, give what a call alone gives."""
    g = torch.Generator(device=DEV).manual_seed(27)
    xs = [torch.randn((1000, 2064), generator=g, device=DEV).to(torch.bfloat16) for _ in range(2)]
    srcs = [torch.randint(-3, 1003, (rows,), generator=g, device=DEV, dtype=torch.int32) for _ in xs]
    run = lambda x, src: fp8.dequantize(fp8.quantize(x, src), torch.bfloat16)
    want = [run(x, s) for x, s in zip(xs, srcs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(3):
        got = []
        for x, src, s in zip(xs, srcs, streams):
            with torch.cuda.stream(s):
                got.append(run(x, src))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in xs:
        x, src, gr = xs[0].clone(), srcs[0].clone(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = run(x, src)
        graphs.append((gr, x, src, out))
    for order in ((0, 1), (1, 0)):
        for (gr, x, src, out), i in zip(graphs, order):
            x.copy_(xs[i])
            src.copy_(srcs[i])
        torch.cuda.synchronize()
        for (gr, *_), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, want[i]) for (_, _, _, out), i in zip(graphs, order))


@pytest.mark.gpu
def test_quantize_past_32_bit_offsets():
    rows, cols = 301_000, 7168                    # 2.16e9 values
    x = torch.zeros((rows, cols), dtype=torch.bfloat16, device=DEV)
    x[-1] = torch.randn(cols, device=DEV).to(torch.bfloat16)
    q = fp8.quantize(x)
    c, s = ref.quantize(x[-1:])
    assert torch.equal(ref.unsigned_zeros(q.codes[-1:]), c) and torch.equal(q.scales[-1:].double(), s)
    assert not q.codes[:-1].view(torch.uint8).any()
    tail = fp8.dequantize(q, torch.bfloat16)[-1:]
    v = ref.row_values(q.codes[-1:], s)
    fp4_ref.check_rounded(tail, v, v.abs() * 2.0 ** -24)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("V,n,k", [(1, 1, 16), (3, 300, 272), (2, 128, 128), (5, 129, 2064)])
def test_quantize_weights(dtype, V, n, k):
    g = torch.Generator(device=DEV).manual_seed(n)
    w = (torch.randn((V, n, k), generator=g, device=DEV) * 0.02).to(DT[dtype])
    w[V - 1, n - 1, k - 1] = float("inf")
    codes, scales = fp8.quantize_weights(w)
    nb, kb = ref.blocks(n), ref.blocks(k)
    pad = torch.zeros((V, nb * 128, kb * 128), dtype=torch.float64, device=DEV)
    pad[:, :n, :k] = w.double()
    b = pad.view(V, nb, 128, kb, 128).transpose(2, 3).reshape(V, nb, kb, -1)
    ok = torch.isfinite(b).all(-1)
    s = ref.scale_of(torch.where(ok, b.abs().amax(-1), 0 * b[..., 0]), False)
    c = ref.codes_of(b, s, ok).view(V, nb, kb, 128, 128).transpose(2, 3).reshape(V, nb * 128, -1)
    _same_scales(scales, torch.where(ok, s, torch.full_like(s, float("nan"))))
    assert torch.equal(ref.unsigned_zeros(codes), c[:, :n, :k])


# ---------------------------------------------------------------------------
# Product
# ---------------------------------------------------------------------------
def _mats(g, V, n, k, gain=1.0):
    """Random codes of every kind but NaN, scales over a few binades."""
    codes = torch.randint(0, 254, (V, n, k), generator=g, device=DEV, dtype=torch.uint8)
    codes += (codes >= 127).to(torch.uint8)
    scales = torch.exp2(torch.rand((V, ref.blocks(n), ref.blocks(k)), generator=g, device=DEV) * 5 - 14)
    return codes.view(torch.float8_e4m3fn), scales * gain


def _rows(g, rows, k):
    return fp8.quantize(torch.randn((rows, k), generator=g, device=DEV))


def _segs(counts, experts=None, start=0):
    at, out = start, []
    for i, r in enumerate(counts):
        out.append((i if experts is None else experts[i], at, r))
        at += r
    return out, torch.tensor([(*s, 0) for s in out], dtype=torch.int32, device=DEV)


def _check(out, q, mats, segs, k):
    ref.check_product(out, q.codes, q.scales, mats, segs, k)


def _run_product(swiglu, dtype, n, k, counts, V=None, experts=None, seed=1, extra=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    V = V or len(counts)
    # gates of a few units, so that the sigmoid is not all 0 and 1
    mats = [_mats(g, V, n, k, 60 / k ** 0.5 if swiglu and i == 0 else 1.0)
            for i in range(2 if swiglu else 1)]
    q = _rows(g, sum(counts) + extra, k)
    w = fp8.Fp8Weights(*mats[0], up=mats[1] if swiglu else None)
    segs, dev = _segs(counts, experts)
    out = fp8.product(q, w, dev, dtype=dtype)
    w.check()
    _check(out, q, mats, segs, k)
    return q, w, mats, segs, dev, out


@pytest.mark.gpu
@SWIGLU
@pytest.mark.parametrize("n,k,counts", [
    (128, 128, [1]),                       # one stage, one tile
    (64, 16, [1, 0, 2]),                   # part of a block of K
    (1, 64, [5]),                          # one feature
    (257, 2064, [0, 7, 0, 0, 33, 1, 0]),   # ragged everything, empty experts
    (384, 1056, [16, 17, 31, 32, 33]),     # around the MMA's row granularity
    (130, 512, [127, 128, 129, 255, 256, 257]),  # around the tiles' row limits
    (200, 768, [700, 3, 1000]),            # several tiles a segment, wide ones with a rest
    (128, 7168, [1, 1, 1, 1]),             # long sums
])
def test_product(swiglu, n, k, counts):
    for dtype in (torch.float32, torch.bfloat16):
        _run_product(swiglu, dtype, n, k, counts)


@pytest.mark.gpu
@SWIGLU
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("n,k,counts", [
    (1100, 1040, [600, 130, 90, 2, 385, 700, 256]),   # wide tiles, narrow ones between
    (2200, 288, [1, 40, 260, 9] * 8),                 # more tiles than CTAs
    (100, 144, [3000]),                               # one feature tile: single CTAs
    (1000, 400, [513]),
])
def test_product_of_wide_and_narrow_tiles(swiglu, dtype, n, k, counts):
    q, w, mats, segs, dev, out = _run_product(swiglu, DT[dtype], n, k, counts)
    for _ in range(5):
        assert torch.equal(fp8.product(q, w, dev, dtype=DT[dtype]), out)
    w.check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("k,rows", [(32, 1), (32, 200), (2048, 1), (2048, 40)])   # K whole, and split
def test_swiglu_of_large_gates(dtype, k, rows):
    """Gates at which exp(-g) is near the end of fp32's range or past it, and silu(g) is small but
    not 0, times an up value that brings it back."""
    gates = [0.0, 0.5, 20.0, 88.0, 100.0, -20.0, -86.5, -87.5, -88.0, -88.5, -89.0, -90.5, -95.0,
             -100.0, -103.0]
    codes = torch.zeros((1, len(gates), k))
    for i, v in enumerate(gates):      # exact sums of multiples of 8 and a rest that e4m3 holds
        whole = int(abs(v)) // 8 * 8
        codes[0, i, 0], codes[0, i, 1] = whole, abs(v) - whole
        codes[0, i] *= -1 if v < 0 else 1
    f8 = lambda t: t.to(torch.float8_e4m3fn)
    assert (f8(codes).float() == codes).all()
    sc = lambda v: torch.full((1, 1, ref.blocks(k)), v, device=DEV)
    one = torch.zeros((1, len(gates), k))
    one[..., 0] = 1
    w = fp8.Fp8Weights(f8(codes).to(DEV), sc(1.0), up=(f8(one).to(DEV), sc(2.0 ** 90)))
    x = torch.zeros((rows, k))
    x[:, :32] = 1
    q = fp8.Fp8Rows(f8(x).to(DEV), torch.ones((rows, ref.blocks(k)), device=DEV))
    out = fp8.product(q, w, dtype=DT[dtype]).double().cpu()
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
@SWIGLU
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("n,k,counts", [
    (3840, 2048, [1]),              # 30 feature tiles: K split, a few stages each
    (1000, 2080, [40, 3, 0, 9]),    # the same over ragged segments, 17 stages in uneven parts
    (6900, 2064, [17]),             # 54 feature tiles, the last of 116 features
    (200, 2080, [33, 7, 20]),       # several rounds of rows
    (128, 7168, [64]),
])
def test_product_split_over_k(swiglu, dtype, n, k, counts):
    _run_product(swiglu, DT[dtype], n, k, counts)


@pytest.mark.gpu
@SWIGLU
@pytest.mark.parametrize("n,k,counts", [
    (300, 4112, [9, 0, 30]),        # clusters of eight, 33 stages in uneven parts
    (1400, 4096, [1]),
    (60, 5120, [5, 22, 31]),        # one feature tile
    (250, 4128, [0, 63, 64, 1]),    # around the rows of a tile
])
def test_product_split_over_k_by_eight(swiglu, n, k, counts):
    for dtype in DT.values():
        q, w, mats, segs, dev, out = _run_product(swiglu, dtype, n, k, counts, extra=3)
        for _ in range(3):
            again = torch.full_like(out, 7.0)
            fp8.product(q, w, dev, out=again)
            assert torch.equal(again[:-3], out[:-3]) and (again[-3:] == 7.0).all()
        w.check()


@pytest.mark.gpu
@SWIGLU
@pytest.mark.parametrize("n,k,counts", [
    (121, 4608, [733]),             # tiles of 61 and 62 rows
    (300, 2080, [65, 0, 200, 3]),   # 17 stages
    (60, 2064, [129, 64, 128]),
    (128, 2048, [2900]),
    (4700, 2064, [9]),              # by three
    (2300, 2320, [20, 50]),
    (3100, 2576, [2]),              # by five
    (2000, 4000, [3]),              # by six, 32 stages
    (1100, 3616, [1]),              # by seven, 29 stages
    (7000, 2064, [16]),             # by two, 55 feature tiles
])
def test_product_split_over_k_by_any_number(swiglu, n, k, counts):
    for dtype in DT.values():
        q, w, mats, segs, dev, out = _run_product(swiglu, dtype, n, k, counts)
        for _ in range(3):
            assert torch.equal(fp8.product(q, w, dev, dtype=dtype), out)
        w.check()


@pytest.mark.gpu
@SWIGLU
@pytest.mark.parametrize("counts", [[65], [140], [193], [66, 193, 130]])
def test_product_split_over_k_by_cut_segments(swiglu, counts):
    """Segments cut into tiles of 48 rows (65: and 17; 140: and 44; 130: and 34; 66: and 18) and of
    64 (193: and one)."""
    for dtype in DT.values():
        q, w, mats, segs, dev, out = _run_product(swiglu, dtype, 121, 4608, counts)
        assert torch.equal(fp8.product(q, w, dev, dtype=dtype), out)
        w.check()


@pytest.mark.gpu
def test_product_many_segments_same_expert():
    """1025 segments, experts out of order and repeated."""
    counts = [(i * 7) % 4 for i in range(1025)]
    _run_product(False, torch.float32, 136, 160, counts, V=5,
                 experts=[(i * 3) % 5 for i in range(1025)])


@pytest.mark.gpu
def test_product_dense_is_one_segment():
    g = torch.Generator(device=DEV).manual_seed(2)
    mats = _mats(g, 1, 200, 544)
    w = fp8.Fp8Weights(*mats)
    for rows in (1, 2, 100, 500):
        q = _rows(g, rows, 544)
        out = fp8.product(q, w, dtype=torch.float32)
        _check(out, q, [mats], [(0, 0, rows)], 544)
        # scales of other strides give the same bits
        for s in (q.scales.contiguous(), torch.stack([q.scales, q.scales * 0], 2)[:, :, 0]):
            assert torch.equal(fp8.product(fp8.Fp8Rows(q.codes, s), w, dtype=torch.float32), out)
        assert torch.equal(fp8.product(fp8.Fp8Rows(q.codes.view(torch.uint8), q.scales), w,
                                       dtype=torch.float32), out)
    q = fp8.Fp8Rows(q.codes[:0], q.scales[:0])
    assert fp8.product(q, w).shape == (0, 200)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("sizes", [(3, 10, 30, 25), (5, 300, 310, 200)], ids=["narrow", "wide"])
def test_product_leaves_other_rows_and_columns(dtype, sizes):
    """Rows in no segment and the columns beside a strided output stay as they were."""
    a, ra, b, rb = sizes
    rows = b + rb + 5
    g = torch.Generator(device=DEV).manual_seed(4)
    mats = _mats(g, 3, 200, 160)
    w = fp8.Fp8Weights(*mats)
    q = _rows(g, rows, 160)
    segs = [(2, a, ra), (0, b - 1, 0), (1, b, rb)]
    dev = torch.tensor([(*s, 0) for s in segs], dtype=torch.int32, device=DEV)
    for at, ld in ((9, 333), (16, 336)):        # rows that start anywhere, and on 32 bytes
        big = torch.full((rows, ld), 7.0, device=DEV, dtype=DT[dtype])
        fp8.product(q, w, dev, out=big[:, at:at + 200])
        _check(big[:, at:at + 200], q, [mats], segs, 160)
        touched = torch.zeros_like(big, dtype=torch.bool)
        for _, r0, r in segs:
            touched[r0:r0 + r, at:at + 200] = True
        assert (big[~touched] == 7.0).all()


WIDE = (2200, [(2, 5, 300), (0, 310, 0), (1, 311, 200), (3, 520, 700), (0, 1230, 90)], 1340)


@pytest.mark.gpu
@SWIGLU
@pytest.mark.parametrize("dtype", list(DT))
def test_wide_tiles_leave_other_rows_and_columns(swiglu, dtype):
    """The same where there is enough for tiles of 256 rows: 1340 rows of 2200 features."""
    n, segs, rows = WIDE
    g = torch.Generator(device=DEV).manual_seed(24)
    mats = [_mats(g, 4, n, 400, 3.0 if swiglu and i == 0 else 1.0) for i in range(2 if swiglu else 1)]
    w = fp8.Fp8Weights(*mats[0], up=mats[1] if swiglu else None)
    q = _rows(g, rows, 400)
    dev = torch.tensor([(*s, 0) for s in segs], dtype=torch.int32, device=DEV)
    for at, ld in ((9, 2333), (16, 2336), (8, 2264)):
        big = torch.full((rows, ld), 7.0, device=DEV, dtype=DT[dtype])
        fp8.product(q, w, dev, out=big[:, at:at + n])
        _check(big[:, at:at + n], q, mats, segs, 400)
        touched = torch.zeros_like(big, dtype=torch.bool)
        for _, r0, r in segs:
            touched[r0:r0 + r, at:at + n] = True
        assert (big[~touched] == 7.0).all()
    w.check()


@pytest.mark.gpu
def test_wide_tiles_keep_nan_apart():
    """NaN in the rows beside a segment, in a row's and in a block of features' scales, and in a
    code, where tiles are of 256 rows."""
    n, segs, rows = WIDE
    g = torch.Generator(device=DEV).manual_seed(25)
    codes, scales = _mats(g, 4, n, 400)
    w = fp8.Fp8Weights(codes, scales)
    q = _rows(g, rows, 400)
    dev = torch.tensor([(*s, 0) for s in segs], dtype=torch.int32, device=DEV)
    out = fp8.product(q, w, dev, dtype=torch.float32)
    inside = torch.zeros(rows, dtype=torch.bool, device=DEV)
    for _, r0, r in segs:
        inside[r0:r0 + r] = True
    q.codes.view(torch.uint8)[~inside] = 0x7F
    q.scales[~inside] = float("nan")
    assert torch.equal(fp8.product(q, w, dev, dtype=torch.float32)[inside], out[inside])
    q.scales[600, 2] = q.scales[304, 3] = float("nan")
    scales[3, 17, 0] = float("nan")       # features 2176 .. 2199, the last block
    codes.view(torch.uint8)[2, 1000, 399] = 0xFF
    bad = torch.isnan(fp8.product(q, w, dev, dtype=torch.float32))
    want = torch.zeros_like(bad)
    want[600] = want[304] = True
    want[520:1220, 2176:] = True
    want[5:305, 1000] = True
    assert torch.equal(bad[inside], want[inside])
    w.check()


@pytest.mark.gpu
@SWIGLU
def test_wide_tiles_on_streams_and_in_graphs(swiglu):
    """Two streams at once and two replayed graphs, over scales of other strides, give the bits of
    a call alone."""
    n, segs, rows = WIDE
    g = torch.Generator(device=DEV).manual_seed(26)
    mats = [_mats(g, 4, n, 1040) for _ in range(2 if swiglu else 1)]
    w = fp8.Fp8Weights(*mats[0], up=mats[1] if swiglu else None)
    dev = torch.tensor([(*s, 0) for s in segs], dtype=torch.int32, device=DEV)
    qs = [_rows(g, rows, 1040) for _ in range(2)]
    same = fp8.Fp8Rows(qs[1].codes, qs[1].scales[:1].expand(rows, -1))        # one row's scales
    qs.append(fp8.Fp8Rows(same.codes, same.scales.contiguous()))
    want = [torch.zeros((rows, n), device=DEV, dtype=torch.bfloat16) for _ in qs]
    for q, o in zip(qs, want):
        fp8.product(q, w, dev, out=o)
    qs[2] = same
    outs = [torch.zeros_like(o) for o in want]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    for _ in range(3):
        for q, o, s in zip(qs, outs, streams):
            with torch.cuda.stream(s):
                fp8.product(q, w, dev, out=o)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    graphs = []
    for q, o in zip(qs, outs):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            fp8.product(q, w, dev, out=o)
        graphs.append(gr)
    for o in outs:
        o.zero_()
    torch.cuda.synchronize()
    for gr, s in zip(graphs, streams):
        with torch.cuda.stream(s):
            gr.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    w.check()


@pytest.mark.gpu
def test_product_of_no_segments():
    g = torch.Generator(device=DEV).manual_seed(14)
    w = fp8.Fp8Weights(*_mats(g, 2, 64, 64))
    out = torch.full((20, 64), 7.0, device=DEV)
    none = torch.empty((0, 4), dtype=torch.int32, device=DEV)
    for segs in (none, torch.zeros((3, 4), dtype=torch.int32, device=DEV)):
        fp8.product(_rows(g, 20, 64), w, segs, out=out)
        assert (out == 7.0).all()
    w.check()


@pytest.mark.gpu
def test_product_skips_bad_segments():
    g = torch.Generator(device=DEV).manual_seed(5)
    mats = _mats(g, 2, 64, 64)
    w = fp8.Fp8Weights(*mats)
    q = _rows(g, 20, 64)
    for bad in ((2, 0, 4), (-1, 0, 4), (0, 17, 4), (0, -1, 4), (1, 0, -3), (0, 2 ** 31 - 1, 2)):
        out = torch.full((20, 64), 7.0, device=DEV)
        segs = torch.tensor([(*bad, 0), (1, 8, 5, 0)], dtype=torch.int32, device=DEV)
        fp8.product(q, w, segs, out=out)
        _check(out, q, [mats], [(1, 8, 5)], 64)
        assert (out[:8] == 7.0).all() and (out[13:] == 7.0).all()
        with pytest.raises(RuntimeError, match=r"wisp engine error \[4\].*segment"):
            w.check()
        w.check()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [9, 300], ids=["narrow", "wide"])
def test_product_of_nonfinite_blocks(rows):
    """A NaN scale or code spoils its row's or its features' products only."""
    g = torch.Generator(device=DEV).manual_seed(6)
    codes, scales = _mats(g, 1, 400, 240)
    scales[0, 2, 1] = float("nan")
    codes.view(torch.uint8)[0, 33, 200] = 0x7F
    w = fp8.Fp8Weights(codes, scales)
    x = torch.randn((rows, 240), generator=g, device=DEV)
    x[4, 70] = float("inf")
    bad = torch.isnan(fp8.product(fp8.quantize(x), w, dtype=torch.float32))
    want = torch.zeros_like(bad)
    want[4] = True
    want[:, 33] = True
    want[:, 256:384] = True
    assert torch.equal(bad, want)


@pytest.mark.gpu
def test_rows_beside_a_segment_do_not_enter_it():
    """The rows around a segment's hold NaN: a tile reads past its rows, and uses none of it."""
    g = torch.Generator(device=DEV).manual_seed(19)
    mats = _mats(g, 1, 300, 272)
    w = fp8.Fp8Weights(*mats)
    for a, n in ((5, 3), (130, 150), (7, 300)):
        q = _rows(g, a + n + 200, 272)
        for r in (slice(0, a), slice(a + n, None)):
            q.codes.view(torch.uint8)[r] = 0x7F
            q.scales[r] = float("nan")
        out = fp8.product(q, w, torch.tensor([(0, a, n, 0)], dtype=torch.int32, device=DEV),
                          dtype=torch.float32)
        _check(out, q, [mats], [(0, a, n)], 272)


@pytest.mark.gpu
def test_product_on_streams_and_in_graphs():
    """Two streams at once, and two captured graphs that share the weights, give the bits of a
    call alone."""
    g = torch.Generator(device=DEV).manual_seed(7)
    mats = _mats(g, 4, 300, 544)
    w = fp8.Fp8Weights(*mats)
    _, segs = _segs([40, 0, 3, 200])
    qs = [_rows(g, 243, 544) for _ in range(2)]
    want = [fp8.product(q, w, segs, dtype=torch.float32) for q in qs]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        own = fp8.dequantize(qs[0])
    qs[0].record_stream(side)
    side.synchronize()
    assert torch.equal(own, fp8.dequantize(qs[0]))
    outs = [torch.zeros_like(want[0]) for _ in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    for _ in range(5):
        for q, o, s in zip(qs, outs, streams):
            with torch.cuda.stream(s):
                fp8.product(q, w, segs, out=o)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    graphs = []
    for q, o in zip(qs, outs):
        o.zero_()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            fp8.product(q, w, segs, out=o)
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
def test_first_calls_in_a_capture():
    """A process whose first calls are captured: what is asked of the device once is asked then."""
    code = """
import torch
from wisp_b200 import fp8, routing
codes = torch.randint(0, 120, (1, 2048, 4096), device="cuda", dtype=torch.uint8)
w = fp8.Fp8Weights(codes, torch.rand((1, 16, 32), device="cuda"))
x, l = torch.randn((1, 4096), device="cuda"), torch.randn((4, 64), device="cuda")
run = lambda: (fp8.product(fp8.quantize(x), w), *routing.select_experts(l, 4))
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = run()
graph.replay()
assert all(torch.equal(a, b) for a, b in zip(got, run()))
w.check()
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    subprocess.run([sys.executable, "-c", code], cwd=root, check=True, timeout=300)


@pytest.mark.gpu
def test_product_past_32_bit_offsets():
    """An output of more than 2^31 values."""
    g = torch.Generator(device=DEV).manual_seed(8)
    mats = _mats(g, 1, 4096, 32)
    w = fp8.Fp8Weights(*mats)
    rows = 530_000
    q = _rows(g, rows, 32)
    out = fp8.product(q, w, dtype=torch.bfloat16)
    w.check()
    for r0 in (0, 524_280, rows - 40):
        part = fp8.Fp8Rows(q.codes[r0:r0 + 40], q.scales[r0:r0 + 40])
        _check(out[r0:r0 + 40], part, [mats], [(0, 0, 40)], 32)


@pytest.mark.gpu
def test_product_of_the_most_rows():
    """2^31 - 256 rows in one segment (34 GB of codes)."""
    rows = 0x7FFFFF00
    g = torch.Generator(device=DEV).manual_seed(18)
    mats = _mats(g, 1, 1, 16)
    w = fp8.Fp8Weights(*mats)
    codes = torch.zeros((rows, 16), dtype=torch.uint8, device=DEV)
    scales = torch.ones((rows, 1), device=DEV)
    spots = (0, rows // 2, rows - 50)
    for r0 in spots:
        codes[r0:r0 + 50] = torch.randint(0, 127, (50, 16), generator=g, device=DEV, dtype=torch.uint8)
    out = fp8.product(fp8.Fp8Rows(codes, scales), w, dtype=torch.bfloat16)
    w.check()
    for r0 in spots:
        part = fp8.Fp8Rows(codes[r0:r0 + 50], scales[r0:r0 + 50])
        _check(out[r0:r0 + 50], part, [mats], [(0, 0, 50)], 16)
    assert int((out != 0).sum()) <= 150


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 8])
def test_weights_made_in_inference_mode_are_checked_outside(bits):
    """What check reports it clears, wherever the weights were made."""
    g = torch.Generator(device=DEV).manual_seed(10)
    values = torch.randn((2, 64, 64), generator=g, device=DEV)
    x = torch.randn((5, 64), generator=g, device=DEV)
    with torch.inference_mode():
        w = fp8.Fp8Weights.from_values(values) if bits == 8 else \
            fp4.Fp4Weights.from_values(abi.WISP_FP4_MX, values)
    q, product = (fp8.quantize(x), fp8.product) if bits == 8 else \
        (fp4.quantize(x, abi.WISP_FP4_MX), fp4.product)
    segs = torch.tensor([[7, 0, 2, 0], [1, 2, 3, 0]], dtype=torch.int32, device=DEV)     # no matrix 7
    for mode in (torch.no_grad, torch.inference_mode, torch.enable_grad):
        with mode():
            product(q, w, segs)
            with pytest.raises(RuntimeError, match=r"wisp engine error \[4\].*skipped"):
                w.check()
            w.check()


@pytest.mark.gpu
def test_weights_from_values_and_no_gradient():
    """An output that requires a gradient is refused under grad mode; weights are constants, taken
    from parameters too."""
    g = torch.Generator(device=DEV).manual_seed(9)
    wv = torch.randn((3, 70, 96), generator=g, device=DEV).to(torch.bfloat16) * 0.02
    w = fp8.Fp8Weights.from_values(torch.nn.Parameter(wv))
    q = _rows(g, 30, 96)
    segs, dev = _segs([10, 5, 15])
    want = fp8.product(q, w, dev, dtype=torch.float32)
    _check(want, q, [fp8.quantize_weights(wv)], segs, 96)
    pair = fp8.Fp8Weights.from_values(wv, up=wv)
    _check(fp8.product(q, pair, dev, dtype=torch.float32), q, [fp8.quantize_weights(wv)] * 2, segs, 96)
    out = torch.zeros((30, 70), device=DEV, requires_grad=True)
    with pytest.raises(RuntimeError, match=r"wisp engine error \[4\].*gradient"):
        fp8.product(q, w, dev, out=out)
    with torch.no_grad():
        fp8.product(q, w, dev, out=out)
    assert torch.equal(out.detach(), want)


# ---------------------------------------------------------------------------
# The MoE layer, and the block it stands in
# ---------------------------------------------------------------------------
def _layer(spec, tokens, seed=11, **kw):
    g = torch.Generator(device=DEV).manual_seed(seed)
    V = spec.n_virtual
    router = (torch.randn((spec.n_experts, spec.hidden), generator=g, device=DEV) * 0.05).to(torch.bfloat16)
    rnd = lambda n, k: torch.randn((V, n, k), generator=g, device=DEV) / k ** 0.5
    gu = fp8.Fp8Weights.from_values(rnd(spec.inter, spec.hidden), up=rnd(spec.inter, spec.hidden))
    dn = fp8.Fp8Weights.from_values(rnd(spec.hidden, spec.inter))
    bias = torch.randn(spec.n_experts, generator=g, device=DEV) * 0.1
    if kw.get("routing") is not None:
        kw["score_bias"] = bias
    return fp8.Fp8MoeLayer(spec, router, None, gu, dn, tokens, **kw)


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
    pow2 = bool(layer._w.pow2)
    h = fp8.product(fp8.quantize(x, rows=tok, pow2=pow2), layer.gate_up, segs, dtype=torch.bfloat16)
    y = fp8.product(fp8.quantize(h, pow2=pow2), layer.down, segs, dtype=torch.bfloat16).double()
    wrow = torch.tensor([1.0 if e == spec.n_experts else wt[t][(idx[t] == e)].item()
                         for e, r in enumerate(rows) for t in r], dtype=torch.float64, device=DEV)
    want = torch.zeros((T, spec.hidden), dtype=torch.float64, device=DEV)
    mag = torch.zeros_like(want)
    want.index_add_(0, tok.long(), y * wrow[:, None])
    mag.index_add_(0, tok.long(), (y * wrow[:, None]).abs())
    # one fused multiply-add per row
    bound = (spec.top_k + 2) * 2.0 ** -24 * mag + 1e-30
    assert ((out.double() - want).abs() <= bound)[keep].all()


def _check_layer_routing(layer, x):
    """The layer's choice against the logits in 64 bits: experts may only differ where their
    choices are closer than the logits' rounding moves them."""
    r = layer.routing
    router, _, bias = layer._keep
    l = x.double() @ router.double().T
    # products of bf16 are exact in fp32; the sums round by 2^-23 of the magnitudes a time
    moved = (x.shape[1] * 2.0 ** -23 * (x.double().abs() @ router.double().abs().T)).max().item()
    idx, w = ref.route(l, layer.spec.top_k, bias, r.scoring == abi.WISP_ROUTE_SOFTMAX, r.n_groups,
                       r.topk_groups, r.group_top, bool(r.renormalize), r.scaling)
    same = (layer.idx.cpu() == idx).all(1)
    assert same.float().mean() > 0.9
    d = (layer.wt.cpu().double() - w)[same].abs()
    # |d score / d logit| <= score, and the sum moves as much again
    assert (d <= (2 * moved + 2.0 ** -23) * w[same].abs() + 1e-30).all()


V3 = dict(n_groups=4, topk_groups=2, group_top=2, scaling=2.5)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 3, 64, 210, 300, 700])
def test_moe_layer(tokens):
    for spec, kw in (
            (synth.MoeSpec("soft", 512, 256, 16, 4, has_shared=True), {}),
            (synth.MoeSpec("sig", 384, 128, 32, 4, scoring=abi.WISP_SCORE_SIGMOID_GROUPED,
                           n_groups=4, topk_groups=2, routed_scaling=2.5), dict(pow2=True)),
            (synth.MoeSpec("bias", 512, 256, 32, 4, has_shared=True),
             dict(routing=routing.policy(abi.WISP_ROUTE_SIGMOID, **V3))),
            (synth.MoeSpec("softbias", 384, 128, 24, 3),
             dict(routing=routing.policy(abi.WISP_ROUTE_SOFTMAX, n_groups=4, topk_groups=2,
                                         group_top=1, renormalize=False)))):
        layer = _layer(spec, tokens, **kw)
        x = torch.randn((tokens, spec.hidden), device=DEV).to(torch.bfloat16)
        out = layer.forward(x)
        layer.check()
        _check_layer(layer, x, out)
        if layer.routing is not None:
            _check_layer_routing(layer, x)
        assert torch.equal(layer.forward(x), out)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [5, 700])   # rows quantised singly, and gathered
@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("own", [False, True], ids=["spec", "routing"])
def test_moe_layer_nan_tokens_stay_apart(tokens, shared, own):
    """A token of NaN has no expert: the plan fills fewer rows, and what the workspace holds behind
    them is not followed."""
    spec = synth.MoeSpec("nan", 512, 256, 16, 4, has_shared=shared)
    layer = _layer(spec, tokens, routing=routing.policy(**V3) if own else None)
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
@pytest.mark.parametrize("tokens", [1, 40, 1100])
def test_moe_layer_of_several_k_stages(tokens):
    """Row lengths of eighteen and nine 128-k stages: K split for one token, a ring that goes round
    for the others."""
    layer = _layer(synth.MoeSpec("deep", 2304, 1152, 8, 2, has_shared=True), tokens)
    x = torch.randn((tokens, 2304), device=DEV).to(torch.bfloat16)
    out = layer.forward(x)
    layer.check()
    _check_layer(layer, x, out)
    assert torch.equal(layer.forward(x), out)


def _check_choice(layer, x):
    """Every token's experts and weights against intervals of the 64-bit scores. A logit is a sum of
    products that are exact in fp32 (8 + 8 or 8 + 11 bits): at most `hidden` roundings and a few for
    the parts and the bias, each by 2^-23 of the terms' magnitudes (twice a rounding to nearest).
    With logits off by at most d, a sigmoid is off by at most d / 4 and a softmax by a factor
    e^(2 d). A choice is wrong where no scores within their intervals make it."""
    r, spec = layer.routing, layer.spec
    router, lbias, sbias = layer._keep
    w = router.double()
    l, mag = x.double() @ w.T, x.double().abs() @ w.T.abs()
    if lbias is not None:
        l, mag = l + lbias.double(), mag + lbias.double().abs()
    d = (spec.hidden + 16) * 2.0 ** -23 * mag
    if r.scoring == abi.WISP_ROUTE_SOFTMAX:
        s, f = torch.softmax(l, 1), torch.exp(2 * d.amax(1, keepdim=True))
        lo, hi = s / f, s * f
    else:
        s = torch.sigmoid(l)
        lo, hi = s - d / 4, s + d / 4
    b = torch.zeros_like(l) if sbias is None else sbias.double().expand_as(l)
    clo, chi = (lo + b - 1e-12).cpu(), (hi + b + 1e-12).cpu()
    lo, hi, idx, wt = lo.cpu(), hi.cpu(), layer.idx.cpu().long(), layer.wt.double().cpu()
    k, G, per = spec.top_k, r.n_groups, spec.n_experts // r.n_groups
    top = min(r.group_top, per)
    glo, ghi = (c.view(-1, G, per).topk(top, 2)[0].sum(2) for c in (clo, chi))
    for t in range(x.shape[0]):
        e = idx[t].tolist()
        assert len(set(e)) == k and min(e) >= 0 and max(e) < spec.n_experts
        assert all(chi[t, p] >= clo[t, q] for p, q in zip(e, e[1:])), (t, "order")
        used = {p // per for p in e}
        assert len(used) <= r.topk_groups
        for g in used:          # not surely behind as many groups as are kept
            assert sum((glo[t] > ghi[t, g]).tolist()) < r.topk_groups, (t, "group", g)
        for g in range(G):      # nothing is surely better and left out
            left = [p for p in range(g * per, (g + 1) * per) if p not in e and clo[t, p] > chi[t, e[-1]]]
            if left:
                assert g not in used, (t, "left out", left)
                others = sum(bool(ghi[t, h] >= glo[t, g]) for h in range(G) if h != g)
                assert others >= r.topk_groups, (t, "group left out", g)
        # the weights of these experts, whose scores carry no score bias
        a, z = lo[t, e].clamp(min=0), hi[t, e]
        if r.renormalize:
            a, z = a / (z.sum() - z + a), z / (a.sum() - a + z)
        eps = 2.0 ** -23
        assert (wt[t] >= a * r.scaling * (1 - eps)).all() and (wt[t] <= z * r.scaling * (1 + eps)).all(), t


CHOICES = {
    "sigmoid": dict(scoring=abi.WISP_ROUTE_SIGMOID, n_groups=4, topk_groups=2, scaling=2.5),
    "softmax": dict(scoring=abi.WISP_ROUTE_SOFTMAX, n_groups=8, topk_groups=3, group_top=1),
    "softmax as it is": dict(scoring=abi.WISP_ROUTE_SOFTMAX, renormalize=False),
}


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 4, 5, 64, 700])    # logits of a few tokens, by parts of K
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("policy", list(CHOICES))
def test_moe_layer_router_with_both_biases(policy, dtype, tokens):
    """One bias before the scores, one for the choice alone; either kind of router."""
    spec = synth.MoeSpec("biases", 1536, 128, 32, 4)
    g = torch.Generator(device=DEV).manual_seed(31)
    lbias = torch.randn(32, generator=g, device=DEV) * 0.7
    base = _layer(spec, tokens, routing=routing.policy(**CHOICES[policy]))
    router, _, sbias = base._keep
    x = torch.randn((tokens, spec.hidden), generator=g, device=DEV).to(torch.bfloat16)
    for lb, sb in ((lbias, sbias), (lbias, None), (None, sbias)):
        layer = fp8.Fp8MoeLayer(spec, router.to(DT[dtype]), lb, base.gate_up, base.down, tokens,
                                routing=base.routing, score_bias=sb)
        out = layer.forward(x)
        layer.check()
        _check_choice(layer, x)
        _check_layer(layer, x, out)
    if tokens >= 64:                   # the check tells the two biases apart
        layer._keep = (router, sbias, None)
        with pytest.raises(AssertionError):
            _check_choice(layer, x)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 4, 64, 700])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_moe_layer_without_a_routing_routes_as_the_other_layers(dtype, tokens):
    """The logits' bias and the router's type reach the routing that the layers share."""
    g = torch.Generator(device=DEV).manual_seed(32)
    lbias = torch.randn(32, generator=g, device=DEV) * 0.7
    for spec in (synth.MoeSpec("soft", 1536, 128, 32, 4),
                 synth.MoeSpec("sig", 1536, 128, 32, 4, scoring=abi.WISP_SCORE_SIGMOID_GROUPED, n_groups=4,
                               topk_groups=2, routed_scaling=2.5)):
        base = _layer(spec, tokens)
        router = base._keep[0].to(DT[dtype])
        layer = fp8.Fp8MoeLayer(spec, router, lbias, base.gate_up, base.down, tokens)
        x = torch.randn((tokens, spec.hidden), generator=g, device=DEV).to(torch.bfloat16)
        out = layer.forward(x)
        layer.check()
        _check_layer(layer, x, out)
        w = abi.WispMoeWeights(router.data_ptr(), lbias.data_ptr(), None, None)
        nbytes = abi.lib().wisp_b200_route_workspace_bytes(C.byref(layer.cfg))
        ws = torch.empty(nbytes, dtype=torch.uint8, device=DEV)
        idx, wt = torch.empty_like(layer.idx), torch.empty_like(layer.wt)
        abi.call("wisp_b200_route_ws", C.byref(layer.cfg), C.byref(w), x.data_ptr(), None, idx.data_ptr(),
                 wt.data_ptr(), ws.data_ptr(), nbytes, torch.cuda.current_stream().cuda_stream)
        assert torch.equal(layer.idx, idx) and torch.equal(layer.wt, wt)
        base.forward(x)
        assert tokens < 64 or not torch.equal(base.idx, idx)


@pytest.mark.gpu
@POW2
@pytest.mark.parametrize("tokens", [1, 24])
def test_moe_layer_of_256_experts(pow2, tokens):
    """The shape whose times the documents give: 256 experts of 2 x 2048 x 7168 and a shared one,
    four of eight groups, eight experts a token. Every product against 64 bits, and the layer against
    these stages."""
    spec = synth.MoeSpec("large", 7168, 2048, 256, 8, has_shared=True)
    V = spec.n_virtual
    g = torch.Generator(device=DEV).manual_seed(41)

    def mats(n, k):
        codes = torch.randint(0, 256, (V, n, k), generator=g, device=DEV, dtype=torch.uint8)
        codes &= 0xBF                   # magnitudes below 2, none of them NaN
        scales = torch.rand((V, n // 128, k // 128), generator=g, device=DEV) * 2 / k ** 0.5
        return codes, scales

    sets = [mats(2048, 7168), mats(2048, 7168), mats(7168, 2048)]
    gate_up, down = fp8.Fp8Weights(*sets[0], up=sets[1]), fp8.Fp8Weights(*sets[2])
    router = (torch.randn((256, 7168), generator=g, device=DEV) * 0.02).to(torch.bfloat16)
    sbias = torch.randn(256, generator=g, device=DEV) * 0.05
    layer = fp8.Fp8MoeLayer(spec, router, None, gate_up, down, tokens, pow2=pow2, score_bias=sbias,
                            routing=routing.policy(n_groups=8, topk_groups=4, scaling=2.5))
    x = torch.randn((tokens, 7168), generator=g, device=DEV).to(torch.bfloat16)
    out = layer.forward(x)
    layer.check()
    assert torch.equal(layer.forward(x), out)
    _check_choice(layer, x)
    _check_layer(layer, x, out)
    # the stages that _check_layer goes through
    idx = layer.idx.cpu()
    rows = [[t for t in range(tokens) if e in idx[t].tolist()] for e in range(256)] + [list(range(tokens))]
    segs, dev = _segs([len(r) for r in rows])
    tok = torch.tensor([t for r in rows for t in r], dtype=torch.int32, device=DEV)
    q = _check_quantize(x, pow2, rows=tok, src=x[tok.long()])
    h = fp8.product(q, gate_up, dev, dtype=torch.bfloat16)
    _check(h, q, sets[:2], segs, 7168)
    q = _check_quantize(h, pow2)
    _check(fp8.product(q, down, dev, dtype=torch.bfloat16), q, sets[2:], segs, 2048)


@pytest.mark.gpu
@POW2
@pytest.mark.parametrize("shared", [False, True], ids=["routed", "shared"])
@pytest.mark.parametrize("hidden,tokens,top_k", [
    (512, 3277, 5), (512, 3276, 4), (1024, 2049, 4), (2048, 1023, 4), (2048, 3277, 5), (2048, 2060, 3),
    (2048, 2060, 1),
])
def test_moe_layer_rows_quantised_singly_and_copied(hidden, tokens, top_k, shared, pow2):
    """Both sides of where the layer copies its tokens' codes instead of quantising every row, for
    either kind of scale, with tokens of NaN, which have no rows."""
    spec = synth.MoeSpec("copy", hidden, 128, 16, top_k, has_shared=shared)
    layer = _layer(spec, tokens, pow2=pow2, routing=routing.policy(**V3))
    layer.workspace.fill_(0x7f)
    x = torch.randn((tokens, hidden), device=DEV).to(torch.bfloat16)
    bad = torch.zeros(tokens, dtype=torch.bool, device=DEV)
    bad[2::97] = True
    x[bad] = float("nan")
    out = layer.forward(x)
    layer.check()
    assert (layer.idx[bad] == -1).all() and (layer.idx[~bad] >= 0).all()
    _check_layer(layer, x, out, ~bad)
    assert out[bad].isnan().all() if shared else (out[bad] == 0).all()
    assert torch.equal(layer.forward(x)[~bad], out[~bad])


@pytest.mark.gpu
def test_layer_has_no_gradient():
    layer = _layer(synth.MoeSpec("soft", 512, 256, 16, 4), 3)
    x = torch.randn((3, 512), device=DEV).to(torch.bfloat16).requires_grad_()
    with pytest.raises(RuntimeError, match=r"wisp engine error \[4\].*gradient"):
        layer.forward(x)
    with torch.no_grad():
        y = layer.forward(x)
    assert torch.equal(y, layer.forward(x.detach()))


@pytest.mark.gpu
def test_blocks_of_norms_and_layers():
    """Two blocks as a model runs them (norm, MoE layer, norm of its output with gate and residual,
    next norm), eager and as one replayed graph."""
    spec = synth.MoeSpec("blk", 512, 256, 16, 4, has_shared=True)
    T, M = 24, spec.hidden
    layers = [_layer(spec, T, seed=s, routing=routing.policy(**V3)) for s in (21, 22)]
    g = torch.Generator(device=DEV).manual_seed(23)
    wts = [(1 + 0.1 * torch.randn(M, generator=g, device=DEV)).to(torch.bfloat16) for _ in range(3)]

    def model(x, check=False):
        _, n = norm.block_norm(x, pre_weight=wts[0])
        for i, layer in enumerate(layers):
            y = layer.forward(n)
            if check:
                layer.check()
                _check_layer(layer, n, y)
                _check_layer_routing(layer, n)
            x, n = norm.block_norm(x, y, post=False, pre_weight=wts[i + 1])
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
