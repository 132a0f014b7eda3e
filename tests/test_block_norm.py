"""The norms around a block against 64 bits; refusals on the CPU."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

import fp4_ref as ref
from wisp_b200 import abi, norm

P = 1 << 20   # a non-null aligned stand-in pointer; never dereferenced here
DEV = "cuda"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.mark.parametrize("kw,match", [
    (dict(tokens=-1), "tokens"), (dict(hidden=0), "hidden"), (dict(hidden=32769), "hidden"),
    (dict(x_type=3), "type"), (dict(n_type=-1), "type"), (dict(gate_kind=4), "gate_kind"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(xo=None, n=None), "output"),
    (dict(y=None), "without y"), (dict(gate_kind=0), "disagree"), (dict(gate=None), "disagree"),
    (dict(post_norm=0), "post_w"), (dict(n=None), "pre_w"), (dict(ld_x=63), "stride"),
    (dict(ld_y=63), "stride"), (dict(ld_n=0), "stride"), (dict(gate_kind=3, ld_gate=8), "stride"),
    (dict(x=None), "null"), (dict(x=P + 1), "aligned"), (dict(n=P + 1), "aligned"),
])
def test_refusals(kw, match):
    a = dict(tokens=4, hidden=64, x_type=1, y_type=0, w_type=1, gate_type=0, n_type=1, post_norm=1,
             gate_kind=1, residual_scale=1.0, eps=1e-6, weight_offset=0.0, ld_x=64, ld_y=64,
             ld_gate=64, ld_x_out=64, ld_n=64)
    ptr = dict(x=P, y=P, gate=P, post_w=P, pre_w=P, xo=P, n=P)
    for k, v in kw.items():
        (ptr if k in ptr else a)[k] = v
    c = abi.WispBlockNorm(**a)
    with pytest.raises(RuntimeError, match=r"wisp engine error \[4\].*" + match):
        abi.call("wisp_b200_block_norm", C.byref(c), *ptr.values(), None)


def test_in_place_needs_the_same_rows():
    c = abi.WispBlockNorm(tokens=2, hidden=8, x_type=1, n_type=1, ld_x=8, ld_y=8, ld_x_out=16, ld_n=8)
    with pytest.raises(RuntimeError, match=r"wisp engine error \[4\].*in place"):
        abi.call("wisp_b200_block_norm", C.byref(c), P, 2 * P, None, None, None, P, 3 * P, None)


def test_no_tokens_launch_nothing():
    c = abi.WispBlockNorm(tokens=0, hidden=64, ld_x=64, ld_n=64)
    abi.call("wisp_b200_block_norm", C.byref(c), P, None, None, None, None, None, P, None)

    # rows and a block's output of no tokens have no address
    c = abi.WispBlockNorm(tokens=0, hidden=64, post_norm=1, gate_kind=1, ld_x=64, ld_y=64,
                          ld_x_out=64, ld_n=64)
    abi.call("wisp_b200_block_norm", C.byref(c), None, None, P, P, P, None, None, None)


@pytest.mark.parametrize("which", ["x", "y", "gate", "post_weight", "pre_weight", "x_out", "n_out"])
def test_no_gradient(which):
    """A gradient that would be lost without a word is refused; without grad mode the call goes on
    (here to the refusal of CPU tensors)."""
    kw = dict(y=torch.ones(2, 8), gate=torch.ones(8), post_weight=torch.ones(8),
              pre_weight=torch.ones(8), x_out=torch.ones(2, 8), n_out=torch.ones(2, 8))
    x = torch.ones(2, 8)
    (x if which == "x" else kw[which]).requires_grad_()
    with pytest.raises(RuntimeError, match=r"wisp engine error \[4\].*gradient"):
        norm.block_norm(x, **kw)
    for mode in (torch.no_grad, torch.inference_mode):
        with mode(), pytest.raises(RuntimeError, match="no CPU path"):
            norm.block_norm(x, **kw)


@pytest.mark.gpu
def test_parameters_without_grad_mode():
    x = torch.randn(5, 64, device=DEV)
    w = torch.nn.Parameter(torch.rand(64, device=DEV))
    with torch.no_grad():
        got = norm.block_norm(x, x, post_weight=w, pre_weight=w)
    want = norm.block_norm(x, x, post_weight=w.detach(), pre_weight=w.detach())
    assert all(torch.equal(a, b) and not a.requires_grad for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [3, 400])
@pytest.mark.parametrize("M", [8184, 8192, 8193, 8200, 16376, 16383, 16384, 16385, 16392])
def test_wide_rows(T, M):
    _run(T, M)


@pytest.mark.gpu
def test_empty_batch():
    x, w = torch.empty((0, 64), device=DEV, dtype=torch.bfloat16), torch.ones(64, device=DEV)
    xo, n = norm.block_norm(x, x.float(), gate=w, post_weight=w, pre_weight=w)
    assert xo.shape == n.shape == (0, 64)
    assert norm.block_norm(x)[1].shape == (0, 64)


def _run(T, M, x="bf16", y="fp32", w="bf16", gate="channel", n="bf16", post=True, pre=True, rs=1.0,
         off=0.0, eps=1e-6, seed=0, scale=3.0):
    g = torch.Generator(device=DEV).manual_seed(seed + T * M)
    r = lambda *s: torch.randn(s, generator=g, device=DEV)
    X = r(T, M).to(DT[x])
    Y = (scale * r(T, M)).to(DT[y]) if y else None
    G = {"none": None, "channel": r(M), "token": r(T, 1), "element": r(T, M)}[gate]
    G = None if G is None else G.to(DT[w])
    pw = (1 - off + 0.1 * r(M)).to(DT[w]) if post and y else None
    qw = (1 - off + 0.1 * r(M)).to(DT[w]) if pre else None
    xo, no = norm.block_norm(X, Y, gate=G, residual_scale=rs, post_weight=pw, pre_weight=qw,
                             post=post, pre=pre, eps=eps, weight_offset=off, dtype=DT[n])
    xr, dx, nr, dn = ref.block_norm(X, Y, G, rs, pw, qw, post, pre, eps, off)
    if Y is None:
        assert xo is X
    else:
        assert xo.dtype == X.dtype
        ref.check_rounded(xo, xr, dx)
    if pre:
        assert no.dtype == DT[n]
        ref.check_rounded(no, nr, dn)
    else:
        assert no is None


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 5, 297])
@pytest.mark.parametrize("M", [1, 7, 8, 64, 248, 264, 520, 1000, 1024, 1032, 2077, 7168, 8193, 32761, 32768])
def test_sizes(T, M):
    _run(T, M)
    _run(T, M, y=None, gate="none", post=False, n="fp32")


@pytest.mark.gpu
@pytest.mark.parametrize("x", list(DT))
@pytest.mark.parametrize("y", list(DT))
@pytest.mark.parametrize("w", list(DT))
def test_types(x, y, w):
    for n in DT:
        _run(9, 264, x=x, y=y, w=w, n=n, rs=0.7)


@pytest.mark.gpu
@pytest.mark.parametrize("gate", ["none", "channel", "token", "element"])
@pytest.mark.parametrize("post,pre", [(True, True), (True, False), (False, True), (False, False)])
def test_parts(gate, post, pre):
    for T, M in ((3, 520), (400, 77)):
        _run(T, M, gate=gate, post=post, pre=pre, rs=-0.5, off=1.0)


@pytest.mark.gpu
def test_without_weights_and_eps():
    X, Y = torch.randn(4, 96, device=DEV), torch.randn(4, 96, device=DEV)
    X[2] = Y[2] = 0.0
    for eps in (1e-6, 0.0, 1.0):
        xo, no = norm.block_norm(X, Y, eps=eps, dtype=torch.float32)
        xr, dx, nr, dn = ref.block_norm(X, Y, None, 1.0, None, None, True, True, eps, 0.0)
        keep = [0, 1, 3] if eps == 0.0 else [0, 1, 2, 3]   # 0 / 0 on the all-zero row
        ref.check_rounded(xo[keep], xr[keep], dx[keep])
        ref.check_rounded(no[keep], nr[keep], dn[keep])


@pytest.mark.gpu
def test_strides_offsets_and_in_place():
    g = torch.Generator(device=DEV).manual_seed(1)
    big = torch.randn((3, 11, 217), generator=g, device=DEV).to(torch.bfloat16)
    X, Y, G = (big[i, :, 3:203] for i in range(3))      # odd strides, 6 bytes off
    xr, dx, nr, dn = ref.block_norm(X, Y, G, 1.0, None, None, True, True, 1e-6, 0.0)
    out = torch.full((11, 300), 7.0, device=DEV, dtype=torch.float16)
    xo, no = norm.block_norm(X, Y, gate=G, x_out=X, n_out=out[:, 1:201])
    assert xo.data_ptr() == X.data_ptr()
    ref.check_rounded(X, xr, dx)
    ref.check_rounded(no, nr, dn)
    assert (out[:, :1] == 7.0).all() and (out[:, 201:] == 7.0).all()
    assert torch.equal(big[0, :, :3], big[0, :, :3]) and no.data_ptr() == out[:, 1:].data_ptr()


@pytest.mark.gpu
def test_nonfinite_rows_stay_apart():
    X, Y = torch.randn(5, 64, device=DEV), torch.randn(5, 64, device=DEV)
    Y[1, 3], X[3, 5] = float("nan"), float("inf")
    xo, no = norm.block_norm(X, Y, dtype=torch.float32)
    ok = [0, 2, 4]
    xr, dx, nr, dn = ref.block_norm(X[ok], Y[ok], None, 1.0, None, None, True, True, 1e-6, 0.0)
    ref.check_rounded(xo[ok], xr, dx)
    ref.check_rounded(no[ok], nr, dn)
    assert torch.isnan(xo[1]).all() and torch.isnan(no[1]).all()


@pytest.mark.gpu
def test_past_32_bit_offsets():
    T, M = 262_500, 8192                                 # 2.15e9 values
    X = torch.ones((T, M), dtype=torch.bfloat16, device=DEV)
    X[-2:] = torch.randn((2, M), device=DEV).to(torch.bfloat16)
    _, n = norm.block_norm(X)
    _, _, nr, dn = ref.block_norm(X[-2:], None, None, 1.0, None, None, False, True, 1e-6, 0.0)
    ref.check_rounded(n[-2:], nr, dn)


@pytest.mark.gpu
def test_streams():
    X, Y = torch.randn(300, 1024, device=DEV), torch.randn(300, 1024, device=DEV)
    want = norm.block_norm(X, Y)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = norm.block_norm(X, Y)
    s.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# Rows and columns at which every CTA of the many-row form goes through its ring of rows more than
# twice, with a last round that only some of the CTAs have: 17 rows each through 4 slots (7168),
# 14 through 5 (3373, rows that start anywhere), 17 through 4 (1024) and 19 through 8 (520).
RING = [(2500, 7168), (2501, 7167), (4001, 3373), (20_011, 1024), (22_003, 520)]


@pytest.mark.gpu
@pytest.mark.parametrize("gate", ["none", "channel", "token", "element"])
@pytest.mark.parametrize("T,M", RING)
def test_many_rows_parts(T, M, gate):
    for post, pre in ((True, True), (True, False), (False, True), (False, False)):
        _run(T, M, gate=gate, post=post, pre=pre, rs=-0.5, off=1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("x", list(DT))
@pytest.mark.parametrize("y", [None, *DT])
@pytest.mark.parametrize("T,M", [(2501, 7168), (4001, 3373)])
def test_many_rows_types(T, M, x, y):
    for w, n in (("fp16", "bf16"), ("bf16", "fp32"), ("fp32", "fp16")):
        _run(T, M, x=x, y=y, w=w, n=n, gate="token" if y else "none", post=y is not None, rs=0.7)


@pytest.mark.gpu
@pytest.mark.parametrize("pad,at", [(64, 16), (17, 3)])     # aligned rows, rows that start anywhere
@pytest.mark.parametrize("T,M", [(11, 200), (900, 72), (2500, 7168), (4001, 3376), (20_011, 1024)])
def test_in_place_leaves_what_lies_beside(T, M, pad, at):
    """x' in place in the columns of a wider buffer, n into the columns of another: what lies
    beside them, and the other inputs, stay as they were."""
    g = torch.Generator(device=DEV).manual_seed(T + M + pad)
    big = torch.randn((T, M + pad), generator=g, device=DEV).to(torch.bfloat16)
    ybig = torch.randn((T, M + pad), generator=g, device=DEV).to(torch.float16)
    X, Y = big[:, at:at + M], ybig[:, at:at + M]
    G = torch.randn((T, M), generator=g, device=DEV).to(torch.bfloat16)
    out = torch.full((T, M + pad), 7.0, device=DEV, dtype=torch.float32)
    xr, dx, nr, dn = ref.block_norm(X, Y, G, 0.9, None, None, True, True, 1e-6, 0.0)
    before, ybefore = big.clone(), ybig.clone()
    xo, no = norm.block_norm(X, Y, gate=G, residual_scale=0.9, x_out=X, n_out=out[:, at:at + M])
    assert xo.data_ptr() == X.data_ptr() and no.data_ptr() == out[:, at:].data_ptr()
    ref.check_rounded(X, xr, dx)
    ref.check_rounded(no, nr, dn)
    for a, b in ((big, before), (out, torch.full_like(out, 7.0))):
        assert torch.equal(a[:, :at], b[:, :at]) and torch.equal(a[:, at + M:], b[:, at + M:])
    assert torch.equal(ybig, ybefore)


@pytest.mark.gpu
def test_error_word():
    """A wait that gave up (none can be made to here: the word is set by hand) is reported once."""
    X = torch.randn((2500, 1024), device=DEV)
    norm.block_norm(X)
    norm.check()
    word = norm.error_word()
    assert word.shape == (1,) and word.dtype == torch.int32 and word.device == X.device
    word.fill_(1)
    with pytest.raises(RuntimeError, match=r"wisp engine error \[7\].*waiting"):
        norm.check(X.device)
    assert word.item() == 0
    norm.check(0)
