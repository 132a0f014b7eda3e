"""The 4-bit block-scaled formats and the block norms in 64 bits, for the tests.

Everything here follows the formats' definitions on CPU or GPU tensors of
float64 and shares no code with the library.
"""
from __future__ import annotations

import torch

from wisp_b200 import abi

MX, NV = abi.WISP_FP4_MX, abi.WISP_FP4_NV
BLOCK = {MX: 32, NV: 16}
GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def exp2i(e: torch.Tensor) -> torch.Tensor:
    """2^e in 64 bits for whole e (torch.pow(2, e) is a last bit off for some e on the GPU)."""
    return torch.ldexp(torch.ones_like(e, dtype=torch.float64), e.to(torch.int32))


def scale_values(sb: torch.Tensor, fmt: int) -> torch.Tensor:
    u = sb.to(torch.int64)
    if fmt == MX:
        v = exp2i(u - 127)
        return torch.where(u == 255, torch.full_like(v, float("nan")), v)
    e, m = u // 8, (u % 8).double()
    v = torch.where(e == 0, m / 512.0, (1 + m / 8.0) * exp2i(e - 7))
    return torch.where(u == 0x7F, torch.full_like(v, float("nan")), v)


def values(codes: torch.Tensor, sb: torch.Tensor, fmt: int, ts=None) -> torch.Tensor:
    """float64 values of packed codes [..., K/2]."""
    c = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2).to(torch.int64)
    v = GRID.to(codes.device)[c & 7]
    v = torch.where(c >= 8, -v, v) * scale_values(sb, fmt).repeat_interleave(BLOCK[fmt], dim=-1)
    return v if ts is None else v * ts.double()


def quantize(x: torch.Tensor, fmt: int, ts=None):
    """(packed codes, scale bytes) of rows x by exhaustive search over the code values: the
    nearest, the even code of two equally near ones."""
    b = x.double().reshape(x.shape[0], -1, BLOCK[fmt])
    top = b.abs().amax(-1)
    finite = torch.isfinite(b).all(-1)
    if fmt == MX:
        t = torch.where(finite & (top > 0), top, torch.ones_like(top))
        e = torch.frexp(t)[1].double() - 1 - 2
        sb = torch.where(top > 0, (e + 127).clamp(0, 254), torch.zeros_like(e)).to(torch.int64)
        scale = exp2i(sb - 127)
        sb = torch.where(finite, sb, torch.full_like(sb, 255))
    else:
        g = float(ts)
        good = finite & (0 < g < float("inf"))
        t = torch.where(good, top / (6.0 * g) if g else top, torch.zeros_like(top))
        tab = scale_values(torch.arange(0x7F, device=x.device), NV)
        i = torch.searchsorted(tab, t.clamp(max=448.0)).clamp(1, 0x7E)
        lo, hi = tab[i - 1], tab[i]
        dn, up = t.clamp(max=448.0) - lo, hi - t.clamp(max=448.0)
        sb = torch.where((up < dn) | ((up == dn) & (i % 2 == 0)), i, i - 1)
        scale = tab[sb] * g
        sb = torch.where(good, sb, torch.full_like(sb, 0x7F))
        finite = good
    s = scale[..., None]
    a = torch.where(finite[..., None], b.abs(), torch.zeros_like(b))
    # |x| against the midpoints of neighbouring codes times the scale (exact in 64 bits)
    grid = GRID.to(x.device)
    c = torch.zeros_like(a, dtype=torch.int64)
    for j in range(7):
        mid = (grid[j] + grid[j + 1]) / 2 * s
        c += ((a > mid) | ((a == mid) & (j % 2 == 1))).to(torch.int64)
    c = torch.where(s > 0, c, torch.zeros_like(c))
    sign = torch.signbit(b) & finite[..., None]
    c = (c + 8 * sign.to(torch.int64)).reshape(x.shape)
    return (c[:, 0::2] | c[:, 1::2] << 4).to(torch.uint8), sb.to(torch.uint8)


def half_step(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def check_product(out, q, mats, counts_segs, k):
    """Rows of `out` against the products in 64 bits. mats: [(codes, scales, ts)] (one, or gate
    and up); counts_segs: (expert, row0, rows). The bound, per value: the products of 4-bit
    values are exact in fp32, so only sums round, at most k of them, each by 2^-23 of the sum of
    the terms' magnitudes (2^-24 when rounding to nearest, twice that where the adder
    truncates), and scaling and the rounding to the output type come once more."""
    x = values(q.codes, q.scales, q.fmt, q.tensor_scale)
    worst = 0.0
    for e, r0, r in counts_segs:
        if r == 0:
            continue
        y, d = [], []
        for codes, scales, ts in mats:
            w = values(codes[e], scales[e], q.fmt, None if ts is None else ts[e])
            y.append(x[r0:r0 + r] @ w.T)
            d.append((k + 4) * 2.0 ** -23 * (x[r0:r0 + r].abs() @ w.abs().T))
        if len(mats) == 2:
            s = torch.sigmoid(y[0])
            ref = y[0] * s * y[1]
            # |silu'| <= 1.1; expf, the sum, the quotient and two products: 8 roundings
            tol = 1.1 * d[0] * (y[1].abs() + d[1]) + (y[0] * s).abs() * d[1] + \
                8 * 2.0 ** -23 * ref.abs()
        else:
            ref, tol = y[0], d[0]
        tol = tol * 1.001 + half_step(out.dtype) * (ref.abs() + tol)
        # half a subnormal step of the output type
        tol = tol + torch.finfo(out.dtype).smallest_normal * torch.finfo(out.dtype).eps
        err = (out[r0:r0 + r].double() - ref).abs()
        assert torch.isfinite(out[r0:r0 + r]).all()
        worst = max(worst, (err / tol).max().item())
    assert worst <= 1.0, f"error {worst:.3g} times the bound"


def block_norm(x, y, gate, rs, post_w, pre_w, post, pre, eps, off):
    """(x', n) in 64 bits and a bound on each in fp32 arithmetic before the last rounding."""
    c = 80 * 2.0 ** -24
    # a row's sum of squares: at most 32 terms in a thread and 10 levels of a tree, each
    # rounding 2^-24 of it; the root halves that; division, root, reciprocal, weights and gate
    # come to under 12 more. 80 covers twice their sum.
    x = x.double()
    dx = torch.zeros_like(x)
    if y is not None:
        p = y.double()
        if post:
            p = p / torch.sqrt(p.square().mean(1, keepdim=True) + eps)
            if post_w is not None:
                p = p * (off + post_w.double())
        if gate is not None:
            p = p * gate.double()
        dx = c * (p.abs() + (rs * x).abs())
        x = rs * x + p
    n = dn = None
    if pre:
        r = 1 / torch.sqrt(x.square().mean(1, keepdim=True) + eps)
        w = torch.ones_like(x) if pre_w is None else (off + pre_w.double()).expand_as(x)
        n = x * r * w
        shift = torch.sqrt(dx.square().mean(1, keepdim=True)) * r
        dn = c * n.abs() + dx * r * w.abs() + shift * n.abs()
    return x, dx, n, dn


def check_rounded(out, ref, tol):
    f = torch.finfo(out.dtype)
    bound = tol + f.eps / 2 * (ref.abs() + tol) + f.smallest_normal * f.eps
    worst = ((out.double() - ref).abs() / bound).max().item()
    assert worst <= 1.0, f"error {worst:.3g} times the bound"
