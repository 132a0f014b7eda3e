"""The 8-bit block-scaled format and the routing with a balance bias in 64 bits, for the tests.

Everything here follows the definitions on CPU or GPU tensors of float64 and shares no code
with the library.
"""
from __future__ import annotations

import torch

B = 128


def decode(codes: torch.Tensor) -> torch.Tensor:
    """float64 values of e4m3 codes."""
    u = codes.view(torch.uint8).to(torch.int32)
    e, m = (u >> 3) & 15, (u & 7).double()
    v = torch.where(e == 0, m / 512.0, torch.ldexp(1 + m / 8.0, e - 7))
    v = torch.where((u & 127) == 127, torch.full_like(v, float("nan")), v)
    return torch.where(u >= 128, -v, v)


def grid(device) -> torch.Tensor:
    """The 127 magnitudes, by code."""
    return decode(torch.arange(127, dtype=torch.uint8, device=device))


def blocks(n: int) -> int:
    return -(-n // B)


def spread(scales: torch.Tensor, n: int, dim: int) -> torch.Tensor:
    return scales.double().repeat_interleave(B, dim=dim).narrow(dim, 0, n)


def row_values(codes, scales) -> torch.Tensor:
    return decode(codes) * spread(scales, codes.shape[1], 1)


def weight_values(codes, scales) -> torch.Tensor:
    """[n, k] values of one matrix."""
    return decode(codes) * spread(spread(scales, codes.shape[0], 0), codes.shape[1], 1)


def scale_of(top: torch.Tensor, pow2: bool) -> torch.Tensor:
    """float64 scales of blocks of the given (finite) largest magnitudes: fp32(top / 448), or the
    least power of two that is not below it, at least 2^-126."""
    if not pow2:
        return (top / 448.0).float().double()
    t = top.clamp(min=2.0 ** -126)
    e = torch.frexp(t)[1] - 12          # 2^e is below any top / 448
    s = torch.ldexp(torch.ones_like(t), e)
    for _ in range(6):
        s = torch.where(448.0 * s < top, 2 * s, s)
    return torch.where(top > 0, s.clamp(min=2.0 ** -126), torch.zeros_like(s))


def codes_of(b: torch.Tensor, s: torch.Tensor, ok: torch.Tensor) -> torch.Tensor:
    """e4m3 codes (uint8) of values b [..., m] over scales s [...], by comparing magnitudes with
    the borders of neighbouring codes times the scale (exact in 64 bits: 5 and 24 bits)."""
    g = grid(b.device)
    mid = (g[1:] + g[:-1]) / 2
    a = torch.where(ok[..., None], b.abs(), torch.zeros_like(b))
    c = torch.zeros_like(a, dtype=torch.int32)
    for j in range(126):
        t = mid[j] * s[..., None]
        c += ((a > t) | ((a == t) & (j % 2 == 1))).int()
    c = torch.where(s[..., None] > 0, c, torch.zeros_like(c))
    neg = torch.signbit(b) & (c > 0)
    return (c + 128 * neg.int()).to(torch.uint8)


def quantize(x: torch.Tensor, pow2: bool = False):
    """(codes uint8 [R, C] with zeros unsigned, scales float64 [R, blocks]) of rows x."""
    R, C = x.shape
    pad = torch.zeros((R, blocks(C) * B - C), dtype=torch.float64, device=x.device)
    b = torch.cat([x.double(), pad], 1).view(R, -1, B)
    ok = torch.isfinite(b).all(-1)
    top = torch.where(ok, b.abs().amax(-1), torch.zeros_like(b[..., 0]))
    s = scale_of(top, pow2)
    c = codes_of(b, s, ok)
    s = torch.where(ok, s, torch.full_like(s, float("nan")))
    return c.view(R, -1)[:, :C], s


def unsigned_zeros(codes: torch.Tensor) -> torch.Tensor:
    u = codes.view(torch.uint8)
    return torch.where(u == 128, torch.zeros_like(u), u)


def half_step(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def check_product(out, codes, scales, mats, segs, k):
    """Rows of `out` against the products in 64 bits. mats: [(codes, scales)] (one, or gate and
    up); segs: (expert, row0, rows). The bound, per value: products of e4m3 values are exact in
    fp32 (8 significant bits), so of a block of 128 only sums round, at most 128 of them, each by
    2^-23 of the sum of the terms' magnitudes (2^-24 rounding to nearest, twice that where the
    adder truncates); the block's scaling rounds twice (weight scale; its sum with the row scale's
    product) and the blocks' sums once each, each by 2^-24 of what they hold: 128 + 2 + k / 128
    times 2^-23 in all covers that. The rounding to the output type comes once more."""
    x = row_values(codes, scales)
    worst = 0.0
    for e, r0, r in segs:
        if r == 0:
            continue
        y, d = [], []
        for c, s in mats:
            w = weight_values(c[e], s[e])
            y.append(x[r0:r0 + r] @ w.T)
            d.append((130 + blocks(k)) * 2.0 ** -23 * (x[r0:r0 + r].abs() @ w.abs().T))
        if len(mats) == 2:
            sg = torch.sigmoid(y[0])
            ref = y[0] * sg * y[1]
            # |silu'| <= 1.1; the exponential, its square, the sum, the quotient and three
            # products: 8 roundings. 16-bit outputs: the fast exponential's argument, |g| / 2 *
            # log2(e) rounded to fp32, twice over: |g| 2^-23, a factor 2 for the instruction
            tol = 1.1 * d[0] * (y[1].abs() + d[1]) + (y[0] * sg).abs() * d[1] + \
                8 * 2.0 ** -23 * ref.abs() + (y[0].abs() * 2.0 ** -22 * ref.abs()
                                              if out.dtype != torch.float32 else 0.0)
        else:
            ref, tol = y[0], d[0]
        tol = tol * 1.001 + half_step(out.dtype) * (ref.abs() + tol)
        # half a subnormal step of the output type
        tol = tol + torch.finfo(out.dtype).smallest_normal * torch.finfo(out.dtype).eps
        got = out[r0:r0 + r].double()
        assert torch.isfinite(got).all()
        worst = max(worst, ((got - ref).abs() / tol).max().item())
    assert worst <= 1.0, f"error {worst:.3g} times the bound"


def route(logits, top_k, bias=None, softmax=False, n_groups=1, topk_groups=1, group_top=2,
          renormalize=True, scaling=1.0):
    """(idx, weights float64) token by token, by the definition, on the CPU."""
    l = logits.double().cpu()
    T, E = l.shape
    per = E // n_groups
    idx = torch.full((T, top_k), -1, dtype=torch.int32)
    wt = torch.zeros((T, top_k), dtype=torch.float64)
    for t in range(T):
        if softmax:
            m = l[t].max()
            x = torch.exp(l[t] - m)
            score = x / x.sum()
        else:
            score = 1 / (1 + torch.exp(-l[t]))
        choice = score if bias is None else score + bias.double().cpu()
        can = [e for e in range(E) if choice[e] > -float("inf")]
        if topk_groups < n_groups:
            best = {}
            for g in range(n_groups):
                c = sorted((choice[e].item() for e in can if e // per == g), reverse=True)
                if c:
                    best[g] = sum(c[:group_top])
            kept = sorted(best, key=lambda g: (-best[g], g))[:topk_groups]
            can = [e for e in can if e // per in kept]
        picks = sorted(can, key=lambda e: (-choice[e].item(), e))[:top_k]
        w = torch.tensor([score[e].item() for e in picks], dtype=torch.float64)
        if renormalize and len(picks):
            w = w / w.sum() if w.sum() > 0 else torch.zeros_like(w)
        idx[t, :len(picks)] = torch.tensor(picks, dtype=torch.int32)
        wt[t, :len(picks)] = w * scaling
    return idx, wt
