"""The 4-bit block-scaled expert operators and the block norms, as measured work.

Three operators of one MoE block: ``quantise`` (rows to 4-bit codes with one
scale per block, and back to values), ``product`` (4-bit rows by the 4-bit
matrices of the experts they go to, with SwiGLU for gate and up) and ``norm``
(the norms after and before a block, its gate and its residual).
"""
import math
import random

import torch

own = False

DEV = "cuda"
BLOCK = {"mx": 32, "nv": 16}
DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# --------------------------------------------------------------------------
# Cases
# --------------------------------------------------------------------------
def listed():
    return [
        # One decoded token on its way into the experts: latency.
        dict(name="quantise_token", op="quantise", fmt="mx", dtype="bf16", tokens=1, rows=1,
             gather=False, cols=7168),
        # A prefill of 4096 tokens, each gathered once for every expert it goes to.
        dict(name="quantise_prefill_rows", op="quantise", fmt="nv", dtype="bf16", tokens=4096,
             rows=32768, gather=True, cols=7168),
        # One projection of an expert, quantised when a checkpoint is loaded.
        dict(name="quantise_weights", op="quantise", fmt="mx", dtype="fp32", tokens=14336,
             rows=14336, gather=False, cols=4096),
        # A ragged batch whose row length is no multiple of a wide load's span.
        dict(name="quantise_ragged", op="quantise", fmt="nv", dtype="fp16", tokens=331, rows=997,
             gather=True, cols=2064),
        # One token through one always-on projection: latency, few output tiles.
        dict(name="product_token", op="product", fmt="mx", swiglu=False, out="fp32", k=7168,
             n=2048, entries=1, shared=False, tokens=1, top_k=1, skew=0.0, plan=1),
        # Decode of 40 tokens over 64 experts and a shared one: a few rows each.
        dict(name="gate_up_decode", op="product", fmt="nv", swiglu=True, out="bf16", k=7168,
             n=2048, entries=64, shared=True, tokens=40, top_k=8, skew=0.0, plan=2),
        # Prefill of 4096 tokens over 256 unevenly loaded experts and a shared one.
        dict(name="gate_up_prefill", op="product", fmt="mx", swiglu=True, out="bf16", k=7168,
             n=2048, entries=256, shared=True, tokens=4096, top_k=8, skew=1.0, plan=3),
        # The same layer's way back, at full precision for the weighted sum.
        dict(name="down_prefill", op="product", fmt="nv", swiglu=False, out="fp32", k=2048,
             n=7168, entries=256, shared=True, tokens=4096, top_k=8, skew=1.0, plan=3),
        # Odd sizes, experts that no token goes to.
        dict(name="product_ragged", op="product", fmt="mx", swiglu=True, out="fp16", k=2080,
             n=1000, entries=11, shared=False, tokens=333, top_k=2, skew=3.0, plan=4),
        # Between two blocks of a decoded token.
        dict(name="norm_token", op="norm", tokens=1, hidden=7168, x="bf16", y="fp32", w="bf16",
             gate="channel", post=True, pre=True, n="bf16", scale=1.0),
        # Between two blocks of a prefill, the block's output in 32 bits.
        dict(name="norm_prefill", op="norm", tokens=4096, hidden=7168, x="bf16", y="fp32",
             w="bf16", gate="channel", post=True, pre=True, n="bf16", scale=1.0),
        # A ragged batch with a gate of its own for each token, odd row length.
        dict(name="norm_ragged", op="norm", tokens=333, hidden=2077, x="fp16", y="fp16", w="fp32",
             gate="token", post=True, pre=True, n="fp16", scale=0.5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantise", "product", "norm"])
    if op == "quantise":
        fmt = rng.choice(["mx", "nv"])
        tokens, gather = _log(rng, 1, 4096), rng.random() < 0.5
        return dict(op=op, fmt=fmt, dtype=rng.choice(["bf16", "fp16", "fp32"]), tokens=tokens,
                    rows=_log(rng, 1, 8 * tokens) if gather else tokens, gather=gather,
                    cols=BLOCK[fmt] * _log(rng, 2, 7168 // BLOCK[fmt]))
    if op == "product":
        entries = _log(rng, 1, 64)
        return dict(op=op, fmt=rng.choice(["mx", "nv"]), swiglu=rng.random() < 0.5,
                    out=rng.choice(["bf16", "fp16", "fp32"]), k=32 * _log(rng, 4, 7168 // 32),
                    n=_log(rng, 64, 4096), entries=entries, shared=rng.random() < 0.5,
                    tokens=_log(rng, 1, 4096), top_k=rng.randint(1, min(8, entries)),
                    skew=rng.choice([0.0, 1.0, 2.0]), plan=rng.randrange(1 << 30))
    return dict(op=op, tokens=_log(rng, 1, 4096), hidden=_log(rng, 64, 7168),
                x=rng.choice(["bf16", "fp16", "fp32"]), y=rng.choice(["bf16", "fp16", "fp32"]),
                w=rng.choice(["bf16", "fp32"]),
                gate=rng.choice(["none", "channel", "token", "element"]),
                post=rng.random() < 0.75, pre=rng.random() < 0.75,
                n=rng.choice(["bf16", "fp16", "fp32"]), scale=rng.choice([1.0, 0.5, 0.7071]))


def _counts(case):
    """Rows of each entry: every token's draws over the experts, then the shared one's."""
    rng = random.Random(case["plan"])
    w = [math.exp(rng.gauss(0.0, case["skew"])) for _ in range(case["entries"])]
    n = [0] * case["entries"]
    for e in rng.choices(range(case["entries"]), w, k=case["tokens"] * case["top_k"]):
        n[e] += 1
    return n + ([case["tokens"]] if case["shared"] else [])


# --------------------------------------------------------------------------
# Inputs
# --------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(g, shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def _pack(codes):
    return (codes[..., 0::2] | (codes[..., 1::2] << 4)).contiguous()


def _weights(g, fmt, entries, n, k):
    """Codes, scales and tensor scales of `entries` matrices whose values are spread as normal
    ones are after quantisation (drawn byte by byte from a table of such codes)."""
    a = torch.randn((4096, BLOCK[fmt]), generator=g, device=DEV)
    c, _ = _quantise(a, fmt, torch.full((1,), 3.0 / 2688, device=DEV) if fmt == "nv" else None)
    table = _pack(c).reshape(-1)
    codes = torch.empty((entries, n, k // 2), dtype=torch.uint8, device=DEV)
    for e in range(entries):
        codes[e] = table[torch.randint(0, table.numel(), (n, k // 2), generator=g, device=DEV)]
    lo, hi = (118, 122) if fmt == "mx" else (0x70, 0x7F)
    scales = torch.randint(lo, hi, (entries, n, k // BLOCK[fmt]), generator=g, device=DEV,
                           dtype=torch.uint8)
    ts = None
    if fmt == "nv":
        ts = torch.empty((entries,), device=DEV).uniform_(1e-5, 3e-5, generator=g)
    return codes, scales, ts


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    if op == "quantise":
        x = _randn(g, (case["tokens"], case["cols"]))
        # a few channels run far larger than the rest, as activations do
        x = (x * torch.where(torch.rand((case["cols"],), generator=g, device=DEV) < 0.01, 20.0, 1.0)
             ).to(DTYPE[case["dtype"]])
        s = dict(case=case, x=x, rows=None, ts=None)
        if case["gather"]:
            s["rows"] = torch.randint(0, case["tokens"], (case["rows"],), generator=g, device=DEV,
                                      dtype=torch.int32)
        if case["fmt"] == "nv":
            s["ts"] = (x.float().abs().max() / 2688.0).reshape(1)
        return s
    if op == "product":
        counts = _counts(case)
        rows, fmt = sum(counts), case["fmt"]
        mats = 2 if case["swiglu"] else 1
        w = [_weights(g, fmt, len(counts), case["n"], case["k"]) for _ in range(mats)]
        x = _randn(g, (case["tokens"], case["k"]), torch.bfloat16)
        ts = (x.float().abs().max() / 2688.0).reshape(1) if fmt == "nv" else None
        c, b = _quantise(x.float(), fmt, ts)
        c = _pack(c)
        src = torch.randint(0, case["tokens"], (rows,), generator=g, device=DEV)
        s = dict(case=case, counts=counts, w=w, codes=c[src], scales=b[src], ts=ts)
        if own:
            from wisp_b200 import abi, fp4
            f = abi.WISP_FP4_MX if fmt == "mx" else abi.WISP_FP4_NV
            at, seg = 0, []
            for e, r in enumerate(counts):
                seg.append((e, at, r, 0))
                at += r
            s["segments"] = torch.tensor(seg, dtype=torch.int32, device=DEV)
            s["xq"] = fp4.Fp4Rows(f, s["codes"], s["scales"], ts)
            s["weights"] = fp4.Fp4Weights(f, *w[0], up=w[1] if mats == 2 else None)
        return s
    T, M = case["tokens"], case["hidden"]
    s = dict(case=case, x=_randn(g, (T, M), DTYPE[case["x"]], 2.0), y=None, gate=None, post_w=None,
             pre_w=None)
    if case["post"] or case["gate"] != "none" or not case["pre"]:
        s["y"] = _randn(g, (T, M), DTYPE[case["y"]], 3.0)
        shape = {"none": None, "channel": (M,), "token": (T, 1), "element": (T, M)}[case["gate"]]
        if shape is not None:
            s["gate"] = torch.sigmoid(_randn(g, shape)).to(DTYPE[case["w"]])
    if case["post"]:
        s["post_w"] = (1.0 + _randn(g, (M,), scale=0.1)).to(DTYPE[case["w"]])
    if case["pre"]:
        s["pre_w"] = (1.0 + _randn(g, (M,), scale=0.1)).to(DTYPE[case["w"]])
    return s


# --------------------------------------------------------------------------
# The plain forms
# --------------------------------------------------------------------------
def _quantise(x, fmt, ts):
    """4-bit codes [R, C] and scale bytes [R, C / block] of float rows. Each value goes to the
    nearest of +-GRID times its block's scale, ties to the even code. The decision is made in
    64 bits: a value next to the border of two codes would fall on it in 32."""
    R, C = x.shape
    b = x.double().reshape(R, C // BLOCK[fmt], BLOCK[fmt])
    top = b.abs().amax(dim=2)
    if fmt == "mx":
        # 2^(floor(log2 max) - 2), the power of two that brings the largest into [4, 8)
        e = (torch.frexp(top)[1] - 3).clamp(-127, 127)
        e = torch.where(top > 0, e, torch.full_like(e, -127))
        scale = torch.ldexp(torch.ones_like(top), e)
        sb = (e + 127).to(torch.uint8)
    else:
        t = top / (6.0 * ts.double())
        e = (torch.frexp(t)[1] - 1).clamp(min=-6)
        step = torch.ldexp(torch.ones_like(t), e - 3)
        s = (torch.round(t / step) * step).clamp(max=448.0)
        sb = s.float().to(torch.float8_e4m3fn).view(torch.uint8)
        scale = s * ts.double()
    q = b.abs() / torch.where(scale > 0, scale, torch.ones_like(scale))[..., None]
    q = torch.where((scale > 0)[..., None], q, torch.zeros_like(q))
    c = (q > 0.25).to(torch.uint8)
    for border, up in ((0.75, 1), (1.25, 0), (1.75, 1), (2.5, 0), (3.5, 1), (5.0, 0)):
        c += (q >= border) if up else (q > border)
    c |= torch.signbit(b).to(torch.uint8) << 3
    return c.reshape(R, C), sb.reshape(R, -1)


def _scale_values(sb, fmt):
    """The values of scale bytes, in 32 bits (exact)."""
    if fmt == "mx":
        return torch.ldexp(torch.ones(sb.shape, device=DEV), sb.int() - 127)
    return sb.view(torch.float8_e4m3fn).float()


def _values(codes, sb, fmt):
    """The values of packed codes times their block scales, in 32 bits (exact products)."""
    grid = torch.tensor(GRID + tuple(-v for v in GRID), device=DEV)
    c = torch.stack((codes & 15, codes >> 4), dim=-1).reshape(codes.shape[0], -1)
    v = grid[c.int()].reshape(c.shape[0], -1, BLOCK[fmt]) * _scale_values(sb, fmt)[..., None]
    return v.reshape(c.shape)


def _plain_quantise(s):
    case = s["case"]
    c, sb = _quantise(s["x"], case["fmt"], s["ts"])
    v = _values(_pack(c), sb, case["fmt"])
    if s["ts"] is not None:
        v = v * s["ts"]
    v = v.to(DTYPE[case["dtype"]])
    return v if s["rows"] is None else v[s["rows"].long()]


def _plain_product(s):
    case, fmt = s["case"], s["case"]["fmt"]
    out = torch.empty((s["codes"].shape[0], case["n"]), dtype=DTYPE[case["out"]], device=DEV)
    at = 0
    for e, r in enumerate(s["counts"]):
        if r == 0:
            continue
        x = _values(s["codes"][at:at + r], s["scales"][at:at + r], fmt)
        y = []
        for codes, scales, ts in s["w"]:
            z = x @ _values(codes[e], scales[e], fmt).t()
            y.append(z if ts is None else z * (ts[e] * s["ts"]))
        if case["swiglu"]:
            y[0] = y[0] / (1.0 + torch.exp(-y[0])) * y[1]
        out[at:at + r] = y[0].to(out.dtype)
        at += r
    return out


def _plain_norm(s):
    case = s["case"]
    x = s["x"].float()
    if s["y"] is not None:
        p = s["y"].float()
        if case["post"]:
            p = p * torch.rsqrt((p * p).mean(dim=1, keepdim=True) + 1e-6) * s["post_w"].float()
        if s["gate"] is not None:
            p = p * s["gate"].float()
        x = case["scale"] * x + p
    out = {"x": x.to(s["x"].dtype)} if s["y"] is not None else {}
    if case["pre"]:
        n = x * torch.rsqrt((x * x).mean(dim=1, keepdim=True) + 1e-6) * s["pre_w"].float()
        out["n"] = n.to(DTYPE[case["n"]])
    return out


# --------------------------------------------------------------------------
# One pass
# --------------------------------------------------------------------------
def run(s):
    case = s["case"]
    op = case["op"]
    if not own:
        return {"quantise": _plain_quantise, "product": _plain_product, "norm": _plain_norm}[op](s)
    if op == "quantise":
        from wisp_b200 import abi, fp4
        f = abi.WISP_FP4_MX if case["fmt"] == "mx" else abi.WISP_FP4_NV
        return fp4.dequantize(fp4.quantize(s["x"], f, s["ts"], rows=s["rows"]), s["x"].dtype)
    if op == "product":
        from wisp_b200 import fp4
        return fp4.product(s["xq"], s["weights"], s["segments"], dtype=DTYPE[case["out"]])
    from wisp_b200 import norm
    x, n = norm.block_norm(s["x"], s["y"], gate=s["gate"], residual_scale=case["scale"],
                           post_weight=s["post_w"], pre_weight=s["pre_w"], post=case["post"],
                           pre=case["pre"], eps=1e-6, dtype=DTYPE[case["n"]])
    out = {"x": x} if s["y"] is not None else {}
    if case["pre"]:
        out["n"] = n
    return out


def work(case):
    op = case["op"]
    if op == "quantise":
        # the rows read once, their values written once (rounding and scaling: about 4 a value)
        n = case["rows"] * case["cols"]
        size = SIZE[case["dtype"]]
        read = min(case["tokens"], case["rows"]) * case["cols"] * size + \
            (4 * case["rows"] if case["gather"] else 0)
        return {"bytes": read + n * size, "flops": 4 * n}
    if op == "product":
        counts = _counts(case)
        rows, mats = sum(counts), 2 if case["swiglu"] else 1
        per = case["k"] // 2 + case["k"] // BLOCK[case["fmt"]]
        used = sum(1 for r in counts if r)
        return {"bytes": used * mats * case["n"] * per + rows * per +
                rows * case["n"] * SIZE[case["out"]],
                "flops": 2 * rows * case["k"] * case["n"] * mats}
    T, M = case["tokens"], case["hidden"]
    has_y = case["post"] or case["gate"] != "none" or not case["pre"]
    b = T * M * SIZE[case["x"]]
    flops = 0
    if has_y:
        b += T * M * (SIZE[case["y"]] + SIZE[case["x"]])
        b += {"none": 0, "channel": M, "token": T, "element": T * M}[case["gate"]] * SIZE[case["w"]]
        flops += 4 * T * M
    if case["post"]:
        b, flops = b + M * SIZE[case["w"]], flops + 4 * T * M
    if case["pre"]:
        b, flops = b + T * M * SIZE[case["n"]] + M * SIZE[case["w"]], flops + 4 * T * M
    return {"bytes": b, "flops": flops}


# --------------------------------------------------------------------------
# From the definitions, in 64 bits
# --------------------------------------------------------------------------
def _decode64(codes, sb, fmt):
    """Bytes to values by the formats' bit fields: code = sign, 2 exponent bits, 1 mantissa bit;
    scale = 8 exponent bits, or 4 exponent and 3 mantissa bits."""
    c = torch.empty((codes.shape[0], codes.shape[1] * 2), dtype=torch.int32, device=DEV)
    c[:, 0::2], c[:, 1::2] = codes.int() % 16, codes.int() // 16
    e, m = (c // 2) % 4, (c % 2).double()
    v = torch.where(e == 0, 0.5 * m, (1.0 + 0.5 * m) * torch.pow(2.0, (e - 1).double()))
    v = torch.where(c >= 8, -v, v)
    u = sb.int()
    if fmt == "mx":
        s = torch.pow(2.0, (u - 127).double())
    else:
        e, m = u // 8, (u % 8).double()
        s = torch.where(e == 0, m / 512.0, (1.0 + m / 8.0) * torch.pow(2.0, (e - 7).double()))
    return v * s.repeat_interleave(BLOCK[fmt], dim=1)


def _exact_rows(x, fmt, ts):
    """Values of quantised rows: rounding to an even multiple of the step of each binade."""
    b = x.double().reshape(x.shape[0], -1, BLOCK[fmt])
    top = b.abs().max(dim=2, keepdim=True)[0]
    if fmt == "mx":
        low = torch.full_like(top, 2.0 ** -126)
        k = torch.floor(torch.log2(torch.maximum(top, low)))
        k = torch.where(torch.pow(2.0, k) > top, k - 1, k)
        k = torch.where(torch.pow(2.0, k + 1) <= top, k + 1, k)
        scale = torch.pow(2.0, torch.clamp(k - 2, min=-127.0))
    else:
        t = top / (6.0 * ts.double())
        step = torch.full_like(t, 2.0 ** -9)
        for i in range(-5, 9):
            step = torch.where(t >= 2.0 ** i, torch.full_like(t, 2.0 ** (i - 3)), step)
        scale = torch.clamp(torch.round(t / step) * step, max=448.0) * ts.double()
    q = torch.where(scale > 0, b.abs() / scale, torch.zeros_like(b))
    step = torch.where(q < 2.0, 0.5, torch.where(q < 4.0, 1.0, 2.0)).double()
    return (torch.sign(b) * torch.clamp(torch.round(q / step) * step, max=6.0) * scale
            ).reshape(x.shape)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantise":
        v = _exact_rows(s["x"], case["fmt"], s["ts"])
        return v if s["rows"] is None else v.index_select(0, s["rows"].long())
    if case["op"] == "product":
        fmt, parts, at = case["fmt"], [], 0
        for e, r in enumerate(s["counts"]):
            x = _decode64(s["codes"][at:at + r], s["scales"][at:at + r], fmt)
            y = [x.matmul(_decode64(c[e], b[e], fmt).T) * (1.0 if t is None else
                                                           t[e].double() * s["ts"].double())
                 for c, b, t in s["w"]]
            parts.append(y[0] * torch.sigmoid(y[0]) * y[1] if len(y) == 2 else y[0])
            at += r
        return torch.cat(parts)
    x, out = s["x"].double(), {}
    if s["y"] is not None:
        p = s["y"].double()
        if case["post"]:
            p = s["post_w"].double() * p / torch.sqrt(p.square().sum(1, True) / p.shape[1] + 1e-6)
        if s["gate"] is not None:
            p = s["gate"].double() * p
        x = out["x"] = p + x * case["scale"]
    if case["pre"]:
        out["n"] = s["pre_w"].double() * x / torch.sqrt(x.square().sum(1, True) / x.shape[1] + 1e-6)
    return out
