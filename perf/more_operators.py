"""The 8-bit block-scaled expert operators and the routing with a bias for balance, as
measured work.

Three operators of one MoE layer: ``rows`` (rows to e4m3 codes with one scale per 128
values, and back to values), ``product`` (8-bit rows by the 8-bit matrices of the experts
they go to, one scale per 128 x 128 block, with SwiGLU for gate and up) and ``route``
(scores from logits, a bias that chooses and does not weigh, groups, top-k, weights).
"""
import math
import random

import torch

own = False

DEV = "cuda"
BLOCK = 128
TOP = 448.0            # the largest e4m3 value
DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


# --------------------------------------------------------------------------
# Cases
# --------------------------------------------------------------------------
def listed():
    return [
        # One decoded token on its way into the experts: latency.
        dict(name="rows_token", op="rows", dtype="bf16", tokens=1, rows=1, gather=False, cols=7168,
             pow2=False),
        # A prefill of 4096 tokens, each gathered once for every expert it goes to.
        dict(name="rows_prefill", op="rows", dtype="bf16", tokens=4096, rows=32768, gather=True,
             cols=7168, pow2=False),
        # A ragged batch whose row length ends inside a block, scales that are powers of two.
        dict(name="rows_ragged", op="rows", dtype="fp16", tokens=331, rows=997, gather=True,
             cols=2064, pow2=True),
        # One token through one always-on projection: latency, few output tiles.
        dict(name="product_token", op="product", swiglu=False, out="fp32", k=7168, n=2048,
             entries=1, shared=False, tokens=1, top_k=1, skew=0.0, plan=1),
        # Decode of 40 tokens over 64 experts and a shared one: a few rows each.
        dict(name="gate_up_decode", op="product", swiglu=True, out="bf16", k=7168, n=2048,
             entries=64, shared=True, tokens=40, top_k=8, skew=0.0, plan=2),
        # Prefill of 4096 tokens over 256 unevenly loaded experts and a shared one.
        dict(name="gate_up_prefill", op="product", swiglu=True, out="bf16", k=7168, n=2048,
             entries=256, shared=True, tokens=4096, top_k=8, skew=1.0, plan=3),
        # The same layer's way back, at full precision for the weighted sum.
        dict(name="down_prefill", op="product", swiglu=False, out="fp32", k=2048, n=7168,
             entries=256, shared=True, tokens=4096, top_k=8, skew=1.0, plan=3),
        # A dense projection over a large batch: bound by the tensor cores.
        dict(name="product_dense", op="product", swiglu=False, out="bf16", k=7168, n=8192,
             entries=1, shared=False, tokens=8192, top_k=1, skew=0.0, plan=5),
        # Odd sizes, experts that no token goes to, k and n that end inside a block.
        dict(name="product_ragged", op="product", swiglu=True, out="fp16", k=2064, n=1000,
             entries=11, shared=False, tokens=333, top_k=2, skew=3.0, plan=4),
        # The routing of one decoded token: latency.
        dict(name="route_token", op="route", scoring="sigmoid", dtype="fp32", tokens=1,
             experts=256, top_k=8, groups=8, kept=4, group_top=2, bias=True, renorm=True,
             scaling=2.5),
        # The routing of a prefill.
        dict(name="route_prefill", op="route", scoring="sigmoid", dtype="fp32", tokens=4096,
             experts=256, top_k=8, groups=8, kept=4, group_top=2, bias=True, renorm=True,
             scaling=2.5),
        # A ragged batch over an odd number of experts, 16-bit logits with many ties.
        dict(name="route_ragged", op="route", scoring="softmax", dtype="bf16", tokens=3331,
             experts=77, top_k=6, groups=7, kept=3, group_top=1, bias=False, renorm=False,
             scaling=1.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rows", "product", "product", "route"])
    if op == "rows":
        tokens, gather = _log(rng, 1, 4096), rng.random() < 0.5
        return dict(op=op, dtype=rng.choice(["bf16", "fp16", "fp32"]), tokens=tokens,
                    rows=_log(rng, 1, 8 * tokens) if gather else tokens, gather=gather,
                    cols=16 * _log(rng, 4, 7168 // 16), pow2=rng.random() < 0.5)
    if op == "product":
        entries = _log(rng, 1, 64)
        return dict(op=op, swiglu=rng.random() < 0.5, out=rng.choice(["bf16", "fp16", "fp32"]),
                    k=16 * _log(rng, 8, 7168 // 16), n=_log(rng, 64, 4096), entries=entries,
                    shared=rng.random() < 0.5, tokens=_log(rng, 1, 4096),
                    top_k=rng.randint(1, min(8, entries)), skew=rng.choice([0.0, 1.0, 2.0]),
                    plan=rng.randrange(1 << 30))
    groups = rng.choice([1, 1, 2, 4, 7, 8])
    per = _log(rng, 2, 384 // groups)
    kept = rng.randint(1, groups)
    return dict(op=op, scoring=rng.choice(["softmax", "sigmoid"]),
                dtype=rng.choice(["fp32", "bf16", "fp16"]), tokens=_log(rng, 1, 4096),
                experts=groups * per, top_k=rng.randint(1, min(16, kept * per)), groups=groups,
                kept=kept, group_top=rng.choice([1, 2]), bias=rng.random() < 0.6,
                renorm=rng.random() < 0.6, scaling=rng.choice([1.0, 2.5]))


def _counts(case):
    """Rows of each entry: every token's draws over the experts, then the shared one's."""
    rng = random.Random(case["plan"])
    w = [math.exp(rng.gauss(0.0, case["skew"])) for _ in range(case["entries"])]
    n = [0] * case["entries"]
    for e in rng.choices(range(case["entries"]), w, k=case["tokens"] * case["top_k"]):
        n[e] += 1
    return n + ([case["tokens"]] if case["shared"] else [])


def _blocks(n):
    return (n + BLOCK - 1) // BLOCK


# --------------------------------------------------------------------------
# Inputs
# --------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _activations(g, shape, dtype):
    """Normal values; a few channels run far larger than the rest, as activations do."""
    x = torch.randn(shape, generator=g, device=DEV)
    hot = torch.rand((shape[1],), generator=g, device=DEV) < 0.01
    return (x * torch.where(hot, 20.0, 1.0)).to(dtype)


def _weights(g, entries, n, k):
    """e4m3 codes and block scales of `entries` matrices: normal values whose largest in a
    block is near the largest code."""
    codes = torch.empty((entries, n, k), dtype=torch.float8_e4m3fn, device=DEV)
    for e in range(entries):
        codes[e] = (torch.randn((n, k), generator=g, device=DEV) * 100.0).clamp_(-TOP, TOP)
    scales = torch.empty((entries, _blocks(n), _blocks(k)), device=DEV)
    return codes, scales.uniform_(1e-4, 4e-4, generator=g)


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    if op == "rows":
        s = dict(case=case, rows=None,
                 x=_activations(g, (case["tokens"], case["cols"]), DTYPE[case["dtype"]]))
        if case["gather"]:
            s["rows"] = torch.randint(0, case["tokens"], (case["rows"],), generator=g, device=DEV,
                                      dtype=torch.int32)
        return s
    if op == "product":
        counts = _counts(case)
        rows, mats = sum(counts), 2 if case["swiglu"] else 1
        w = [_weights(g, len(counts), case["n"], case["k"]) for _ in range(mats)]
        x = _activations(g, (case["tokens"], case["k"]), torch.bfloat16)
        c, b = _quantise(x, False)
        src = torch.randint(0, case["tokens"], (rows,), generator=g, device=DEV)
        # (e4m3 rows are indexed as bytes); scales stored block by block
        s = dict(case=case, counts=counts, w=w, scales=b[src].t().contiguous().t(),
                 codes=c.view(torch.uint8)[src].view(torch.float8_e4m3fn))
        if own:
            from wisp_b200 import fp8
            at, seg = 0, []
            for e, r in enumerate(counts):
                seg.append((e, at, r, 0))
                at += r
            s["segments"] = torch.tensor(seg, dtype=torch.int32, device=DEV)
            s["xq"] = fp8.Fp8Rows(s["codes"], s["scales"])
            s["weights"] = fp8.Fp8Weights(*w[0], up=w[1] if mats == 2 else None)
        return s
    logits = torch.randn((case["tokens"], case["experts"]), generator=g, device=DEV) * 1.7
    logits += torch.randn((case["experts"],), generator=g, device=DEV)
    s = dict(case=case, logits=logits.to(DTYPE[case["dtype"]]), bias=None)
    if case["bias"]:
        s["bias"] = torch.randn((case["experts"],), generator=g, device=DEV) * 0.1
    return s


# --------------------------------------------------------------------------
# The plain forms
# --------------------------------------------------------------------------
def _to_blocks(x):
    """[R, C] to [R, blocks, 128], the last block filled up with zeros."""
    pad = _blocks(x.shape[1]) * BLOCK - x.shape[1]
    return torch.nn.functional.pad(x, (0, pad)).reshape(x.shape[0], -1, BLOCK)


def _quantise(x, pow2):
    """e4m3 codes [R, C] and scales [R, blocks] of rows. Each value goes to the nearest e4m3
    value times its block's scale, ties to the even code; the decision is made in 64 bits (a
    value next to the border of two codes would fall on it in 32)."""
    R, C = x.shape
    b = _to_blocks(x.double())
    top = b.abs().amax(dim=2)
    if pow2:
        m, e = torch.frexp(top)            # top / 448 = m / 0.875 * 2^(e - 9)
        e = torch.where(m > 0.875, e - 8, e - 9).clamp(min=-126)
        scale = torch.where(top > 0, torch.ldexp(torch.ones_like(top), e), torch.zeros_like(top))
    else:
        scale = (top / TOP).float().double()
    q = b / torch.where(scale > 0, scale, torch.ones_like(scale))[..., None]
    q = torch.where((scale > 0)[..., None], q, torch.zeros_like(q))
    e = torch.frexp(q)[1].clamp(min=-5)    # steps of 2^(e - 4), of 2^-9 below 2^-6
    step = torch.ldexp(torch.ones_like(q), e - 4)
    q = (torch.round(q / step) * step).clamp(-TOP, TOP)
    return q.float().to(torch.float8_e4m3fn).reshape(R, -1)[:, :C].contiguous(), scale.float()


def _plain_rows(s):
    case = s["case"]
    c, b = _quantise(s["x"], case["pow2"])
    v = (c.float() * b.repeat_interleave(BLOCK, dim=1)[:, :case["cols"]]).to(s["x"].dtype)
    if s["rows"] is not None:
        v, b = v[s["rows"].long()], b[s["rows"].long()]
    return {"values": v, "scales": b}


def _plain_product(s):
    case = s["case"]
    n, k = case["n"], case["k"]
    out = torch.empty((s["codes"].shape[0], n), dtype=DTYPE[case["out"]], device=DEV)
    at = 0
    for e, r in enumerate(s["counts"]):
        if r == 0:
            continue
        x = s["codes"][at:at + r].float()
        x *= s["scales"][at:at + r].repeat_interleave(BLOCK, dim=1)[:, :k]
        y = []
        for codes, scales in s["w"]:
            w = codes[e].float()
            w *= scales[e].repeat_interleave(BLOCK, dim=1)[:, :k].repeat_interleave(BLOCK, dim=0)[:n]
            y.append(x @ w.t())
        if case["swiglu"]:
            y[0] = y[0] / (1.0 + torch.exp(-y[0])) * y[1]
        out[at:at + r] = y[0].to(out.dtype)
        at += r
    return out


def _plain_route(s):
    """Scores and choice in 64 bits: two experts whose choices lie next to each other would
    change places in 32."""
    case = s["case"]
    l = s["logits"].double()
    if case["scoring"] == "softmax":
        e = torch.exp(l - l.amax(dim=1, keepdim=True))
        score = e / e.sum(dim=1, keepdim=True)
    else:
        score = 1.0 / (1.0 + torch.exp(-l))
    choice = score if s["bias"] is None else score + s["bias"].double()
    G = case["groups"]
    if case["kept"] < G:
        per = choice.reshape(choice.shape[0], G, -1)
        top = per.sort(dim=2, descending=True)[0][:, :, :case["group_top"]].sum(dim=2)
        order = top.sort(dim=1, descending=True, stable=True)[1][:, :case["kept"]]
        keep = torch.zeros_like(top, dtype=torch.bool).scatter(1, order, True)
        choice = torch.where(keep[:, :, None], per, torch.full_like(per, -math.inf))
        choice = choice.reshape(l.shape)
    idx = choice.sort(dim=1, descending=True, stable=True)[1][:, :case["top_k"]]
    w = score.gather(1, idx)
    if case["renorm"]:
        w = w / w.sum(dim=1, keepdim=True)
    return {"idx": idx.int(), "weights": (w * case["scaling"]).float()}


# --------------------------------------------------------------------------
# One pass
# --------------------------------------------------------------------------
def run(s):
    case = s["case"]
    op = case["op"]
    if not own:
        return {"rows": _plain_rows, "product": _plain_product, "route": _plain_route}[op](s)
    if op == "rows":
        from wisp_b200 import fp8
        q = fp8.quantize(s["x"], rows=s["rows"], pow2=case["pow2"])
        return {"values": fp8.dequantize(q, s["x"].dtype), "scales": q.scales}
    if op == "product":
        from wisp_b200 import fp8
        return fp8.product(s["xq"], s["weights"], s["segments"], dtype=DTYPE[case["out"]])
    from wisp_b200 import abi, routing
    idx, w = routing.select_experts(
        s["logits"], case["top_k"], bias=s["bias"],
        scoring=abi.WISP_ROUTE_SOFTMAX if case["scoring"] == "softmax" else abi.WISP_ROUTE_SIGMOID,
        n_groups=case["groups"], topk_groups=case["kept"], group_top=case["group_top"],
        renormalize=case["renorm"], scaling=case["scaling"])
    return {"idx": idx, "weights": w}


def work(case):
    op = case["op"]
    if op == "rows":
        # the rows read once, their values and scales written once (rounding and scaling: about
        # 4 a value)
        n = case["rows"] * case["cols"]
        size = SIZE[case["dtype"]]
        read = min(case["tokens"], case["rows"]) * case["cols"] * size + \
            (4 * case["rows"] if case["gather"] else 0)
        return {"bytes": read + n * size + 4 * case["rows"] * _blocks(case["cols"]), "flops": 4 * n}
    if op == "product":
        counts = _counts(case)
        rows, mats = sum(counts), 2 if case["swiglu"] else 1
        n, k = case["n"], case["k"]
        used = sum(1 for r in counts if r)
        return {"bytes": used * mats * (n * k + 4 * _blocks(n) * _blocks(k)) +
                rows * (k + 4 * _blocks(k)) + rows * n * SIZE[case["out"]],
                "flops": 2 * rows * k * n * mats}
    # every logit read once; its score and its place among the others: about 8 a logit
    T, E = case["tokens"], case["experts"]
    return {"bytes": T * E * SIZE[case["dtype"]] + (4 * E if case["bias"] else 0) +
            8 * T * case["top_k"], "flops": 8 * T * E}


# --------------------------------------------------------------------------
# From the definitions, in 64 bits
# --------------------------------------------------------------------------
def _decode64(codes):
    """e4m3 bytes to values by their bit fields: sign, 4 exponent bits, 3 mantissa bits."""
    u = codes.view(torch.uint8).int()
    e, m = (u // 8) % 16, (u % 8).double()
    v = torch.where(e == 0, m / 512.0, torch.ldexp(1.0 + m / 8.0, e - 7))
    return torch.where(u >= 128, -v, v)


def _spread(scales, n, dim):
    return torch.repeat_interleave(scales.double(), BLOCK, dim=dim).narrow(dim, 0, n)


def _exact_rows(x, pow2):
    """Values and scales of quantised rows: the nearest of all 127 magnitudes, found among the
    borders between neighbours."""
    R, C = x.shape
    grid = _decode64(torch.arange(127, dtype=torch.uint8, device=x.device))
    pad = torch.zeros((R, _blocks(C) * BLOCK - C), dtype=torch.float64, device=x.device)
    b = torch.cat((x.double(), pad), dim=1).view(R, -1, BLOCK)
    t = b.abs().max(dim=2)[0] / TOP
    if pow2:
        # the logarithm is a guess that the comparisons put right
        p = torch.ceil(torch.log2(torch.clamp(t, min=2.0 ** -140))).int()
        low, at, high = (torch.ldexp(torch.ones_like(t), p + i) for i in (-1, 0, 1))
        scale = torch.where(low >= t, low, torch.where(at >= t, at, high))
        scale = torch.where(t > 0, scale.clamp(min=2.0 ** -126), torch.zeros_like(t))
    else:
        scale = t.to(torch.float32).double()
    q = torch.where(scale[..., None] > 0, b.abs() / scale[..., None], torch.zeros_like(b))
    mid = (grid[1:] + grid[:-1]) / 2
    at = torch.searchsorted(mid, q.contiguous())           # borders below q
    on = mid[at.clamp(max=125)] == q                       # on a border: to the even code
    at = torch.where(on & (at % 2 == 1) & (at < 126), at + 1, at)
    v = torch.sign(b) * grid[at] * scale[..., None]
    return v.view(R, -1)[:, :C], scale


def _exact_route(s):
    case = s["case"]
    l = s["logits"].double()
    T, E = l.shape
    score = torch.softmax(l, 1) if case["scoring"] == "softmax" else torch.sigmoid(l)
    left = score.clone() if s["bias"] is None else score + s["bias"].double()[None]
    G, per = case["groups"], E // case["groups"]
    columns = torch.arange(E, device=l.device)
    if case["kept"] < G:
        best = left.view(T, G, per).topk(min(case["group_top"], per), dim=2)[0].sum(2)
        rank = ((best[:, None, :] > best[:, :, None]) |
                ((best[:, None, :] == best[:, :, None]) &
                 (torch.arange(G, device=l.device)[None, None, :] <
                  torch.arange(G, device=l.device)[None, :, None]))).sum(2)
        left[rank.repeat_interleave(per, dim=1) >= case["kept"]] = -math.inf
    picks = []
    for _ in range(case["top_k"]):
        top = left.max(dim=1, keepdim=True)[0]
        i = torch.where(left == top, columns, E).min(dim=1)[0]
        picks.append(i)
        left[torch.arange(T, device=l.device), i] = -math.inf
    idx = torch.stack(picks, 1)
    w = torch.gather(score, 1, idx)
    if case["renorm"]:
        w = w / w.sum(1, True)
    return {"idx": idx.to(torch.int32), "weights": w * case["scaling"]}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rows":
        v, b = _exact_rows(s["x"], case["pow2"])
        if s["rows"] is not None:
            v, b = v.index_select(0, s["rows"].long()), b.index_select(0, s["rows"].long())
        return {"values": v, "scales": b}
    if case["op"] == "product":
        parts, at, n, k = [], 0, case["n"], case["k"]
        for e, r in enumerate(s["counts"]):
            x = _decode64(s["codes"][at:at + r]) * _spread(s["scales"][at:at + r], k, 1)
            y = [x.matmul((_decode64(c[e]) * _spread(_spread(b[e], n, 0), k, 1)).T)
                 for c, b in s["w"]]
            parts.append(y[0] * torch.sigmoid(y[0]) * y[1] if len(y) == 2 else y[0])
            at += r
        return torch.cat(parts)
    return _exact_route(s)
