"""Routing from logits with a balance bias, against the definition in 64 bits; refusals on the
CPU."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

import fp8_ref as ref
from wisp_b200 import abi, routing

P = 1 << 20   # a non-null aligned stand-in pointer; never dereferenced here
DEV = "cuda"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("kw,match", [
    (dict(scoring=2), "scoring"), (dict(n_groups=0), "n_groups"), (dict(n_groups=33), "n_groups"),
    (dict(n_groups=3), "n_groups"), (dict(topk_groups=0), "topk_groups"),
    (dict(topk_groups=5), "topk_groups"), (dict(group_top=0), "group_top"),
    (dict(group_top=3), "group_top"), (dict(top_k=0), "top_k"), (dict(top_k=33), "top_k"),
    (dict(top_k=17), "top_k"), (dict(dt=3), "logits_type"), (dict(ld=31), "ld"),
    (dict(tokens=-1), "tokens"), (dict(experts=1028, ld=2000), "n_experts"), (dict(experts=0), "n_experts"),
    (dict(logits=None), "null"), (dict(idx=None), "null"), (dict(w=None), "null"),
    (dict(logits=P + 2, dt=0), "aligned"), (dict(bias=P + 2), "aligned"),
    (dict(tokens=0x7FFFFF01), "2\\^31"),
])
def test_select_refuses(kw, match):
    a = dict(scoring=0, n_groups=4, topk_groups=2, group_top=2, logits=P, dt=1, ld=32, tokens=5,
             experts=32, top_k=4, bias=None, idx=P, w=P)
    a.update(kw)
    r = abi.WispRouting(a["scoring"], a["n_groups"], a["topk_groups"], a["group_top"], 1, 1.0)
    with pytest.raises(RuntimeError, match=r"wisp engine error \[4\].*" + match):
        abi.call("wisp_b200_select_experts", C.byref(r), a["logits"], a["dt"], a["ld"], a["tokens"],
                 a["experts"], a["top_k"], a["bias"], a["idx"], a["w"], None)


def test_select_without_a_routing_or_tokens():
    with pytest.raises(RuntimeError, match=r"wisp engine error \[4\].*null routing"):
        abi.call("wisp_b200_select_experts", None, P, 0, 32, 5, 32, 4, None, P, P, None)
    r = routing.policy()
    abi.call("wisp_b200_select_experts", C.byref(r), None, 0, 32, 0, 32, 4, None, None, None, None)


def test_policy_refuses_what_would_be_cut_off():
    for kw in (dict(n_groups=2 ** 32 + 1), dict(topk_groups=-1), dict(scoring=2 ** 32),
               dict(group_top=2 ** 33 + 2)):
        with pytest.raises(RuntimeError, match=r"wisp engine error \[4\]"):
            routing.policy(**kw)


def test_python_refusals():
    x = torch.zeros(2, 16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        routing.select_experts(x, 2)
    big = torch.empty((2 ** 32 + 1, 16), device="meta")
    for bad in (lambda: routing.select_experts(x.t(), 2), lambda: routing.select_experts(x[0], 2),
                lambda: routing.select_experts(x.long(), 2),
                lambda: routing.select_experts(x, 2, bias=torch.zeros(15)),
                lambda: routing.select_experts(x, 2, bias=torch.zeros(16).double()),
                lambda: routing.select_experts(x.clone().requires_grad_(), 2),
                lambda: routing.select_experts(x, 2, bias=torch.zeros(16, requires_grad=True)),
                lambda: routing.select_experts(big, 2)):
        with pytest.raises(RuntimeError, match=r"wisp engine error \[4\]"):
            bad()


def _check(logits, k, scoring, bias=None, **kw):
    softmax = scoring == abi.WISP_ROUTE_SOFTMAX
    idx, w = routing.select_experts(logits, k, bias=bias, scoring=scoring, **kw)
    want, ww = ref.route(logits, k, bias, softmax, **kw)
    assert torch.equal(idx.cpu(), want)
    # one rounding to fp32; the 64-bit steps before it round at 2^-50 or below
    d = (w.double().cpu() - ww).abs()
    assert (d <= 2.0 ** -24 * (1 + 2.0 ** -20) * ww.abs() + 2.0 ** -149).all()
    return idx, w


SCORING = pytest.mark.parametrize("scoring", [0, 1], ids=["softmax", "sigmoid"])


@pytest.mark.gpu
@SCORING
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("tokens,experts,k,groups,kept,top", [
    (1, 1, 1, 1, 1, 1), (1, 256, 8, 8, 4, 2), (5, 32, 32, 1, 1, 2), (7, 33, 4, 3, 2, 2),
    (130, 77, 6, 7, 3, 1), (3, 64, 1, 32, 1, 2), (9, 96, 12, 32, 31, 1), (4, 1024, 32, 4, 3, 2),
    (2, 500, 9, 5, 5, 2), (66, 160, 6, 8, 3, 1), (4, 8, 2, 1, 1, 2), (3, 31, 31, 31, 31, 2),
])
def test_select(scoring, dtype, tokens, experts, k, groups, kept, top):
    g = torch.Generator(device=DEV).manual_seed(tokens * experts)
    logits = (torch.randn((tokens, experts), generator=g, device=DEV) * 2).to(DT[dtype])
    bias = torch.randn((experts,), generator=g, device=DEV) * 0.1
    for b in (None, bias):
        for renorm, scaling in ((True, 2.5), (False, 1.0)):
            _check(logits, k, scoring, b, n_groups=groups, topk_groups=kept, group_top=top,
                   renormalize=renorm, scaling=scaling)


@pytest.mark.gpu
@SCORING
def test_ties_and_close_choices(scoring):
    """Equal choices go to the lower expert, equal groups to the lower group; choices that fp32
    would round to the same value keep their order."""
    x = torch.zeros((6, 64), device=DEV)
    x[1, ::3] = 1.0
    x[2, 63] = 1.0
    x[3] = 1.0 + torch.arange(64, device=DEV) * 2.0 ** -23
    x[4] = 14.0 + torch.arange(63, -1, -1, device=DEV) * 2.0 ** -20     # sigmoids near 1
    x[5, :32] = -0.0
    for groups, kept in ((1, 1), (8, 3), (32, 5)):
        for top in (1, 2):
            _check(x, 6, scoring, None, n_groups=groups, topk_groups=kept, group_top=top)
            _check(x, 6, scoring, torch.zeros(64, device=DEV), n_groups=groups, topk_groups=kept,
                   group_top=top)
    idx, _ = routing.select_experts(x[3:4], 4, scoring=scoring)
    assert idx.tolist() == [[63, 62, 61, 60]]


@pytest.mark.gpu
@SCORING
@pytest.mark.parametrize("base", [-500.0, -3.0, 0.0, 12.0, 40.0])
def test_logits_a_few_roundings_apart(scoring, base):
    """Logits, and choices under a bias that brings them next to each other, apart by 2^-24 to 2^-15
    of their size: on both sides of where fp32 can tell."""
    g = torch.Generator(device=DEV).manual_seed(int(base) + 600)
    e = 40
    for step in range(15, 25):
        i = torch.randint(-6, 7, (30, e), generator=g, device=DEV).double()
        x = (base + i * max(abs(base), 1.0) * 2.0 ** -step).float()
        # choices around 1/2, `step` binary places apart, for the first token's logits
        score = torch.softmax(x[0].double(), 0) if scoring == 0 else torch.sigmoid(x[0].double())
        bias = (0.5 + i[1] * 2.0 ** -step - score).float()
        x[10:20] = x[0]
        for b in (None, bias):
            for groups, kept, top in ((1, 1, 1), (8, 3, 2), (10, 4, 1)):
                _check(x, 7, scoring, b, n_groups=groups, topk_groups=kept, group_top=top)


@pytest.mark.gpu
@SCORING
@pytest.mark.parametrize("size", [3.0, 100.0, 2.0 ** 20, 3.0e38])
def test_groups_of_large_biases_that_cancel(scoring, size):
    """The two best choices of a group are a large bias and its negative, so that its sum is that of
    the scores, which fp32 has lost."""
    g = torch.Generator(device=DEV).manual_seed(13)
    x = torch.randn((256, 8, 5), generator=g, device=DEV) * 0.5
    x[:, :, 1] = x[:, :, 0]
    # the groups beside them: one score up and one down, by nearly the same
    d, e = torch.randn((2, 256, 4), generator=g, device=DEV)
    x[:, 1::2, 0] = x[:, ::2, 0] + d * 2.0 ** -16
    x[:, 1::2, 1] = x[:, ::2, 1] - d * 2.0 ** -16 + e * 2.0 ** -21
    bias = torch.full((8, 5), -3.2e38, device=DEV)
    bias[:, 0], bias[:, 1] = size, -size
    # one group whose sum is larger than fp32's range holds
    if size > 1e38:
        bias[6, 1] = size
    for kept in (1, 3, 4):
        _check(x.reshape(256, 40), 2, scoring, bias.reshape(40), n_groups=8, topk_groups=kept)


@pytest.mark.gpu
@pytest.mark.parametrize("below", [3.0, 5.44, 9.0])
def test_softmax_of_many_logits_below_the_largest(below):
    """1023 logits about 5.4 below the largest are where a sum of quick exponentials is off the
    most; the bias brings choices as close as that, and closer."""
    g = torch.Generator(device=DEV).manual_seed(14)
    e = 1024
    x = -below + torch.randn((1, e), generator=g, device=DEV).repeat(2, 1) * 2.0 ** -12
    x[:, 17] = 0.0
    score = torch.softmax(x[0].double(), 0)
    for step in range(17, 27):
        i = torch.randint(-3, 4, (e,), generator=g, device=DEV).double()
        bias = (score.max() * (2.0 + i * 2.0 ** -step) - score).float()
        for groups, kept, top in ((1, 1, 1), (16, 3, 2), (16, 3, 1)):
            _check(x, 8, abi.WISP_ROUTE_SOFTMAX, bias, n_groups=groups, topk_groups=kept,
                   group_top=top)


@pytest.mark.gpu
@SCORING
def test_values_that_cannot_be_chosen(scoring):
    """-infinite logits and biases, NaN, infinities, extreme logits, rows with too few experts left
    or none."""
    x = torch.randn((12, 48), generator=torch.Generator(device=DEV).manual_seed(5), device=DEV)
    x[0, 5] = NAN
    x[1, 5] = INF
    x[2, 5:40] = -INF
    x[3] = -INF
    x[4, 1:] = -INF
    x[5] = NAN
    x[6] = torch.finfo(torch.float32).min
    x[7, 3] = torch.finfo(torch.float32).max
    x[8] *= 400.0
    x[9] = INF
    x[10] = -1000.0
    bias = torch.randn((48,), generator=torch.Generator(device=DEV).manual_seed(6), device=DEV)
    masked = bias.clone()
    masked[6:46] = -INF
    masked[2] = NAN
    masked[47] = INF
    gone = torch.full_like(bias, -INF)
    for b in (None, bias, masked, gone):
        for groups, kept, top in ((1, 1, 1), (6, 2, 2), (6, 2, 1), (24, 8, 2)):
            for renorm in (True, False):
                idx, w = _check(x, 16, scoring, b, n_groups=groups, topk_groups=kept, group_top=top,
                                renormalize=renorm)
                assert (w[idx < 0] == 0).all()
    idx, w = routing.select_experts(x, 16, bias=gone, scoring=scoring)
    assert (idx == -1).all() and (w == 0).all()


@pytest.mark.gpu
def test_select_strided_rows_and_many_tokens():
    g = torch.Generator(device=DEV).manual_seed(9)
    big = torch.randn((700, 83), generator=g, device=DEV).to(torch.bfloat16)
    _check(big[:, 3:80], 6, abi.WISP_ROUTE_SOFTMAX, n_groups=7, topk_groups=3)
    idx, w = routing.select_experts(big[:0], 4)
    assert idx.shape == w.shape == (0, 4)
    # offsets past 32 bits
    rows = 2 ** 31 // 1024 + 3
    x = torch.zeros((rows, 1024), dtype=torch.bfloat16, device=DEV)
    x[-1, 1000:] = torch.arange(24, device=DEV).bfloat16() / 8
    idx, w = routing.select_experts(x, 4, scoring=abi.WISP_ROUTE_SOFTMAX)
    assert idx[-1].tolist() == [1023, 1022, 1021, 1020] and idx[-2].tolist() == [0, 1, 2, 3]


@pytest.mark.gpu
def test_select_on_a_stream_and_in_a_graph():
    g = torch.Generator(device=DEV).manual_seed(11)
    x = torch.randn((40, 64), generator=g, device=DEV)
    want = routing.select_experts(x, 4, n_groups=8, topk_groups=4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = routing.select_experts(x, 4, n_groups=8, topk_groups=4)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    static = x.clone()
    with torch.cuda.graph(graph):
        got = routing.select_experts(static, 4, n_groups=8, topk_groups=4)
    static.copy_(x.flip(0))
    graph.replay()
    assert torch.equal(got[0], want[0].flip(0)) and torch.equal(got[1], want[1].flip(0))


@pytest.mark.gpu
def test_dispatch_of_a_selection_with_empty_slots():
    """The selection feeds wisp_b200_dispatch_plan; slots without an expert are routed nowhere."""
    T, E, k = 20, 16, 4
    g = torch.Generator(device=DEV).manual_seed(12)
    x = torch.randn((T, E), generator=g, device=DEV)
    x[3] = NAN
    x[7, 2:] = -INF
    bias = torch.zeros(E, device=DEV)
    bias[9] = -INF
    idx, w = routing.select_experts(x, k, bias=bias)
    cfg = abi.WispMoeConfig()
    cfg.tokens, cfg.hidden, cfg.inter, cfg.n_experts, cfg.top_k, cfg.group_size = T, 128, 128, E, k, 128
    counts = torch.empty(E, dtype=torch.int32, device=DEV)
    segs = torch.empty((E, 4), dtype=torch.int32, device=DEV)
    tok = torch.full((T * k,), -7, dtype=torch.int32, device=DEV)
    wt = torch.empty(T * k, device=DEV)
    abi.call("wisp_b200_dispatch_plan", C.byref(cfg), idx.data_ptr(), w.data_ptr(), counts.data_ptr(),
             segs.data_ptr(), tok.data_ptr(), wt.data_ptr(), torch.cuda.current_stream().cuda_stream)
    flat = idx.flatten().tolist()
    at = 0
    for e in range(E):
        rows = [i // k for i, v in enumerate(flat) if v == e]
        assert segs[e].tolist() == [e, at, len(rows), 0]
        assert tok[at:at + len(rows)].tolist() == rows
        at += len(rows)
    assert counts[9] == 0 and at == sum(v >= 0 for v in flat) and 3 not in tok[:at].tolist()
