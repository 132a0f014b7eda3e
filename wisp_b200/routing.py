"""Which experts each token goes to, from the router's logits: softmax or sigmoid scores, a
bias that chooses without weighing, groups, top-k (wisp_b200_select_experts in
include/wisp_b200.h)."""
from __future__ import annotations

import ctypes as C
from functools import lru_cache

import torch

from . import abi
from .fp4 import INT_MAX, dtype_code, elsewhere, invalid, refuse_grad, row_stride, same_device, stream_of, \
    wants_grad


def policy(scoring: int = abi.WISP_ROUTE_SIGMOID, n_groups: int = 1, topk_groups: int = 1,
           group_top: int = 2, renormalize: bool = True, scaling: float = 1.0) -> abi.WispRouting:
    """How tokens are routed, for select_experts and fp8.Fp8MoeLayer."""
    counts = [int(v) for v in (scoring, n_groups, topk_groups, group_top)]
    if not all(0 <= v <= INT_MAX for v in counts):
        raise invalid(f"scoring, n_groups, topk_groups, group_top: {counts}")
    return abi.WispRouting(*counts, 1 if renormalize else 0, float(scaling))


@lru_cache(maxsize=64)
def _policy(scoring, n_groups, topk_groups, group_top, renormalize, scaling):
    r = policy(scoring, n_groups, topk_groups, group_top, renormalize, scaling)
    return r, C.byref(r)


def check_bias(bias: torch.Tensor | None, n_experts: int, what: str = "bias") -> None:
    if bias is not None and (bias.dtype != torch.float32 or bias.shape != (n_experts,) or
                             not bias.is_contiguous()):
        raise invalid(f"{what}: contiguous float32 [{n_experts}]")


def select_experts(logits: torch.Tensor, top_k: int, *, bias: torch.Tensor | None = None,
                   scoring: int = abi.WISP_ROUTE_SIGMOID, n_groups: int = 1, topk_groups: int = 1,
                   group_top: int = 2, renormalize: bool = True, scaling: float = 1.0):
    """(idx int32 [tokens, top_k], weights float32 [tokens, top_k]) of logits [tokens, experts]
    (float32, bfloat16 or float16):

        score  = softmax(logits) or sigmoid(logits);  choice = score + bias
        the topk_groups of n_groups groups with the largest sum of their group_top best choices
        idx    = the top_k of their experts by choice, largest first
        weight = score (renormalize: / the sum over the top_k) * scaling

    Computed in 64 bits; ties go to the lower index. NaN and -infinite choices are never taken;
    slots without an expert have idx -1 and weight 0. No gradient: tensors that require one are
    refused under grad mode, and those with a tangent."""
    if wants_grad(logits, bias):
        refuse_grad()
    ld = row_stride(logits, "logits")
    tokens, experts = logits.shape
    dt = dtype_code(logits.dtype, "logits")
    check_bias(bias, experts)
    other = elsewhere(logits)
    if other is not None:
        with other:
            return select_experts(logits, top_k, bias=bias, scoring=scoring, n_groups=n_groups,
                                  topk_groups=topk_groups, group_top=group_top,
                                  renormalize=renormalize, scaling=scaling)
    if bias is not None:
        same_device(logits, bias=bias)
    if not 0 < top_k <= 32:
        raise invalid(f"top_k={top_k} (1..32)")
    # (as numbers: what the cache keeps may not change behind it)
    _, r = _policy(int(scoring), int(n_groups), int(topk_groups), int(group_top),
                   bool(renormalize), float(scaling))
    idx = logits.new_empty((tokens, top_k), dtype=torch.int32)
    w = logits.new_empty((tokens, top_k), dtype=torch.float32)
    abi.call("wisp_b200_select_experts", r, logits.data_ptr(), dt, ld, tokens, experts,
             top_k, None if bias is None else bias.data_ptr(), idx.data_ptr(), w.data_ptr(),
             stream_of(logits))
    return idx, w
