"""Forward-mode automatic differentiation: no operator has a tangent, so a tensor that carries one
is refused instead of losing it. On CPU tensors, where the calls end at their refusals."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from wisp_b200 import abi, fp4, fp8, norm, routing

U8 = torch.uint8
Z = lambda *s, dtype=torch.float32: torch.zeros(s, dtype=dtype)

# each takes the tensor that may carry a tangent
CALLS = {
    "fp8 quantize": (lambda t: fp8.quantize(t), (2, 64)),
    "fp8 rows": (lambda t: fp8.dequantize(fp8.Fp8Rows(Z(2, 64, dtype=U8), t)), (2, 1)),
    "fp8 weights": (lambda t: fp8.Fp8Weights(Z(1, 2, 64, dtype=U8), t), (1, 1, 1)),
    "fp4 quantize": (lambda t: fp4.quantize(t, abi.WISP_FP4_MX), (2, 64)),
    "fp4 tensor scale": (lambda t: fp4.quantize(Z(2, 64), abi.WISP_FP4_NV, t), (1,)),
    "logits": (lambda t: routing.select_experts(t, 2), (2, 16)),
    "bias": (lambda t: routing.select_experts(Z(2, 16), 2, bias=t), (16,)),
    "norm x": (lambda t: norm.block_norm(t, post=False, pre_weight=Z(8)), (2, 8)),
    "norm y": (lambda t: norm.block_norm(Z(2, 8), t, pre=False), (2, 8)),
    "norm weight": (lambda t: norm.block_norm(Z(2, 8), pre_weight=t), (8,)),
    "norm output": (lambda t: norm.block_norm(Z(2, 8), pre_weight=Z(8), n_out=t), (2, 8)),
}


@pytest.mark.parametrize("name", list(CALLS))
def test_tangents_are_refused(name):
    call, shape = CALLS[name]
    with forward_ad.dual_level():
        t = forward_ad.make_dual(torch.ones(shape), torch.ones(shape))
        for mode in (torch.enable_grad, torch.no_grad):      # (both keep tangents)
            with mode(), pytest.raises(RuntimeError, match=r"wisp engine error \[4\].*tangent"):
                call(t)
        # without its tangent, or where none is followed, the call goes on
        with pytest.raises(RuntimeError, match="no CPU path"):
            call(t.detach())
        with torch.inference_mode(), pytest.raises(RuntimeError, match="no CPU path"):
            call(t)
    with pytest.raises(RuntimeError, match="no CPU path"):
        call(torch.ones(shape))
