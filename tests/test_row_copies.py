"""Copies and pickles of quantised rows: their addresses are those of their own tensors. (On the
CPU: an address of memory that has gone must not reach a kernel.)"""
from __future__ import annotations

import copy
import pickle

import pytest
import torch

from wisp_b200 import abi, fp4, fp8


def _fill(t):
    t.untyped_storage().copy_(torch.arange(t.untyped_storage().nbytes()).to(torch.uint8).untyped_storage())
    return t


def _fp8_own():
    """Rows as quantize makes them, in one buffer."""
    q = fp8.Fp8Rows._empty(torch.empty(0), 5, 272)
    _fill(q._buf)
    return q


def _fp8_given():
    return fp8.Fp8Rows(torch.arange(160, dtype=torch.uint8).view(5, 32), torch.rand(5, 2)[:, 1:])


def _fp4_own():
    q = fp4.Fp4Rows._empty(torch.empty(0), abi.WISP_FP4_NV, 5, 272, torch.rand(1))
    _fill(q._buf)
    return q


def _fp4_given():
    return fp4.Fp4Rows(abi.WISP_FP4_MX, torch.arange(80, dtype=torch.uint8).view(5, 16),
                       torch.arange(5, dtype=torch.uint8).view(5, 1))


MAKE = {"fp8 own": _fp8_own, "fp8 given": _fp8_given, "fp4 own": _fp4_own, "fp4 given": _fp4_given}
WAYS = {"copy": copy.copy, "deepcopy": copy.deepcopy, "pickle": lambda q: pickle.loads(pickle.dumps(q))}


@pytest.mark.parametrize("way", list(WAYS))
@pytest.mark.parametrize("make", list(MAKE))
def test_addresses_are_the_copys_own(make, way):
    q = MAKE[make]()
    c = WAYS[way](q)
    assert type(c) is type(q) and (c.rows, c.cols) == (q.rows, q.cols)
    assert c._codes == c.codes.data_ptr() and c._scales == c.scales.data_ptr()
    assert (c._codes == q._codes) == (way == "copy")
    assert torch.equal(c.codes.view(torch.uint8), q.codes.view(torch.uint8))
    assert torch.equal(c.scales.view(torch.uint8) if c.scales.is_contiguous() else c.scales,
                       q.scales.view(torch.uint8) if q.scales.is_contiguous() else q.scales)
    if isinstance(q, fp8.Fp8Rows):
        assert (c._row, c._block) == c.scales.stride()
    else:
        assert c.fmt == q.fmt and c._ts == fp4.ptr(c.tensor_scale)
        assert c.tensor_scale is None or torch.equal(c.tensor_scale, q.tensor_scale)
    q.codes.view(torch.uint8).fill_(0)
    assert (c.codes.view(torch.uint8) != 0).any() == (way != "copy")
