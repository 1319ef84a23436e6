"""Outputs whose rows share memory are refused, on the host before any launch."""
from __future__ import annotations

import ctypes

import pytest

from sparseattentioninfer_b200 import _capi
from test_paged_cpu import FAKE, _attn, _batch, _pages


@pytest.mark.parametrize("strides", [(0, 128), (1024, 0), (64, 128), (1024, 64)])
def test_append_refuses_query_rows_that_overlap(strides):
    a = _capi.PagedAppendArgs()
    _batch(a.batch)
    for n in ("qkv", "q_weight", "k_weight", "cos", "sin", "q_out", "k_pages", "v_pages", "bounds"):
        setattr(a, n, FAKE)
    a.qkv_st, a.q_strides[0], a.q_strides[1] = 1536, *strides
    _pages(a, "k_strides", "v_strides", "b_strides")
    a.Hq, a.Hkv, a.D, a.positions, a.dtype, a.eps = 8, 2, 128, 100, _capi.SA_BF16, 1e-6
    assert _capi.load().sa_paged_append(ctypes.byref(a), None) == _capi.SA_ERR_INVALID


@pytest.mark.parametrize("which,stride", [(0, 64), (1, 64), (1, 8)])
def test_attention_refuses_rows_that_overlap(which, stride):
    a = _attn(o_strides=(which, stride))
    assert _capi.load().sa_paged_attn(ctypes.byref(a), None) == _capi.SA_ERR_INVALID
    assert b"out" in _capi.load().sa_last_error()
