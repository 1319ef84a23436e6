"""Refusals of a caller's workspace, on the host before any launch."""
from __future__ import annotations

import ctypes

import pytest

from sparseattentioninfer_b200 import _capi
from test_paged_cpu import FAKE, _attn


@pytest.mark.parametrize("blocks", [None, FAKE])
@pytest.mark.parametrize("off", [4, 8, 12])
def test_a_workspace_that_is_not_aligned_is_refused(blocks, off):
    """The kernels store 16 bytes at a time to it: partial results, or pages of a tile."""
    lib = _capi.load()
    if blocks:
        a = _attn(batch=dict(N=500), max_q=250, blocks=blocks, n_blocks=40, blocks_strides=(0, 80))
    else:
        a = _attn(batch=dict(max_pages=4000, table_stride=4000), max_len=64000, split_len=4096)
    a.blocks_strides[1] = 40
    n = ctypes.c_int64(-1)
    assert lib.sa_paged_attn_workspace(ctypes.byref(a), ctypes.byref(n)) == 0 and n.value > 0
    a.workspace = FAKE + off
    assert lib.sa_paged_attn(ctypes.byref(a), None) == _capi.SA_ERR_INVALID
    assert b"aligned" in lib.sa_last_error()


@pytest.mark.parametrize("blocks", [None, FAKE])
@pytest.mark.parametrize("split_len", [0, 64])
def test_hints_up_to_the_largest_int(blocks, split_len):
    """max_q steers by what it says of the batch, which has no more tokens than N."""
    n = ctypes.c_int64(-1)
    need = []
    for max_q in (500, 2 ** 31 - 1):
        a = _attn(batch=dict(N=500, B=1), max_q=max_q, split_len=split_len, blocks=blocks, n_blocks=40)
        a.blocks_strides[0], a.blocks_strides[1] = 80, 40
        assert _capi.load().sa_paged_attn_workspace(ctypes.byref(a), ctypes.byref(n)) == 0
        need.append(n.value)
    assert need[0] == need[1]
