"""Argument checks of the paged-cache entry points, on the host before any launch."""
from __future__ import annotations

import ctypes

import pytest
import torch

from sparseattentioninfer_b200 import _capi, ops

FAKE = 1 << 20  # never dereferenced: validation fails before any launch


def _batch(b, **over):
    b.table = b.cu_q = b.seq_lens = FAKE
    b.table_stride, b.B, b.N, b.max_pages, b.num_pages, b.page_size = 10, 2, 5, 10, 40, 16
    for k, v in over.items():
        setattr(b, k, v)


def _pages(a, *names, D=128, Hkv=2, page=16):
    for n in names:
        st = getattr(a, n)
        st[0], st[1], st[2] = Hkv * page * D, page * D, D


def _attn(batch=None, **over):
    a = _capi.PagedAttnArgs()
    _batch(a.batch, **(batch or {}))
    a.q = a.out = a.k_pages = a.v_pages = FAKE
    a.Hq, a.Hkv, a.D, a.dtype, a.scale, a.max_q, a.max_len, a.num_sms = 8, 2, 128, _capi.SA_BF16, 0.1, 1, 160, 148
    a.q_strides[0] = a.o_strides[0] = 1024
    a.q_strides[1] = a.o_strides[1] = 128
    _pages(a, "k_strides", "v_strides")
    for k, v in over.items():
        if isinstance(v, tuple):
            getattr(a, k)[v[0]] = v[1]
        else:
            setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,code", [
    (dict(q=None), _capi.SA_ERR_INVALID),
    (dict(k_pages=None), _capi.SA_ERR_INVALID),
    (dict(k_pages=FAKE + 8), _capi.SA_ERR_INVALID),
    (dict(q=FAKE + 2), _capi.SA_ERR_INVALID),
    (dict(D=96), _capi.SA_ERR_UNSUPPORTED),
    (dict(dtype=7), _capi.SA_ERR_UNSUPPORTED),
    (dict(Hq=7), _capi.SA_ERR_INVALID),
    (dict(scale=0.0), _capi.SA_ERR_INVALID),
    (dict(scale=float("nan")), _capi.SA_ERR_INVALID),
    (dict(max_q=0), _capi.SA_ERR_INVALID),
    (dict(max_len=0), _capi.SA_ERR_INVALID),
    (dict(split_len=-1), _capi.SA_ERR_INVALID),
    (dict(blocks=FAKE, n_blocks=0), _capi.SA_ERR_INVALID),
    (dict(q_strides=(0, 1020)), _capi.SA_ERR_INVALID),
    (dict(o_strides=(1, 0)), _capi.SA_ERR_INVALID),
    (dict(k_strides=(2, 132)), _capi.SA_ERR_INVALID),
    (dict(v_strides=(0, 1 << 36)), _capi.SA_ERR_INVALID),
    (dict(batch=dict(page_size=48)), _capi.SA_ERR_UNSUPPORTED),
    (dict(batch=dict(page_size=256)), _capi.SA_ERR_UNSUPPORTED),
    (dict(batch=dict(N=0)), _capi.SA_ERR_INVALID),
    (dict(batch=dict(cu_q=None)), _capi.SA_ERR_INVALID),
    (dict(batch=dict(table_stride=9)), _capi.SA_ERR_INVALID),
    (dict(batch=dict(max_pages=1 << 28, table_stride=1 << 28)), _capi.SA_ERR_INVALID),
])
def test_attention_refusals(over, code):
    lib = _capi.load()
    a = _attn(**over)
    assert lib.sa_paged_attn(ctypes.byref(a), None) == code
    assert lib.sa_last_error()
    n = ctypes.c_int64(-1)
    assert lib.sa_paged_attn_workspace(ctypes.byref(a), ctypes.byref(n)) == code and n.value == -1


def test_attention_workspace_is_wanted_only_for_long_splits():
    lib = _capi.load()
    n = ctypes.c_int64(-1)

    def need(**over):
        assert lib.sa_paged_attn_workspace(ctypes.byref(_attn(**over)), ctypes.byref(n)) == 0
        return n.value

    assert need() == 0
    long = dict(batch=dict(max_pages=4000, table_stride=4000), max_len=64000)
    splits = -(-64000 // 4096)
    assert need(split_len=4096, **long) == 5 * 8 * splits * (128 + 2)
    assert need(split_len=64000, **long) == 0
    a = _attn(split_len=4096, **long)
    assert lib.sa_paged_attn(ctypes.byref(a), None) == _capi.SA_ERR_WORKSPACE
    assert b"workspace" in lib.sa_last_error()
    assert lib.sa_paged_attn(None, None) == lib.sa_paged_attn_workspace(None, ctypes.byref(n)) == _capi.SA_ERR_INVALID


@pytest.mark.parametrize("over,code", [
    (dict(qkv=None), _capi.SA_ERR_INVALID),
    (dict(cos=FAKE + 4), _capi.SA_ERR_INVALID),
    (dict(D=32), _capi.SA_ERR_UNSUPPORTED),
    (dict(dtype=2), _capi.SA_ERR_UNSUPPORTED),
    (dict(Hkv=3), _capi.SA_ERR_INVALID),
    (dict(positions=0), _capi.SA_ERR_INVALID),
    (dict(qkv_st=1538), _capi.SA_ERR_INVALID),
    (dict(bounds=FAKE + 8), _capi.SA_ERR_INVALID),
    (dict(v_pages=None), _capi.SA_ERR_INVALID),
])
def test_append_refusals(over, code):
    a = _capi.PagedAppendArgs()
    _batch(a.batch)
    for n in ("qkv", "q_weight", "k_weight", "cos", "sin", "q_out", "k_pages", "v_pages", "bounds"):
        setattr(a, n, FAKE)
    a.qkv_st, a.q_strides[0], a.q_strides[1] = 1536, 1024, 128
    _pages(a, "k_strides", "v_strides", "b_strides")
    a.Hq, a.Hkv, a.D, a.positions, a.dtype, a.eps = 8, 2, 128, 100, _capi.SA_FP16, 1e-6
    for k, v in over.items():
        setattr(a, k, v)
    assert _capi.load().sa_paged_append(ctypes.byref(a), None) == code
    assert _capi.load().sa_paged_append(None, None) == _capi.SA_ERR_INVALID


@pytest.mark.parametrize("over,code", [
    (dict(out=None), _capi.SA_ERR_INVALID),
    (dict(bounds=None), _capi.SA_ERR_INVALID),
    (dict(recent=0), _capi.SA_ERR_INVALID),
    (dict(first=-1), _capi.SA_ERR_INVALID),
    (dict(first=4, recent=4), _capi.SA_ERR_INVALID),
    (dict(keep=5000, first=0), _capi.SA_ERR_INVALID),
    (dict(max_q=0), _capi.SA_ERR_INVALID),
    (dict(D=256), _capi.SA_ERR_UNSUPPORTED),
    (dict(batch=dict(max_pages=20000, table_stride=20000)), _capi.SA_ERR_UNSUPPORTED),
])
def test_select_refusals(over, code):
    a = _capi.PagedSelectArgs()
    over = dict(over)
    _batch(a.batch, **over.pop("batch", {}))
    a.q = a.bounds = a.out = FAKE
    a.q_strides[0], a.q_strides[1], a.out_strides[0], a.out_strides[1] = 1024, 128, 10 ** 4, 5000
    _pages(a, "b_strides")
    a.Hq, a.Hkv, a.D, a.dtype, a.keep, a.first, a.recent, a.max_q = 8, 2, 128, _capi.SA_BF16, 6, 1, 2, 1
    for k, v in over.items():
        setattr(a, k, v)
    assert _capi.load().sa_paged_select(ctypes.byref(a), None) == code
    assert _capi.load().sa_paged_select(None, None) == _capi.SA_ERR_INVALID


def test_wrappers_refuse_host_tensors_and_wrong_shapes():
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16)
    pages = torch.zeros(5, 2, 16, 64, dtype=torch.bfloat16)
    batch = (torch.zeros(1, 2, dtype=torch.int32), torch.tensor([0, 3], dtype=torch.int32),
             torch.tensor([3], dtype=torch.int32))
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.paged_attention(q, pages, pages, *batch)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.paged_block_select(q, torch.zeros(5, 2, 2, 64, dtype=torch.bfloat16), *batch, page_size=16, keep=2)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.paged_qk_norm_rope_append(torch.zeros(3, 8, 64, dtype=torch.bfloat16), None, None, q[0], q[0], pages,
                                      pages, *batch, Hq=4, Hkv=2)
