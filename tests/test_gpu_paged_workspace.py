"""A caller's workspace cut from a larger buffer."""
from __future__ import annotations

import pytest
import torch

import _paged as P
from sparseattentioninfer_b200 import _capi, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("kept", [False, True])
def test_slices_of_an_arena(kept):
    """16-byte aligned slices serve, others are refused before anything is launched."""
    bt = P.Batch([900], [200], Hq=8, Hkv=2, D=64, page=16, device=DEV)
    q = torch.randn(200, 8, 64, generator=bt.g).to(torch.bfloat16).to(DEV)
    args = (q, bt.pool(), bt.pool(), *bt.batch)
    kw = dict(max_q=200, max_len=1100, split_len=64)
    if kept:
        kw["blocks"] = torch.arange(40, dtype=torch.int32, device=DEV).expand(200, 2, 40)
    n = ops.paged_attention_workspace(*args, **kw)
    assert n > 0
    want = ops.paged_attention(*args, **kw)
    arena = torch.full((n + 12,), float("nan"), device=DEV)
    for at in (1, 2, 3, 5):
        with pytest.raises(ValueError, match="aligned"):
            ops.paged_attention(*args, workspace=arena[at:at + n], **kw)
    assert arena.isnan().all()
    assert torch.equal(ops.paged_attention(*args, workspace=arena[4:4 + n], **kw), want)
    assert arena[:4].isnan().all() and arena[4 + n:].isnan().all() and _capi.device_error() == 0
