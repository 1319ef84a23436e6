"""Lists of kept pages at their limits."""
from __future__ import annotations

import pytest
import torch

import _paged as P
from sparseattentioninfer_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("call", [ops.paged_attention, ops.paged_attention_workspace])
def test_lists_without_entries_are_refused(call):
    bt = P.Batch([40], [3], Hq=4, Hkv=2, D=64, page=16, device=DEV)
    q = torch.randn(3, 4, 64, generator=bt.g).to(torch.bfloat16).to(DEV)
    k, v = bt.pool(), bt.pool()
    lists = torch.zeros(3, 2, 4, dtype=torch.int32, device=DEV)
    for none in (lists[..., :0], lists[..., :0].clone()):
        with pytest.raises(ValueError, match="blocks"):
            call(q, k, v, *bt.batch, blocks=none)
    # (a batch without rows is no such call)
    cu = torch.zeros(2, dtype=torch.int32, device=DEV)
    call(q[:0], k, v, bt.batch[0], cu, bt.batch[2], blocks=lists[:0])
