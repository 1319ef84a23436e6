"""Lists of kept pages at their limits: none, and lists that do not ascend."""
from __future__ import annotations

import pytest
import torch

import _paged as P
from sparseattentioninfer_b200 import _capi, ops

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


@pytest.mark.parametrize("max_q", [1, 250])
@pytest.mark.parametrize("split_len", [None, 64])
def test_a_list_ends_at_its_first_bad_entry(max_q, split_len):
    """An entry that does not ascend or lies behind the token ends the list, by rows and
    by tiles alike: no page counts twice, and nothing behind it counts."""
    bt = P.Batch([700, 60], [250, 150], Hq=8, Hkv=4, D=128, page=32, device=DEV, seed=9)
    q = (1.5 * torch.randn(bt.N, 8, 128, generator=bt.g)).to(torch.bfloat16)
    k, v = bt.pool(), bt.pool()
    g = torch.Generator().manual_seed(3)
    lists = torch.full((bt.N, 4, 20), -1, dtype=torch.int32)
    for r, b, pos in bt.tokens():
        for h in range(4):
            got = torch.randperm(pos // 32 + 1, generator=g)[:20].sort().values
            lists[r, h, :got.numel()] = got.int()
    sound = lists.clone()
    bad = {4: ([3, 1, 3], 1), 37: ([0, 3, 10 ** 6], 2), 255: ([1, 1, 2], 1), 300: ([0, 2, 7, 8], 2),
           90: ([5, 1, 6, 9], 1), 91: ([2, 3, 3, 4, 5], 2), 120: ([4, 2 ** 31 - 1, 5], 1), 249: ([22, 22, 22, 23], 1),
           100: (list(range(19)) + [3], 19)}
    for r, (entries, good) in bad.items():
        for t, n in ((lists, len(entries)), (sound, good)):
            t[r, 1] = -1
            t[r, 1, :n] = torch.tensor(entries[:n])
    kw = dict(max_q=max_q, max_len=max(bt.lens), split_len=split_len)
    got = torch.full(q.shape, 3.0, dtype=q.dtype, device=DEV)
    ops.paged_attention(q.to(DEV), k, v, *bt.batch, blocks=lists.to(DEV), out=got, **kw)
    assert _capi.device_error() == 2
    ref, mag = P.attention(bt, q, k, v, 128 ** -0.5, sound)
    assert ((got.cpu().double() - ref).abs() <= P.attention_tolerance(ref, mag, q.dtype)).all()
