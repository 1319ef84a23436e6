"""Page selection where scores cancel."""
from __future__ import annotations

import pytest
import torch

import _paged as P
from sparseattentioninfer_b200 import _capi, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _check(bt, q, bounds, keep, first, recent, **kw):
    out = torch.full((bt.N, bt.Hkv, keep), 99, dtype=torch.int32, device=DEV)
    ops.paged_block_select(q.to(DEV), bounds.to(DEV), *bt.batch, page_size=bt.page, keep=keep, first=first,
                           recent=recent, out=out, **kw)
    assert torch.equal(out.cpu(), P.select(bt, q, bounds, keep, first, recent))
    assert _capi.device_error() == 0


@pytest.mark.parametrize("new", [1, 7])
@pytest.mark.parametrize("pages", [20, 40, 300])
@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 64), (torch.float16, 128)])
@pytest.mark.parametrize("signs", ["both", "negative", "positive"])
def test_scores_that_cancel(new, pages, dtype, D, signs):
    """Scores some 2^15 times below the 32-bit sums' error, of one sign or both: the order
    is that of the 64-bit sums, and every entry of the result is written."""
    bt = P.Batch([pages * 16 - new], [new], Hq=1, Hkv=1, D=D, page=16, dtype=dtype, device=DEV, seed=pages)
    q = torch.zeros(new, 1, D, dtype=dtype)
    q[:, 0, [0, 1, 40]] = 1
    # (bf16 2^-30, fp16 its subnormals: multiples of 2^-24)
    i = torch.arange(pages)
    if dtype == torch.bfloat16:
        small = 2.0 ** -30 * (1 + (i * 5 % 64) / 64) * 2.0 ** (i // 64)
    else:
        small = 2.0 ** -24 * (1 + i * 7 % 512)
    sign = {"both": 1.0 - 2.0 * (i % 2), "negative": -torch.ones(pages), "positive": torch.ones(pages)}[signs]
    rows = torch.zeros(pages, D)
    rows[:, 0], rows[:, 1], rows[:, 40] = 1, -1, sign * small
    bounds = torch.zeros(bt.pages, 1, 2, D, dtype=dtype)
    bounds[bt.table[0].long()] = rows.to(dtype)[:, None, None].expand(-1, 1, 2, -1)
    for keep, first, recent in ((9, 1, 2), (12, 0, 1), (4, 1, 1)):
        _check(bt, q, bounds, keep, first, recent, max_q=new)
