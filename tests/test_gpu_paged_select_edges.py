"""Page selection where scores cancel, bounds are not finite and tables are long."""
from __future__ import annotations

import math

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


@pytest.mark.parametrize("new", [1, 5])
@pytest.mark.parametrize("side", [0, 1])
def test_a_bound_that_is_no_number_ranks_its_page_lowest(new, side):
    """A NaN in either bound, whatever the sign of the heads' values in that channel."""
    bt = P.Batch([50 * 16], [new], Hq=2, Hkv=1, D=64, page=16, device=DEV)
    q = torch.randn(new, 2, 64, generator=bt.g).to(torch.bfloat16)
    q[:, :, 7] = -q[:, :, 7].abs() - 0.5
    q[:, :, 9] = q[:, :, 9].abs() + 0.5
    bounds = torch.ones(bt.pages, 1, 2, 64, dtype=torch.bfloat16)
    bounds[bt.table[0, 5:20].long(), 0, side, 7] = math.nan
    bounds[bt.table[0, 20:30].long(), 0, side, 9] = math.nan
    _check(bt, q, bounds, 30, 1, 1, max_q=new)


@pytest.mark.parametrize("new", [1, 5])
def test_zero_times_an_infinite_bound_is_zero(new):
    """Heads whose value in the channel is 0 take nothing from it, others do."""
    bt = P.Batch([50 * 16], [new], Hq=3, Hkv=1, D=64, page=16, device=DEV)
    q = torch.randn(new, 3, 64, generator=bt.g).to(torch.bfloat16)
    q[:, :, 7] = 0
    q[:, 0, 9] = 0
    q[:, 1:, 9] = -1
    bounds = torch.ones(bt.pages, 1, 2, 64, dtype=torch.bfloat16)
    low = torch.randn(bt.pages, 64, generator=bt.g)
    bounds[:, 0, 0], bounds[:, 0, 1] = low.to(torch.bfloat16), (low + 1).to(torch.bfloat16)
    plain = bounds.clone()
    some = bt.table[0, 5:30].long()
    bounds[some, 0, 0, 7], bounds[some, 0, 1, 7] = -math.inf, math.inf
    bounds[some, 0, 1, 9] = math.inf  # (the heads of -1 take the low one)
    plain[some, 0, :, 7] = 0
    plain[some, 0, 1, 9] = plain[some, 0, 0, 9]
    got = ops.paged_block_select(q.to(DEV), bounds.to(DEV), *bt.batch, page_size=16, keep=12, max_q=new)
    assert torch.equal(got.cpu(), P.select(bt, q, plain, 12, 1, 1))
    assert _capi.device_error() == 0


@pytest.mark.parametrize("pages,Hkv", [(5000, 2), (16384, 1)])
@pytest.mark.parametrize("spread", [1.0, 0.0])
def test_long_tables(pages, Hkv, spread):
    """One token over more pages than a CTA's registers hold, up to the longest table;
    with all pages equal, too."""
    bt = P.Batch([pages * 16 - 3, 40], [1, 1], Hq=3 * Hkv, Hkv=Hkv, D=64, page=16, device=DEV)
    q = torch.randn(2, 3 * Hkv, 64, generator=bt.g).to(torch.bfloat16)
    low = torch.randn(bt.pages, Hkv, 64, generator=bt.g) * spread
    bounds = torch.stack([low - 1, low + 1], 2).to(torch.bfloat16)
    _check(bt, q, bounds, 64, 1, 2, max_q=1)
    _check(bt, q, bounds, 4096, 0, 1, max_q=1)
