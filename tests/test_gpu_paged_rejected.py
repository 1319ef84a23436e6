"""Page bounds after drafts were rejected and their slots written again."""
from __future__ import annotations

import math

import pytest
import torch

import _paged as P
from sparseattentioninfer_b200 import _capi, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("D,page,dtype,layout", [
    (64, 16, torch.bfloat16, "heads"), (128, 32, torch.float16, "slots"), (64, 64, torch.float16, "wide"),
    (128, 128, torch.bfloat16, "heads"),
])
@pytest.mark.parametrize("poison", [100.0, math.nan, math.inf])
def test_bounds_are_of_the_keys_that_stay(D, page, dtype, layout, poison):
    """Prompts, drafts with extreme keys, then other tokens over the drafts' slots: bit for
    bit the bounds of the keys that the pages then hold, as if the drafts had never been."""
    Hq, Hkv, B = 4, 2, 4
    g = torch.Generator().manual_seed(D + page)
    wide = 4
    table = torch.randperm(B * wide + 1, generator=g)[:B * wide].view(B, wide).int()
    first = P.Batch([0] * B, [1] * B, Hq=Hq, Hkv=Hkv, D=D, page=page, dtype=dtype, device=DEV, layout=layout)
    pool = torch.full((B * wide + 1, Hkv, page, D), float("nan"), dtype=dtype)
    k, v = first.place(pool), first.place(pool)
    bounds = torch.full((B * wide + 1, Hkv, 2, D), float("nan"), dtype=dtype, device=DEV)
    w = torch.ones(D, dtype=dtype, device=DEV)
    cos, sin = (torch.full((4 * page, D), c, dtype=dtype, device=DEV) for c in (1.0, 0.0))

    def append(lens, new, fill=None):
        bt = P.Batch(lens, new, Hq=Hq, Hkv=Hkv, D=D, page=page, dtype=dtype, device=DEV, width=wide, layout=layout)
        bt.table, bt.pages = table, B * wide + 1
        x = torch.randn(bt.N, Hq + 2 * Hkv, D, generator=g).to(dtype)
        if fill is not None:
            x[:, Hq:, ::3] = fill
            x[:, Hq:, 1::3] = -fill
        ops.paged_qk_norm_rope_append(x.to(DEV), None if fill else w, None if fill else w, cos, sin, k, v, *bt.batch,
                                      Hq=Hq, Hkv=Hkv, k_bounds=bounds)
        assert _capi.device_error() == 0
        return bt

    start = [page // 2 - 1, 2 * page - 2, page, 1]
    append([0] * B, start)  # (pages shared by a CTA's warps where sequences bring many tokens)
    lens = start
    for drafts, kept, again in (([5] * B, [2, 1, 0, 3], [1] * B), ([3, 4, 5, 6], [1, 2, 0, 0], [17, 16, 20, 31]),
                                ([page - 7] * B, [0, 1, 2, 3], [2, 0, 1, 1])):
        append(lens, drafts, poison)
        # the kept drafts are sound tokens in earnest: write those again too
        bt = append(lens, [a + b for a, b in zip(kept, again)])
        lens = bt.lens
        want = P.bounds_of(bt, k, fill=float("nan"))
        used = torch.cat([table[b, :math.ceil(n / page)] for b, n in enumerate(lens)]).long()
        got = bounds.cpu()
        assert torch.equal(got[used], want[used]) and not want[used].isnan().any()
