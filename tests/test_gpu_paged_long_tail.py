"""Attention in half precision over a long tail of keys far below the row's strongest, and with scores past 24 bits."""
from __future__ import annotations

import pytest
import torch

import _paged as P
from sparseattentioninfer_b200 import _capi, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
KEYS = 40000


def tail_tolerance(ref, mag, keys, top, tiles):
    """attention_tolerance, whose 2 u mag takes each weight's rounding as relative, and
    the weights that are too small for that: multiples of 2^-24, the least fp16, of 2^-7
    times the row's largest weight in tiles and of 2^-15 times it by rows, each is off by
    half of that at most."""
    return P.attention_tolerance(ref, mag, torch.float16) + keys * 2.0 ** (-32 if tiles else -40) * top


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new", [1, 5, 80])
@pytest.mark.parametrize("how", ["dense", "split", "kept"])
@pytest.mark.parametrize("drop", [12.7, 20.4, 26.3])
def test_a_strong_key_over_a_long_flat_tail(D, new, how, drop):
    """The first key outweighs each other one by 2^drop; its value is 0, theirs are not."""
    bt = P.Batch([KEYS], [new], Hq=4, Hkv=1, D=D, page=64, dtype=torch.float16, device=DEV)
    q = torch.zeros(new, 4, D, dtype=torch.float16)
    q[..., 0] = 8
    keys = torch.zeros(KEYS + new, 1, D)
    keys[0, 0, 0] = 8
    values = 64 + 16 * torch.randn(KEYS + new, 1, D, generator=bt.g)
    values[0] = 0
    k, v = bt.pool(keys=[keys]), bt.pool(keys=[values])
    scale = drop / 64 * 0.6931471805599453
    pages = bt.width
    kw, blocks = dict(max_q=new, max_len=KEYS + new), None
    if how == "split":
        kw["split_len"] = 2048
    if how == "kept":
        blocks = torch.arange(pages, dtype=torch.int32).expand(new, 1, pages).clone()
        last = (KEYS + torch.arange(new)) // 64
        blocks[blocks > last[:, None, None]] = -1
        kw["blocks"] = blocks.to(DEV)
    got = ops.paged_attention(q.to(DEV), k, v, *bt.batch, scale=scale, **kw)
    ref, mag = P.attention(bt, q, k, v, scale)
    tol = tail_tolerance(ref, mag, KEYS + new, values.abs().max().item(), tiles=4 * new > 16)
    err = (got.cpu().double() - ref).abs()
    assert (err <= tol).all(), (err / tol).max()
    assert _capi.device_error() == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("new,how", [(1, "dense"), (1, "split"), (1, "kept"), (5, "dense"), (80, "dense"), (80, "split"),
                                     (300, "kept")])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_past_24_bits(dtype, new, how, sign):
    """Scores of 2^23 to 2^30 (as exponents of 2), where none has bits left for fractions,
    equal or 8 apart: rows are means of values all the same, and of all values alike
    where the scores are equal."""
    n = 1000
    bt = P.Batch([n], [new], Hq=4, Hkv=1, D=64, page=16, dtype=dtype, device=DEV)
    values = 2 + torch.randn(n + new, 1, 64, generator=bt.g)
    v = bt.pool(keys=[values])
    q = torch.zeros(new, 4, 64, dtype=dtype)
    q[..., 0], q[..., 1] = sign * 2.0 ** 13, 1.0
    kw = dict(max_q=new, max_len=n + new)
    if how == "split":
        kw["split_len"] = 64
    if how == "kept":
        blocks = torch.arange(bt.width, dtype=torch.int32).expand(new, 1, bt.width).clone()
        blocks[blocks > ((n + torch.arange(new)) // 16)[:, None, None]] = -1
        kw["blocks"] = blocks.to(DEV)
    low, high = values.amin(0).to(dtype).double(), values.amax(0).to(dtype).double()
    scale = 8 * 0.6931471805599453
    for exponent in range(23, 31):
        for step in (0.0, 1.0):
            keys = torch.zeros(n + new, 1, 64)
            keys[:, 0, 0] = 2.0 ** (exponent - 16)
            keys[:, 0, 1] = step * (torch.arange(n + new) // 100)
            k = bt.pool(keys=[keys])
            got = ops.paged_attention(q.to(DEV), k, v, *bt.batch, scale=scale, **kw).cpu().double()
            assert (got >= low - 0.02 * low.abs()).all() and (got <= high + 0.02 * high.abs()).all(), (exponent, step)
            if step == 0:
                ref, mag = P.attention(bt, torch.zeros_like(q), k, v, 1.0)
                assert ((got - ref).abs() <= P.attention_tolerance(ref, mag, dtype)).all(), exponent
    assert _capi.device_error() == 0
