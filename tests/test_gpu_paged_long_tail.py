"""Attention in half precision over a long tail of keys far below the row's strongest."""
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
