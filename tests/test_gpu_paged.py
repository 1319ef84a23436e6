"""The paged-cache operators against their definitions in 64 bits (tests/_paged.py)."""
from __future__ import annotations

import math
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import _paged as P
from sparseattentioninfer_b200 import _capi, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def rope_tables(n, D, dtype, theta=1e6):
    ang = torch.outer(torch.arange(n, dtype=torch.float64), theta ** (-torch.arange(0, D, 2, dtype=torch.float64) / D))
    ang = torch.cat([ang, ang], -1)
    return ang.cos().to(dtype), ang.sin().to(dtype)


# --------------------------------------------------------------------- append
@pytest.mark.parametrize("ctx,new,Hq,Hkv,D,page,dtype,layout,pad", [
    ([0], [1], 4, 1, 64, 16, torch.bfloat16, "heads", 0),                                  # the very first token
    ([5, 0, 31, 16], [1, 1, 1, 1], 8, 2, 128, 16, torch.bfloat16, "heads", 3),             # decode, page starts and ends
    ([0, 7, 100, 3], [37, 0, 65, 1], 6, 2, 128, 32, torch.float16, "slots", 0),            # ragged, one without tokens
    ([63, 64, 1], [130, 129, 300], 20, 4, 64, 64, torch.bfloat16, "wide", 5),
    ([200] * 40, [2] * 40, 9, 3, 128, 128, torch.float16, "heads", 1),
    ([10], [1000], 16, 8, 64, 128, torch.bfloat16, "slots", 0),
])
@pytest.mark.parametrize("normed", [True, False])
def test_append(ctx, new, Hq, Hkv, D, page, dtype, layout, pad, normed):
    bt = P.Batch(ctx, new, Hq=Hq, Hkv=Hkv, D=D, page=page, dtype=dtype, device=DEV, seed=len(ctx), pad=pad,
                 layout=layout)
    g = bt.g
    total = Hq + 2 * Hkv
    qkv = (3 * torch.randn(bt.N, total, D, generator=g)).to(dtype)
    qw, kw = ((1 + 0.1 * torch.randn(D, generator=g)).to(dtype) for _ in range(2))
    cos, sin = rope_tables(max(bt.lens), D, dtype)
    old = P.Batch(ctx, [0] * len(ctx), Hq=Hq, Hkv=Hkv, D=D, page=page, dtype=dtype)
    old.table, old.pages, old.g = bt.table, bt.pages, g
    k0, v0 = old.pool(), old.pool()
    k_pages, v_pages = bt.place(k0), bt.place(v0)
    bounds = P.bounds_of(bt, k0, lens=ctx, fill=float("nan")).to(DEV)
    q_out = torch.full((bt.N, Hq, D), 7.0, dtype=dtype, device=DEV)
    # (token rows of a wider buffer)
    wide = torch.full((bt.N, total * D + 16), float("nan"), dtype=dtype, device=DEV)
    wide[:, 8:8 + total * D] = qkv.to(DEV).view(bt.N, -1)
    src = wide[:, 8:8 + total * D].view(bt.N, total, D)
    got = ops.paged_qk_norm_rope_append(
        src, qw.to(DEV) if normed else None, kw.to(DEV) if normed else None, cos.to(DEV), sin.to(DEV), k_pages,
        v_pages, *bt.batch, Hq=Hq, Hkv=Hkv, eps=1e-6, k_bounds=bounds, q_out=q_out)
    assert got is q_out and _capi.device_error() == 0
    # q and k: |y c| + |y' s| carries the 32-bit errors (sum of D squares, rsqrt: below 2^-16), one rounding on top
    x = qkv[:, :Hq + Hkv].double()
    if normed:
        x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + 1e-6)
        x = torch.cat([x[:, :Hq] * qw.double(), x[:, Hq:] * kw.double()], 1)
    u = torch.finfo(dtype).eps / 2
    rows = torch.tensor([r for r, _, _ in bt.tokens()])
    pos = torch.tensor([p for _, _, p in bt.tokens()])
    c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
    x = x[rows]
    ref = x * c + torch.cat([-x[..., D // 2:], x[..., :D // 2]], -1) * s
    size = (x * c).abs() + (torch.cat([x[..., D // 2:], x[..., :D // 2]], -1) * s).abs()
    tol = u * ref.abs() + 2.0 ** -16 * size + torch.finfo(dtype).tiny
    assert ((got.cpu().double()[rows] - ref[:, :Hq]).abs() <= tol[:, :Hq]).all()
    if pad:
        assert (got[bt.N - pad:] == 7.0).all()
    kp, vp = k_pages.cpu(), v_pages.cpu()
    k0, v0 = k0.clone(), v0.clone()
    for i, (r, b, p) in enumerate(bt.tokens()):
        page_, slot = int(bt.table[b, p // page]), p % page
        assert ((kp[page_, :, slot].double() - ref[i, Hq:]).abs() <= tol[i, Hq:]).all()
        k0[page_, :, slot] = kp[page_, :, slot]
        v0[page_, :, slot] = qkv[r, Hq + Hkv:]
    assert torch.equal(kp.view(torch.int16), k0.view(torch.int16))  # nothing else was written
    assert torch.equal(vp.view(torch.int16), v0.view(torch.int16))
    want = P.bounds_of(bt, kp, fill=float("nan"))
    assert torch.equal(bounds.cpu().nan_to_num(77.0), want.nan_to_num(77.0))


def test_append_in_pieces_gives_the_same_cache():
    """One call and a token at a time: the same pages and bounds, bit for bit."""
    Hq, Hkv, D, page, n = 4, 2, 128, 16, 50
    bt = P.Batch([3], [n], Hq=Hq, Hkv=Hkv, D=D, page=page, device=DEV)
    qkv = torch.randn(n, Hq + 2 * Hkv, D, generator=bt.g).to(torch.bfloat16).to(DEV)
    w = torch.ones(D, dtype=torch.bfloat16, device=DEV)
    cos, sin = (t.to(DEV) for t in rope_tables(64, D, torch.bfloat16))
    res = []
    for step in (n, 1, 7):
        k, v = (torch.zeros(bt.pages, Hkv, page, D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        bounds = torch.zeros(bt.pages, Hkv, 2, D, dtype=torch.bfloat16, device=DEV)
        table = bt.table.to(DEV)
        qs = []
        for i in range(0, n, step):
            m = min(step, n - i)
            cu, ln = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([0, m], [3 + i + m]))
            qs.append(ops.paged_qk_norm_rope_append(qkv[i:i + m], w, w, cos, sin, k, v, table, cu, ln, Hq=Hq,
                                                    Hkv=Hkv, k_bounds=bounds))
        res.append((torch.cat(qs), k, v, bounds))
    for other in res[1:]:
        for a, b in zip(res[0], other):
            assert torch.equal(a, b)
    assert _capi.device_error() == 0


# ------------------------------------------------------------------ attention
ATTN = [
    # ctx, new, Hq, Hkv, D, page, dtype, layout, pad
    ([0], [1], 1, 1, 64, 16, torch.bfloat16, "heads", 0),
    ([0, 1, 14, 15, 16, 63, 64, 200], [1] * 8, 8, 2, 128, 16, torch.bfloat16, "heads", 2),
    ([700, 3, 128, 255], [1, 1, 0, 1], 12, 4, 64, 32, torch.float16, "slots", 1),
    ([100, 0, 600, 31], [3, 5, 0, 2], 8, 2, 128, 64, torch.bfloat16, "wide", 0),
    ([129, 1000], [1, 4], 40, 2, 128, 128, torch.float16, "heads", 0),      # 20 heads a group
    ([65, 0], [33, 70], 6, 2, 64, 16, torch.bfloat16, "slots", 3),
    ([0, 300, 17], [200, 129, 1], 8, 8, 128, 32, torch.bfloat16, "heads", 0),
    ([0], [260], 10, 2, 128, 64, torch.float16, "heads", 0),                # 5 heads a group
    ([513], [140], 16, 1, 64, 128, torch.bfloat16, "wide", 4),
    ([0, 0, 90], [1, 257, 40], 3, 1, 128, 128, torch.float16, "heads", 0),
]


def _qkv(bt, std=1.5):
    q = (std * torch.randn(bt.N, bt.Hq, bt.D, generator=bt.g)).to(bt.dtype)
    return q, bt.pool(), bt.pool()


def _assert_attention(bt, got, q, k, v, scale, blocks=None, before=None):
    ref, mag = P.attention(bt, q, k, v, scale, blocks)
    n = sum(bt.new)
    err = (got.cpu().double()[:n] - ref[:n]).abs()
    tol = P.attention_tolerance(ref[:n], mag[:n], bt.dtype)
    assert (err <= tol).all(), (err / tol).max()
    if before is not None:
        assert torch.equal(got[n:].cpu(), before[n:].cpu())
    assert _capi.device_error() == 0


@pytest.mark.parametrize("ctx,new,Hq,Hkv,D,page,dtype,layout,pad", ATTN)
@pytest.mark.parametrize("hints", ["exact", "none", "wrong", "split"])
def test_attention(ctx, new, Hq, Hkv, D, page, dtype, layout, pad, hints):
    """Slots behind a sequence's length hold NaN, table entries behind it -7."""
    bt = P.Batch(ctx, new, Hq=Hq, Hkv=Hkv, D=D, page=page, dtype=dtype, device=DEV, seed=Hq + D, pad=pad,
                 layout=layout)
    q, k, v = _qkv(bt)
    kw = {"exact": dict(max_q=max(new), max_len=max(bt.lens)), "none": {}, "wrong": dict(max_q=1),
          "split": dict(max_q=max(new), split_len=64)}[hints]
    out = torch.full((bt.N, Hq, D), 3.0, dtype=dtype, device=DEV)
    before = out.clone()
    got = ops.paged_attention(q.to(DEV), k, v, *bt.batch, out=out, **kw)
    assert got is out
    _assert_attention(bt, got, q, k, v, 1 / math.sqrt(D), before=before)


def _random_blocks(bt, keep, seed=0, empty=False):
    g = torch.Generator().manual_seed(seed)
    out = torch.full((bt.N, bt.Hkv, keep), -1, dtype=torch.int32)
    for r, b, pos in bt.tokens():
        for h in range(bt.Hkv):
            last = pos // bt.page
            n = min(keep, int(torch.randint(0 if empty else 1, last + 2, (1,), generator=g)))
            got = torch.randperm(last + 1, generator=g)[:n].sort().values
            out[r, h, :n] = got.int()
    return out


@pytest.mark.parametrize("ctx,new,Hq,Hkv,D,page,dtype,layout,pad", ATTN)
@pytest.mark.parametrize("keep,split_len", [(1, None), (5, 64), (9, None), (30, 128)])
@pytest.mark.parametrize("max_q", [1, None])
def test_sparse_attention(ctx, new, Hq, Hkv, D, page, dtype, layout, pad, keep, split_len, max_q):
    bt = P.Batch(ctx, new, Hq=Hq, Hkv=Hkv, D=D, page=page, dtype=dtype, device=DEV, seed=keep, pad=pad, layout=layout)
    q, k, v = _qkv(bt)
    blocks = _random_blocks(bt, keep, empty=True)  # some lists are empty: those rows are 0
    out = torch.full((bt.N, Hq, D), 3.0, dtype=dtype, device=DEV)
    before = out.clone()
    ops.paged_attention(q.to(DEV), k, v, *bt.batch, blocks=blocks.to(DEV), split_len=split_len, max_q=max_q,
                        out=out)
    _assert_attention(bt, out, q, k, v, 1 / math.sqrt(D), blocks, before)


# Calls that tiles of 128 rows serve, over kept pages too: groups that divide 128 and
# that do not, more pages than one, two and three batches of 32, single tokens and
# sequences without new ones among the chunks.
TILES = [
    ([2100, 0], [260, 100], 4, 4, 128, 16, torch.bfloat16, "heads", 3),
    ([1000, 40, 7], [333, 64, 1], 16, 8, 64, 16, torch.float16, "slots", 0),
    ([1600, 0, 3], [70, 290, 0], 24, 8, 64, 32, torch.bfloat16, "wide", 2),
    ([129, 0], [150, 301], 40, 8, 128, 64, torch.bfloat16, "heads", 0),
    ([4500], [500], 6, 6, 64, 64, torch.float16, "heads", 1),
    ([600, 0], [190, 400], 20, 10, 128, 128, torch.float16, "heads", 0),
]


@pytest.mark.parametrize("ctx,new,Hq,Hkv,D,page,dtype,layout,pad", TILES)
@pytest.mark.parametrize("keep", [None, 3, 40])
@pytest.mark.parametrize("split_len", [None, 192])
def test_tiles(ctx, new, Hq, Hkv, D, page, dtype, layout, pad, keep, split_len):
    bt = P.Batch(ctx, new, Hq=Hq, Hkv=Hkv, D=D, page=page, dtype=dtype, device=DEV, seed=D + page, pad=pad,
                 layout=layout)
    q, k, v = _qkv(bt)
    blocks = None if keep is None else _random_blocks(bt, keep, seed=1, empty=True)
    kw = dict(max_q=max(new), max_len=max(bt.lens), split_len=split_len,
              blocks=None if blocks is None else blocks.to(DEV))
    if keep == 40:  # (room for the unions of the lists: tiles it is; three small pages may go by rows)
        assert ops.paged_attention_workspace(q.to(DEV), k, v, *bt.batch, **kw) > 0
    out = torch.full((bt.N, Hq, D), 3.0, dtype=dtype, device=DEV)
    before = out.clone()
    ops.paged_attention(q.to(DEV), k, v, *bt.batch, out=out, **kw)
    _assert_attention(bt, out, q, k, v, 1 / math.sqrt(D), blocks, before)


@pytest.mark.parametrize("D,new", [(128, 5), (64, 9), (128, 1)])
@pytest.mark.parametrize("hint", [None, 1, 3])
def test_drafts_of_many_sequences(D, new, hint):
    """A few tokens of each of many sequences: by rows or by tiles, whichever the sizes ask for."""
    bt = P.Batch([1500 + 7 * i for i in range(40)], [new - i % 2 * (new > 1) for i in range(40)], Hq=8, Hkv=2, D=D,
                 page=32, device=DEV)
    q, k, v = _qkv(bt)
    got = ops.paged_attention(q.to(DEV), k, v, *bt.batch, max_q=hint or new, max_len=max(bt.lens))
    _assert_attention(bt, got, q, k, v, 1 / math.sqrt(D))


def test_attention_scale_and_strided_rows():
    bt = P.Batch([40, 3], [5, 9], Hq=4, Hkv=2, D=64, page=16, device=DEV)
    q, k, v = _qkv(bt)
    wide = torch.full((bt.N, 9, 64 + 16), float("nan"), dtype=torch.bfloat16, device=DEV)
    wide[:, 2:6, 8:72] = q.to(DEV)
    res = torch.zeros(6, bt.N, 64, dtype=torch.bfloat16, device=DEV)
    ops.paged_attention(wide[:, 2:6, 8:72], k, v, *bt.batch, scale=0.3, out=res.transpose(0, 1)[:, 1:5])
    _assert_attention(bt, res.transpose(0, 1)[:, 1:5], q, k, v, 0.3)
    assert (res[0] == 0).all() and (res[5] == 0).all()


# -------------------------------------------------------------------- select
@pytest.mark.parametrize("ctx,new,Hq,Hkv,D,page,dtype,layout,pad", ATTN + [
    ([9000, 40, 4111], [1, 1, 3], 8, 2, 128, 16, torch.bfloat16, "heads", 0),
])
@pytest.mark.parametrize("keep,first,recent", [(1, 0, 1), (4, 1, 2), (8, 0, 3), (70, 2, 5)])
def test_select(ctx, new, Hq, Hkv, D, page, dtype, layout, pad, keep, first, recent):
    bt = P.Batch(ctx, new, Hq=Hq, Hkv=Hkv, D=D, page=page, dtype=dtype, device=DEV, seed=3, pad=pad)
    q = torch.randn(bt.N, Hq, D, generator=bt.g).to(dtype)
    bounds = P.bounds_of(bt, bt.pool(), fill=float("nan"))
    out = torch.full((bt.N, Hkv, keep), 99, dtype=torch.int32, device=DEV)
    ops.paged_block_select(q.to(DEV), bounds.to(DEV), *bt.batch, page_size=page, keep=keep, first=first,
                           recent=recent, max_q=max(new), out=out)
    n = sum(new)
    assert torch.equal(out[:n].cpu(), P.select(bt, q, bounds, keep, first, recent)[:n])
    assert (out[n:] == 99).all()
    assert _capi.device_error() == 0


@pytest.mark.parametrize("new,ctx", [(1, 64 * 16), (6, 64 * 16), (1, 10000), (3, 10000)])
def test_select_ties_nan_and_infinities(new, ctx):
    """Equal pages go to the lower index; NaN scores rank with -infinity; 1 ulp decides."""
    bt = P.Batch([ctx], [new], Hq=2, Hkv=1, D=64, page=16, device=DEV)
    q = torch.randn(new, 2, 64, generator=bt.g).to(torch.bfloat16)
    for case in range(4):
        bounds = torch.ones(bt.pages, 1, 2, 64, dtype=torch.bfloat16)
        if case == 1:  # every second page better by one unit in the last place of one channel
            bounds[bt.table[0, ::2].long(), 0, :, 17] *= 1 + 2 ** -7
        if case == 2:
            bounds[bt.table[0, 3:40].long(), 0, 1, 5] = math.nan
            bounds[bt.table[0, 50].long()] = -math.inf
        if case == 3:
            bounds[bt.table[0, 10].long(), 0, 1] = math.inf
            bounds[bt.table[0, 11].long(), 0, 0] = -math.inf
        got = ops.paged_block_select(q.to(DEV), bounds.to(DEV), *bt.batch, page_size=16, keep=20, first=1, recent=1)
        assert torch.equal(got.cpu(), P.select(bt, q, bounds, 20, 1, 1)), case


# -------------------------------------------------------------------- as used
def test_prefill_then_decode_with_kept_pages():
    """Append, select and attend over several steps of three sequences: whole
    prompts, then single tokens over kept pages, against dense attention in 64
    bits over what the cache then holds."""
    Hq, Hkv, D, page, B = 8, 2, 128, 16, 3
    g = torch.Generator().manual_seed(0)
    k, v = (torch.full((64, Hkv, page, D), float("nan"), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    bounds = torch.full((64, Hkv, 2, D), float("nan"), dtype=torch.bfloat16, device=DEV)
    w = torch.ones(D, dtype=torch.bfloat16, device=DEV)
    cos, sin = (t.to(DEV) for t in rope_tables(400, D, torch.bfloat16))
    table = torch.randperm(64, generator=g)[:B * 20].view(B, 20).int()
    lens = [0] * B
    for new in ([100, 33, 257], [1, 1, 1], [1, 0, 1], [4, 1, 2]):
        bt = P.Batch(lens, new, Hq=Hq, Hkv=Hkv, D=D, page=page, device=DEV, width=20)
        bt.table, bt.pages = table, 64
        lens = bt.lens
        qkv = torch.randn(bt.N, Hq + 2 * Hkv, D, generator=g).to(torch.bfloat16).to(DEV)
        q = ops.paged_qk_norm_rope_append(qkv, w, w, cos, sin, k, v, *bt.batch, Hq=Hq, Hkv=Hkv, k_bounds=bounds)
        out = ops.paged_attention(q, k, v, *bt.batch, max_q=max(new), max_len=max(lens))
        _assert_attention(bt, out, q.cpu(), k, v, 1 / math.sqrt(D))
        kept = ops.paged_block_select(q, bounds, *bt.batch, page_size=page, keep=5, first=1, recent=2)
        assert torch.equal(kept.cpu(), P.select(bt, q, bounds, 5, 1, 2))
        out = ops.paged_attention(q, k, v, *bt.batch, blocks=kept)
        _assert_attention(bt, out, q.cpu(), k, v, 1 / math.sqrt(D), kept)


@pytest.mark.parametrize("keep", [None, 4])
def test_captured_steps_replay_as_the_cache_grows(keep):
    """One captured decode step (append, select, attend) replayed for a growing,
    ragged batch equals the same steps run eagerly; the lengths, offsets and page
    table are read on the device."""
    Hq, Hkv, D, page, B, steps = 8, 2, 128, 16, 3, 6
    g = torch.Generator().manual_seed(1)
    start = [14, 0, 95]
    w = torch.ones(D, dtype=torch.bfloat16, device=DEV)
    cos, sin = (t.to(DEV) for t in rope_tables(128, D, torch.bfloat16))
    table = torch.randperm(40, generator=g)[:B * 8].view(B, 8).int().to(DEV)
    pool = [torch.randn(40, Hkv, page, D, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2)]
    inputs = torch.randn(steps, B, Hq + 2 * Hkv, D, generator=g).to(torch.bfloat16).to(DEV)
    cu = torch.arange(B + 1, dtype=torch.int32, device=DEV)
    bt = P.Batch(start, [0] * B, Hq=Hq, Hkv=Hkv, D=D, page=page, width=8)
    bt.table, bt.pages = table.cpu(), 40

    def run(graph):
        k, v = (t.clone() for t in pool)
        bounds = P.bounds_of(bt, k).to(DEV)
        lens = torch.tensor(start, dtype=torch.int32, device=DEV)
        x = inputs[0].clone()

        def step():
            lens.add_(1)
            q = ops.paged_qk_norm_rope_append(x, w, w, cos, sin, k, v, table, cu, lens, Hq=Hq, Hkv=Hkv,
                                              k_bounds=bounds)
            blocks = None if keep is None else ops.paged_block_select(q, bounds, table, cu, lens, page_size=page,
                                                                      keep=keep, max_q=1)
            return ops.paged_attention(q, k, v, table, cu, lens, max_q=1, blocks=blocks, split_len=64)

        outs = []
        if graph:
            cg = torch.cuda.CUDAGraph()
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                step()
            torch.cuda.current_stream().wait_stream(s)
            with torch.cuda.graph(cg):
                out = step()
            for t, u in zip((k, v), pool):
                t.copy_(u)
            bounds.copy_(P.bounds_of(bt, k))
            lens.copy_(torch.tensor(start, dtype=torch.int32))
        for i in range(steps):
            x.copy_(inputs[i])
            if graph:
                cg.replay()
                outs.append(out.clone())
            else:
                outs.append(step())
        return torch.stack(outs), k, v, bounds

    for a, b in zip(run(False), run(True)):
        assert torch.equal(a, b)
    assert _capi.device_error() == 0


def test_side_stream_and_caller_workspace():
    bt = P.Batch([700, 30], [1, 1], Hq=4, Hkv=2, D=64, page=32, device=DEV)
    q, k, v = _qkv(bt)
    q = q.to(DEV)
    args = (q, k, v, *bt.batch)
    kw = dict(max_q=1, max_len=2000, split_len=64)  # more splits than a cluster joins
    n = ops.paged_attention_workspace(*args, **kw)
    assert n > 0
    want = ops.paged_attention(*args, **kw)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    ws = torch.full((n,), float("nan"), device=DEV)
    with torch.cuda.stream(s):
        got = ops.paged_attention(*args, workspace=ws, **kw)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    with pytest.raises(ValueError, match="workspace"):
        ops.paged_attention(*args, workspace=ws[:-1], **kw)
    _assert_attention(bt, got, q.cpu(), k, v, 1 / math.sqrt(64))


def test_pages_past_two_to_the_31_elements():
    """The pages in use lie behind the first 2^31 elements of the pools."""
    Hq, Hkv, D, page = 16, 8, 128, 128
    pages = 2 ** 31 // (Hkv * page * D) + 20
    bt = P.Batch([300, 5], [4, 150], Hq=Hq, Hkv=Hkv, D=D, page=page, device=DEV)
    small = [bt.pool(), bt.pool()]
    big = [torch.empty(pages, Hkv, page, D, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    at = pages - bt.pages
    for b, s in zip(big, small):
        b[at:] = s
    far = (bt.table + at).to(DEV)
    x = torch.randn(bt.N, Hq + 2 * Hkv, D, generator=bt.g).to(torch.bfloat16).to(DEV)
    cos, sin = (t.to(DEV) for t in rope_tables(400, D, torch.bfloat16))
    res = []
    for (k, v), table in ((small, bt.table.to(DEV)), (big, far)):
        bounds = torch.zeros(k.shape[0], Hkv, 2, D, dtype=torch.bfloat16, device=DEV)
        cu, ln = bt.batch[1:]
        q = ops.paged_qk_norm_rope_append(x, None, None, cos, sin, k, v, table, cu, ln, Hq=Hq, Hkv=Hkv,
                                          k_bounds=bounds)
        kept = ops.paged_block_select(q, bounds, table, cu, ln, page_size=page, keep=2)
        res.append([q, kept] + [ops.paged_attention(q, k, v, table, cu, ln, **kw) for kw in
                                (dict(max_q=1), dict(max_q=150), dict(blocks=kept, max_q=1), dict(blocks=kept))])
    for a, b in zip(*res):
        assert torch.equal(a, b)
    assert torch.equal(big[0][at:].view(torch.int16), small[0].view(torch.int16))
    assert _capi.device_error() == 0


def test_many_heads_a_group_and_many_sequences():
    for ctx, new, Hq, Hkv in (([70, 0], [1, 3], 136, 1), ([33] * 70, [1, 2] * 35, 4, 2)):
        bt = P.Batch(ctx, new, Hq=Hq, Hkv=Hkv, D=64, page=16, device=DEV)
        q, k, v = _qkv(bt)
        for kw in ({}, dict(max_q=1)):
            _assert_attention(bt, ops.paged_attention(q.to(DEV), k, v, *bt.batch, **kw), q, k, v, 0.125)


@pytest.mark.parametrize("max_q", [1, 64])
def test_bad_batches_are_reported_and_left_out(max_q):
    """What the device finds wrong sets the error word; the sound sequences come out right."""
    def batch():
        bt = P.Batch([50, 20, 40], [3, 30, 2], Hq=8, Hkv=2, D=64, page=16, device=DEV, seed=5)
        return bt, *_qkv(bt)

    def attend(bt, q, k, v, table, cu, lens):
        out = torch.full(q.shape, 7.0, dtype=q.dtype, device=DEV)
        ops.paged_attention(q.to(DEV), k, v, table, cu, lens, max_q=max_q, out=out)
        assert _capi.device_error() == 2
        assert _capi.device_error() == 0  # read and cleared
        ref, mag = P.attention(bt, q, k, v, 0.125)
        ok = ((out.cpu().double() - ref).abs() <= P.attention_tolerance(ref, mag, q.dtype)).all(-1).all(-1)
        return out, [bool(ok[s:s + n].all()) for s, n in zip(bt.starts, bt.new)]

    bt, q, k, v = batch()
    table, cu, lens = bt.batch
    for bad in (-1, bt.pages, 2 ** 30):  # a page that is not there: its keys are left out
        t = table.clone()
        t[1, 0] = bad
        _, good = attend(bt, q, k, v, t, cu, lens)
        assert good == [True, False, True]
    n = lens.clone()
    n[1] = 29  # fewer keys than new tokens
    out, good = attend(bt, q, k, v, table, cu, n)
    assert good == [True, False, True] and (out[3:33] == 7).all()
    n[1] = 16 * bt.width + 1  # more keys than the table holds
    _, good = attend(bt, q, k, v, table, cu, n)
    assert good[0] and good[2]
    c = cu.clone()
    c[3] = bt.N + 9  # rows that are not there
    out, good = attend(bt, q, k, v, table, c, lens)
    assert good == [True, True, False]
    blocks = _random_blocks(bt, 4)
    blocks[4, 1] = torch.tensor([2, 2, -1, -1])  # not ascending
    blocks[5, 0] = torch.tensor([0, 3, 10 ** 6, -1])  # behind the token
    got = torch.zeros_like(q, device=DEV)
    ops.paged_attention(q.to(DEV), k, v, table, cu, lens, max_q=max_q, out=got, blocks=blocks.to(DEV))
    assert _capi.device_error() == 2
    ref, mag = P.attention(bt, q, k, v, 0.125, blocks.where(blocks < 99, -1))
    ok = ((got.cpu().double() - ref).abs() <= P.attention_tolerance(ref, mag, q.dtype)).flatten(1).all(1)
    assert ok[[i for i in range(bt.N) if i not in (4, 5)]].all()
    # select and append
    bounds = P.bounds_of(bt, k).to(DEV)
    t = table.clone()
    t[1, 1] = bt.pages
    got = ops.paged_block_select(q.to(DEV), bounds, t, cu, lens, page_size=16, keep=2, first=0, recent=1).cpu()
    assert _capi.device_error() == 2
    want = P.select(bt, q, bounds, 2, 0, 1)
    assert torch.equal(got[:3], want[:3]) and torch.equal(got[33:], want[33:])
    cos, sin = (x.to(DEV) for x in rope_tables(52, 64, torch.bfloat16))  # position 52 has no angle
    x = torch.randn(bt.N, 12, 64, generator=bt.g).to(torch.bfloat16).to(DEV)
    kb = k.clone()
    ops.paged_qk_norm_rope_append(x, None, None, cos, sin, kb, v.clone(), t, cu, lens, Hq=8, Hkv=2, k_bounds=bounds)
    assert _capi.device_error() == 2
    changed = (kb.view(torch.int16) != k.view(torch.int16)).flatten(2).any(-1).any(-1).nonzero().flatten().tolist()
    allowed = {int(table[0, 3]), int(table[1, 2]), int(table[1, 3]), int(table[2, 2])}
    assert set(changed) <= allowed and _capi.device_error() == 0


def test_a_sequence_with_nan_does_not_reach_the_others():
    bt = P.Batch([40, 50, 20], [20, 1, 20], Hq=4, Hkv=2, D=64, page=16, device=DEV)
    q, k, v = _qkv(bt)
    want = [ops.paged_attention(q.to(DEV), k, v, *bt.batch, max_q=m) for m in (1, 20)]
    for t in (k, v):
        t[bt.table[1, 1].item()] = float("nan")
    for w, m in zip(want, (1, 20)):
        got = ops.paged_attention(q.to(DEV), k, v, *bt.batch, max_q=m)
        assert torch.equal(got[:20], w[:20]) and torch.equal(got[21:], w[21:]) and got[20].isnan().all()


@pytest.mark.parametrize("max_q", [1, 64])
def test_offsets_that_leave_the_batch_or_decrease(max_q):
    """A last offset far behind the batch drops the last sequence alone, the longest
    though it is; offsets that decrease are reported by each operator."""
    bt = P.Batch([20, 0, 300], [3, 30, 5], Hq=8, Hkv=2, D=64, page=16, device=DEV)
    q, k, v = _qkv(bt)
    table, cu, lens = bt.batch
    ref, mag = P.attention(bt, q, k, v, 0.125)
    far = cu.clone()
    far[3] = 2 ** 30
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device=DEV)
    ops.paged_attention(q.to(DEV), k, v, table, far, lens, max_q=max_q, out=out)
    assert _capi.device_error() == 2
    ok = (out.cpu().double() - ref).abs() <= P.attention_tolerance(ref, mag, q.dtype)
    assert ok[:33].all() and (out[33:] == 7).all()
    bounds = P.bounds_of(bt, k).to(DEV)
    cos, sin = (x.to(DEV) for x in rope_tables(400, 64, torch.bfloat16))
    x = torch.randn(bt.N, 12, 64, generator=bt.g).to(torch.bfloat16).to(DEV)
    for bad in ([0, 9, 3, 38], [0, 33, 3, 3], [0, 3, 33, 20]):
        c = torch.tensor(bad, dtype=torch.int32, device=DEV)
        ops.paged_attention(q.to(DEV), k, v, table, c, lens, max_q=max_q)
        assert _capi.device_error() == 2, bad
        ops.paged_block_select(q.to(DEV), bounds, table, c, lens, page_size=16, keep=4, max_q=max_q)
        assert _capi.device_error() == 2, bad
        ops.paged_qk_norm_rope_append(x, None, None, cos, sin, k.clone(), v.clone(), table, c, lens, Hq=8, Hkv=2)
        assert _capi.device_error() == 2, bad


def test_the_first_calls_of_a_process_may_be_captured():
    """Nothing that the operators set up once needs a call before the capture."""
    code = """
import torch
from sparseattentioninfer_b200 import _capi, ops
D, N, dev = 128, 3, "cuda"
k, v = (torch.randn(64, 2, 16, D, device=dev).bfloat16() for _ in range(2))
bounds = torch.zeros(64, 2, 2, D, device=dev, dtype=torch.bfloat16)
table = torch.arange(64, device=dev, dtype=torch.int32).view(1, 64)
cu = torch.tensor([0, N], device=dev, dtype=torch.int32)
lens = torch.tensor([900], device=dev, dtype=torch.int32)
cos, sin = (torch.randn(1024, D, device=dev).bfloat16() for _ in range(2))
qkv = torch.randn(N, 12, D, device=dev).bfloat16()
def step():
    q = ops.paged_qk_norm_rope_append(qkv, None, None, cos, sin, k, v, table, cu, lens, Hq=8, Hkv=2, k_bounds=bounds)
    kept = ops.paged_block_select(q, bounds, table, cu, lens, page_size=16, keep=8, max_q=N)
    return [q, kept] + [ops.paged_attention(q, k, v, table, cu, lens, **kw) for kw in
            (dict(max_q=N), dict(max_q=N, max_len=1024, split_len=64), dict(max_q=64), dict(blocks=kept, max_q=N))]
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got = step()
g.replay()
torch.cuda.synchronize()
got = [t.clone() for t in got]
assert all(torch.equal(a, b) for a, b in zip(got, step())) and _capi.device_error() == 0
print("same")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                       cwd=str(Path(__file__).resolve().parents[1]))
    assert r.returncode == 0 and r.stdout.strip() == "same", r.stderr[-2000:]


def test_out_of_memory_is_torchs_own_error():
    """A result that does not fit is refused by the allocator before anything is launched."""
    q = torch.zeros(1, 1, 64, dtype=torch.bfloat16, device=DEV)
    k = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16, device=DEV)
    i = torch.zeros(2, dtype=torch.int32, device=DEV)
    with pytest.raises(torch.OutOfMemoryError):
        ops.paged_block_select(q.expand(2 ** 28, 1, 64), k, i[:1].view(1, 1), i, i[:1], page_size=16, keep=4096)


def test_bad_lists_and_pages_in_tiles():
    """Lists that do not ascend, entries behind the token and pages that are not there
    are reported; rows that do not keep them come out right."""
    bt = P.Batch([700, 60], [250, 150], Hq=8, Hkv=4, D=128, page=32, device=DEV, seed=9)
    q, k, v = _qkv(bt)
    table, cu, lens = bt.batch
    blocks = _random_blocks(bt, 20)
    bad_rows = {4: [2, 2], 37: [0, 3, 10 ** 6], 255: [5, 1, 2], 300: [0, 6, 7]}  # (300 sees 3 pages)
    for r, entries in bad_rows.items():
        blocks[r, 1] = -1
        blocks[r, 1, :len(entries)] = torch.tensor(entries)
    kw = dict(max_q=250, max_len=max(bt.lens))
    assert ops.paged_attention_workspace(q.to(DEV), k, v, table, cu, lens, blocks=blocks.to(DEV), **kw) > 0  # tiles
    got = torch.full(q.shape, 3.0, dtype=q.dtype, device=DEV)
    ops.paged_attention(q.to(DEV), k, v, table, cu, lens, blocks=blocks.to(DEV), out=got, **kw)
    assert _capi.device_error() == 2
    sound = blocks.clone()
    for r in bad_rows:
        sound[r, 1] = -1
    ref, mag = P.attention(bt, q, k, v, 128 ** -0.5, sound)
    ok = ((got.cpu().double() - ref).abs() <= P.attention_tolerance(ref, mag, q.dtype)).all(-1)  # [N, Hq]
    ok[list(bad_rows), 2:4] = True  # (the two heads of kv head 1)
    assert ok.all()
    t = table.clone()
    t[0, 7] = bt.pages
    sound = torch.where((blocks == 7) & (torch.arange(bt.N) < 250)[:, None, None], -2, blocks)
    keeps = (sound == -2).any(-1)  # [N, Hkv]
    ops.paged_attention(q.to(DEV), k, v, t, cu, lens, blocks=blocks.to(DEV), out=got, **kw)
    assert _capi.device_error() == 2
    ok = ((got.cpu().double() - ref).abs() <= P.attention_tolerance(ref, mag, q.dtype)).all(-1)
    ok[list(bad_rows), 2:4] = True
    assert (ok | keeps.repeat_interleave(2, 1)).all() and keeps.any() and not keeps.all()
