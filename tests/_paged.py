"""Packed batches on a paged cache, and the paged operators from their
definitions in 64 bits."""
from __future__ import annotations

import math

import torch


class Batch:
    """Sequences with ``ctx`` cached keys and ``new`` new tokens each, pages in random order."""

    def __init__(self, ctx, new, *, Hq, Hkv, D, page, dtype=torch.bfloat16, device="cpu", seed=0, pad=0, spare=2,
                 width=None, layout="heads"):
        self.ctx, self.new, self.page, self.Hq, self.Hkv, self.D, self.dtype = ctx, new, page, Hq, Hkv, D, dtype
        self.lens = [a + b for a, b in zip(ctx, new)]
        self.N, self.B = sum(new) + pad, len(ctx)
        g = self.g = torch.Generator().manual_seed(seed)
        self.width = width or max(1, max(math.ceil(t / page) for t in self.lens))
        need = [math.ceil(t / page) for t in self.lens]
        self.pages = sum(need) + spare
        order = torch.randperm(self.pages, generator=g)
        self.table = torch.full((self.B, self.width), -7, dtype=torch.int32)  # entries behind the length: never read
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.cu_q = torch.tensor([sum(new[:b]) for b in range(self.B + 1)], dtype=torch.int32)
        self.seq_lens = torch.tensor(self.lens, dtype=torch.int32)
        self.starts = [sum(new[:b]) for b in range(self.B)]
        self.layout, self.device = layout, device

    def pool(self, fill=float("nan"), std=1.0, keys=None):
        """[pages, Hkv, page, D] pool holding ``keys`` (or random ones) where the
        sequences' keys are and ``fill`` everywhere else."""
        P, H, ps, D = self.pages, self.Hkv, self.page, self.D
        t = torch.full((P, H, ps, D), fill).to(self.dtype)
        for b, n in enumerate(self.lens):
            x = std * torch.randn(n, H, D, generator=self.g) if keys is None else keys[b]
            for p in range(math.ceil(n / ps)):
                part = x[p * ps:(p + 1) * ps]
                t[int(self.table[b, p]), :, :part.shape[0]] = part.transpose(0, 1).to(self.dtype)
        return self.place(t)

    def place(self, t):
        """The pool on the device in the batch's layout."""
        if self.layout == "slots":  # [pages, page, Hkv, D] underneath
            return t.transpose(1, 2).contiguous().to(self.device).transpose(1, 2)
        if self.layout == "wide":  # every page padded, heads apart
            P, H, ps, D = t.shape
            w = torch.full((P + 1, H + 1, ps, D + 8), float("nan"), dtype=t.dtype)
            w[1:, 1:, :, 8:] = t
            return w.to(self.device)[1:, 1:, :, 8:]
        return t.to(self.device)

    def on(self, *ts):
        return [t.to(self.device) for t in ts]

    @property
    def batch(self):
        return self.on(self.table, self.cu_q, self.seq_lens)

    def keys_of(self, pool, b, n=None):
        """[keys, Hkv, D] of sequence b in 64 bits."""
        n = self.lens[b] if n is None else n
        pos = torch.arange(n)
        return pool.cpu()[self.table[b, pos // self.page].long(), :, pos % self.page].double()

    def tokens(self):
        """(row, sequence, position) of every token."""
        for b in range(self.B):
            for i in range(self.new[b]):
                yield self.starts[b] + i, b, self.ctx[b] + i


def attention(bt: Batch, q, k_pool, v_pool, scale, blocks=None):
    """out [N, Hq, D] and the same sums with |v| (for the rounding of P), in 64 bits; NaN rows are nobody's."""
    out = torch.full(q.shape, float("nan"), dtype=torch.float64)
    mag = out.clone()
    q = q.cpu().double()
    G = bt.Hq // bt.Hkv
    for b in range(bt.B):
        n = bt.new[b]
        if not n:
            continue
        r = slice(bt.starts[b], bt.starts[b] + n)
        k = bt.keys_of(k_pool, b).repeat_interleave(G, 1).transpose(0, 1)  # [Hq, keys, D]
        v = bt.keys_of(v_pool, b).repeat_interleave(G, 1).transpose(0, 1)
        x = q[r].transpose(0, 1) @ k.transpose(1, 2) * scale
        pos = bt.ctx[b] + torch.arange(n)
        seen = (torch.arange(bt.lens[b]) <= pos[:, None]).expand(bt.Hq, -1, -1).clone()
        if blocks is not None:
            kept = torch.zeros(n, bt.Hkv, bt.width + 1, dtype=torch.bool)
            kept.scatter_(2, blocks[r].cpu().long() % (bt.width + 1), True)
            kept = kept[..., torch.arange(bt.lens[b]) // bt.page]
            seen &= kept.transpose(0, 1).repeat_interleave(G, 0)
        x = x.masked_fill(~seen, -math.inf)
        p = torch.exp(x - x.amax(-1, keepdim=True).clamp_min(-1e300))
        p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
        out[r], mag[r] = (p @ v).transpose(0, 1), (p @ v.abs()).transpose(0, 1)
    return out, mag


def attention_tolerance(ref, mag, dtype):
    """|error| bound. u = eps/2 is one rounding to the type. Rounding each P_j moves
    the weighted sum by at most u * sum P_j |v_j| and the sum of the rounded P by
    u, together 2 u mag; the stored value rounds once more, u |o|. In 32 bits, D
    products of a score with |scale q.k| summed to at most 16 err by
    16 * D * 2^-24 <= 2^-13 and the exponentials, sums and joins by less than
    that again: 2^-11 mag covers them."""
    u = torch.finfo(dtype).eps / 2
    return 1.02 * (u * ref.abs() + 2 * u * mag) + 2.0 ** -11 * mag + torch.finfo(dtype).tiny


def bounds_of(bt: Batch, k_pool, lens=None, fill=0.0):
    """[pages, Hkv, 2, D]: lowest and highest key per channel of each page in use."""
    P, H, ps, D = bt.pages, bt.Hkv, bt.page, bt.D
    out = torch.full((P, H, 2, D), fill).to(bt.dtype)
    pool = k_pool.cpu()
    for b, n in enumerate(bt.lens if lens is None else lens):
        for p in range(math.ceil(n / ps)):
            page = int(bt.table[b, p])
            held = pool[page, :, :min(ps, n - p * ps)]
            out[page, :, 0], out[page, :, 1] = held.amin(1), held.amax(1)
    return out


def select(bt: Batch, q, bounds, keep, first, recent):
    """[N, Hkv, keep] by the definition: scores per query head in 64 bits, summed over the group."""
    out = torch.full((bt.N, bt.Hkv, keep), -1, dtype=torch.int32)
    q, bounds, G = q.cpu().double(), bounds.cpu().double(), bt.Hq // bt.Hkv
    for r, b, pos in bt.tokens():
        last = pos // bt.page
        rows = bounds[bt.table[b, :last + 1].long()]  # [pages, Hkv, 2, D]
        for h in range(bt.Hkv):
            qs = q[r, h * G:(h + 1) * G]
            s = torch.maximum(qs[None] * rows[:, h, None, 0], qs[None] * rows[:, h, None, 1]).sum((1, 2))
            s[s.isnan()] = -math.inf
            s[:first] = math.inf
            s[max(0, last + 1 - recent):] = math.inf
            got = s.sort(descending=True, stable=True).indices[:keep].sort().values
            out[r, h, :got.numel()] = got.int()
    return out
