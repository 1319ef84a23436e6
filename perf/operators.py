"""The paged-cache operators and the work they are timed on.

Four operators serve packed batches of sequences whose keys and values live in
pages: ``append`` (q/k norm, position rotation and the write of k/v into the
pages, with the per-page key bounds), ``attend`` (causal attention of the new
tokens over the pages, from one token a sequence to whole prompts), ``select``
(the pages a cheap score keeps for each new token) and ``sparse`` (attention
over the kept pages only).

A batch of B sequences has ``new`` tokens each, packed one after the other
(``cu_q`` [B + 1] holds the starts); ``seq_lens`` [B] counts all keys, the new
ones included, so token i of a sequence with n new ones is at position
``seq_len - n + i``. ``table`` [B, W] holds the page of every ``page`` positions.

``run`` computes an operator in elementary torch operations, or calls the
framework's (``own``).
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _case(name, op, dtype, heads, kv, dim, page, batch, ctx, new, keep=0, first=0, recent=0):
    c = {"op": op, "dtype": dtype, "heads": heads, "kv": kv, "dim": dim, "page": page, "batch": batch,
         "ctx_lo": ctx[0], "ctx_hi": ctx[1], "new_lo": new[0], "new_hi": new[1]}
    if op in ("select", "sparse"):
        c.update(keep=keep, first=first, recent=recent)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # One user's next token: the smallest call, all latency.
        _case("append_token", "append", "bf16", 32, 8, 128, 64, 1, (1000, 1000), (1, 1)),
        # A full decode batch in half precision with small pages and 64-wide heads.
        _case("append_batch_fp16", "append", "fp16", 16, 2, 64, 16, 128, (17, 1501), (1, 1)),
        # Ragged prompts arriving together: the append of a prefill step.
        _case("append_prompts", "append", "bf16", 32, 8, 128, 64, 7, (0, 250), (301, 2501)),
        # One user's next token over a short conversation: latency of attention.
        _case("attend_token", "attend", "bf16", 32, 8, 128, 64, 1, (2047, 2047), (1, 1)),
        # A decode batch of long, ragged conversations: the cache read is all of it.
        _case("attend_batch", "attend", "bf16", 32, 8, 128, 64, 32, (1000, 32000), (1, 1)),
        # Drafted tokens being verified: a few rows a sequence, half precision.
        _case("attend_drafts_fp16", "attend", "fp16", 16, 2, 64, 32, 24, (500, 9000), (2, 5)),
        # Chunks of prompts in progress over their cached parts.
        _case("attend_chunks", "attend", "bf16", 32, 8, 128, 16, 4, (3000, 12000), (200, 600)),
        # Whole prompts: bound by the matrix products.
        _case("attend_prompts", "attend", "bf16", 32, 8, 128, 128, 2, (0, 64), (5003, 8003)),
        # Pages kept for every sequence of a long decode batch.
        _case("select_batch", "select", "bf16", 32, 8, 128, 64, 32, (1000, 32000), (1, 1), 32, 1, 2),
        # Pages kept for every token of two prompt chunks.
        _case("select_chunks", "select", "bf16", 32, 8, 128, 64, 2, (6000, 15000), (700, 1100), 16, 1, 2),
        # Attention of the decode batch over its kept pages.
        _case("sparse_batch", "sparse", "bf16", 32, 8, 128, 64, 32, (1000, 32000), (1, 1), 32, 1, 2),
        # Attention of the prompt chunks over every token's own kept pages.
        _case("sparse_chunks", "sparse", "bf16", 32, 8, 128, 64, 2, (6000, 15000), (700, 1100), 16, 1, 2),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = {}
    for c in listed():
        w, m = work(c), most.setdefault(c["op"], [0, 0, 0])
        most[c["op"]] = [max(m[0], w["bytes"]), max(m[1], w["flops"]), max(m[2], _plain_values(c))]
    while True:
        op = rng.choice(["append", "attend", "select", "sparse"])
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 2, 3, 4, 5, 8])
        batch = _log(rng, 1, 64)
        if rng.random() < 0.5:
            new = (1, rng.choice([1, 1, 4]))
        else:
            n = _log(rng, 2, 4000)
            new = (max(1, n // rng.randint(1, 5)), n)
        ctx = sorted(_log(rng, 1, 30000) - 1 for _ in range(2))
        page = rng.choice([16, 32, 64, 128])
        first, recent = rng.randint(0, 2), rng.randint(1, 3)
        c = _case("", op, rng.choice(["bf16", "bf16", "fp16"]), heads, kv, rng.choice([64, 128, 128]), page, batch,
                  ctx, new, first + recent + _log(rng, 1, 60), first, recent)
        w, m = work(c), most[op]
        if w["bytes"] <= m[0] and w["flops"] <= m[1] and _plain_values(c) <= m[2]:
            return c


def _plain_values(c):
    """The size of the plain form's largest intermediate."""
    ctx, new = _lengths(c)
    n, longest = max(new), max(a + b for a, b in zip(ctx, new))
    if c["op"] == "attend":
        return c["batch"] * (c["heads"] * n * longest + 2 * c["kv"] * longest * c["dim"])
    if c["op"] == "select":
        return c["batch"] * c["kv"] * n * math.ceil(longest / c["page"])
    if c["op"] == "sparse":
        return sum(new) * c["kv"] * c["keep"] * c["page"] * c["dim"]
    return sum(new) * (c["heads"] + 2 * c["kv"]) * c["dim"]


def _lengths(c):
    """Keys already cached and new tokens of every sequence, spread over the case's ranges."""
    steps = [(b * 37 + 11) % 101 for b in range(c["batch"])]
    ctx = [c["ctx_lo"] + (c["ctx_hi"] - c["ctx_lo"]) * s // 100 for s in steps]
    new = [c["new_lo"] + (c["new_hi"] - c["new_lo"]) * ((s * 13) % 101) // 100 for s in steps]
    return ctx, new


def work(c):
    ctx, new = _lengths(c)
    n, H, K, D, page = sum(new), c["heads"], c["kv"], c["dim"], c["page"]
    lens = [a + b for a, b in zip(ctx, new)]
    blocks = [-(-t // page) for t in lens]
    index = 4 * (sum(blocks) + 2 * c["batch"] + 1)
    if c["op"] == "append":
        touched = sum((t - 1) // page - a // page + 1 for t, a in zip(lens, ctx))
        begun = sum(a % page > 0 for a in ctx)
        rows = 2 * n * (H + 2 * K) * D  # 16-bit values read, and written
        return {"bytes": 2 * rows + 2 * n * 2 * D + 2 * K * 2 * D * (touched + begun) + index,
                "flops": n * (H + K) * D * 7}
    if c["op"] == "attend":
        pairs = sum(b * a + b * (b + 1) // 2 for a, b in zip(ctx, new))
        return {"bytes": 2 * (2 * n * H * D + 2 * sum(lens) * K * D) + index, "flops": 4 * D * H * pairs}
    if c["op"] == "select":
        scored = sum((a + i) // page + 1 for a, b in zip(ctx, new) for i in range(b))
        return {"bytes": 2 * (n * H * D + sum(blocks) * K * 2 * D) + 4 * n * K * c["keep"] + index,
                "flops": 4 * D * K * scored + 2 * n * H * D}
    seen = sum(min(c["keep"], (a + i) // page + 1) for a, b in zip(ctx, new) for i in range(b))
    read = sum(min(t, page * sum(min(c["keep"], (a + i) // page + 1) for i in range(b)))
               for t, a, b in zip(lens, ctx, new))
    return {"bytes": 2 * (2 * n * H * D + 2 * K * read * D) + 4 * n * K * c["keep"] + index,
            "flops": 4 * D * H * seen * page}


def prepare(case, seed):
    c, dev = case, torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dtype, H, K, D, page, B = _DTYPES[c["dtype"]], c["heads"], c["kv"], c["dim"], c["page"], c["batch"]
    ctx, new = _lengths(c)
    lens = [a + b for a, b in zip(ctx, new)]
    N, width = sum(new), max(-(-t // page) for t in lens)
    total = B * width + 3

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device=dev, dtype=dtype if math.prod(shape) > 1 << 26
                            else torch.float32) * std).to(dtype)

    s = dict(c, max_q=max(new), max_len=max(lens), N=N)
    # Pages are handed out in the order in which requests came and went.
    s["table"] = torch.randperm(total, generator=g, device=dev)[: B * width].view(B, width).int()
    s["cu_q"] = torch.tensor([sum(new[:b]) for b in range(B + 1)], dtype=torch.int32, device=dev)
    s["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    # Keys of one page resemble one another: a shared part and each key's own.
    if c["op"] != "select":
        s["k_pages"], s["v_pages"] = normal(total, K, page, D), normal(total, K, page, D)
        s["k_pages"] += normal(total, K, 1, D, std=0.5)
    if c["op"] == "append":
        s["qkv"] = normal(N, H + 2 * K, D, std=3.0)
        s["q_weight"], s["k_weight"] = 1 + normal(D, std=0.1), 1 + normal(D, std=0.1)
        angle = torch.outer(torch.arange(s["max_len"], device=dev, dtype=torch.float64),
                            1e6 ** (-torch.arange(0, D, 2, device=dev, dtype=torch.float64) / D)).repeat(1, 2)
        s["cos"], s["sin"] = angle.cos().to(dtype), angle.sin().to(dtype)
        # Bounds of what the pages hold so far.
        s["bounds"] = torch.zeros(total, K, 2, D, dtype=dtype, device=dev)
        have = torch.tensor(ctx, device=dev)
        held = (have.view(B, 1) - torch.arange(width, device=dev) * page).clamp(0, page).view(-1, 1, 1, 1)
        pages = s["table"].flatten().long()
        inside = torch.arange(page, device=dev).view(1, 1, page, 1) < held
        keys = s["k_pages"][pages]
        s["bounds"][pages, :, 0] = keys.masked_fill(~inside, math.inf).amin(2)
        s["bounds"][pages, :, 1] = keys.masked_fill(~inside, -math.inf).amax(2)
        s["q_out"] = torch.zeros(N, H, D, dtype=dtype, device=dev)
        return s
    s["q"] = normal(N, H, D, std=2.0)
    if c["op"] == "select":
        low, high = normal(total, K, D), normal(total, K, D)
        s["bounds"] = torch.stack([torch.minimum(low, high) - 1, torch.maximum(low, high) + 1], 2)
    if c["op"] == "sparse":
        # Every token's pages: the first ones, the last ones and some between, ascending.
        row, pos = _places(s)
        at = pos // page
        every = torch.arange(width, device=dev)
        value = torch.rand(N, K, width, generator=g, device=dev)
        value += 2.0 * ((every < c["first"]) | (every > at.view(N, 1, 1) - c["recent"]))
        s["blocks"] = _best(value, at, c["keep"])
    return s


def _places(s):
    """The sequence and the position of every packed token."""
    t = torch.arange(s["N"], device=s["cu_q"].device)
    row = torch.searchsorted(s["cu_q"][1:].contiguous(), t, right=True)
    return row, s["seq_lens"][row].long() - s["cu_q"][row + 1] + t


def _best(score, last, keep):
    """The ``keep`` best columns up to ``last`` of score [N, K, W], lower ones first where equal, ascending, -1 behind."""
    W = score.shape[-1]
    seen = torch.arange(W, device=score.device) <= last.view(-1, 1, 1)
    order = score.masked_fill(~seen | score.isnan(), -math.inf).sort(dim=-1, descending=True, stable=True).indices[..., :keep]
    order = order.masked_fill(order > last.view(-1, 1, 1), W).sort(-1).values
    out = torch.full((*score.shape[:2], keep), -1, dtype=torch.int32, device=score.device)
    out[..., : order.shape[-1]] = order.masked_fill(order == W, -1)
    return out


def run(state):
    s = state
    if own:
        from sparseattentioninfer_b200 import ops
        batch = (s["table"], s["cu_q"], s["seq_lens"])
        if s["op"] == "append":
            ops.paged_qk_norm_rope_append(
                s["qkv"], s["q_weight"], s["k_weight"], s["cos"], s["sin"], s["k_pages"], s["v_pages"], *batch,
                Hq=s["heads"], Hkv=s["kv"], eps=1e-6, k_bounds=s["bounds"], q_out=s["q_out"])
            return s["q_out"], s["k_pages"], s["v_pages"], s["bounds"]
        if s["op"] == "select":
            return ops.paged_block_select(s["q"], s["bounds"], *batch, page_size=s["page"], keep=s["keep"],
                                          first=s["first"], recent=s["recent"], max_q=s["max_q"])
        return ops.paged_attention(s["q"], s["k_pages"], s["v_pages"], *batch, max_q=s["max_q"],
                                   max_len=s["max_len"], blocks=s.get("blocks"))
    return {"append": _append, "attend": _attend, "select": _select, "sparse": _sparse}[s["op"]](s)


def _append(s):
    H, K, page = s["heads"], s["kv"], s["page"]
    row, pos = _places(s)
    x = s["qkv"][:, : H + K].float()
    x = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-6)
    x = torch.cat([x[:, :H] * s["q_weight"].float(), x[:, H:] * s["k_weight"].float()], 1)
    left, right = x.chunk(2, -1)
    x = x * s["cos"][pos].float()[:, None] + torch.cat([-right, left], -1) * s["sin"][pos].float()[:, None]
    s["q_out"].copy_(x[:, :H])
    to, slot = s["table"][row, pos // page].long(), pos % page
    s["k_pages"][to, :, slot] = x[:, H:].to(s["k_pages"].dtype)
    s["v_pages"][to, :, slot] = s["qkv"][:, H + K:]
    # Bounds of the pages that got keys, over all that these hold now.
    lens = s["seq_lens"].long()
    at = torch.arange(s["table"].shape[1], device=row.device) * page
    got = (at < lens[:, None]) & (at + page > (lens - s["cu_q"].diff())[:, None])
    held = (lens[:, None] - at)[got].view(-1, 1, 1, 1)
    pages = s["table"][got].long()
    keys = s["k_pages"][pages]
    inside = torch.arange(page, device=row.device).view(1, 1, page, 1) < held
    s["bounds"][pages, :, 0] = keys.masked_fill(~inside, math.inf).amin(2)
    s["bounds"][pages, :, 1] = keys.masked_fill(~inside, -math.inf).amax(2)
    return s["q_out"], s["k_pages"], s["v_pages"], s["bounds"]


def _softmax(x):
    x = torch.exp(x - x.amax(-1, keepdim=True).clamp_min(torch.finfo(x.dtype).min))
    return x / x.sum(-1, keepdim=True).clamp_min(torch.finfo(x.dtype).tiny)


def _spread(s, t):
    """Packed rows [N, ...] as [B, max_q, ...], and where they are."""
    count = s["cu_q"].diff()
    i = torch.arange(s["max_q"], device=t.device)
    there = i < count[:, None]
    return t[(s["cu_q"][:-1, None] + i).clamp_max(s["N"] - 1).long()], there


def _attend(s):
    B, G, K, D, page, L = s["batch"], s["heads"] // s["kv"], s["kv"], s["dim"], s["page"], s["max_len"]
    q, there = _spread(s, s["q"])
    M = s["max_q"]
    pages = s["table"][:, : -(-L // page)].long()
    inside = torch.arange(pages.shape[1] * page, device=q.device) < s["seq_lens"][:, None]
    k = s["k_pages"][pages].transpose(1, 2).reshape(B, K, -1, D).float()
    v = s["v_pages"][pages].transpose(1, 2).reshape(B, K, -1, D).float().masked_fill(~inside[:, None, :, None], 0)
    x = q.float().view(B, M, K, G, D).permute(0, 2, 1, 3, 4).reshape(B, K, M * G, D) @ k.transpose(-1, -2)
    x *= 1 / math.sqrt(D)
    at = s["seq_lens"][:, None] - s["cu_q"].diff()[:, None] + torch.arange(M, device=q.device)
    past = torch.arange(k.shape[2], device=q.device) > at.repeat_interleave(G, 1)[..., None]
    o = _softmax(x.masked_fill_(past[:, None], -math.inf)) @ v
    return o.view(B, K, M, G, D).transpose(1, 2).reshape(B, M, K * G, D)[there].to(s["q"].dtype)


def _select(s):
    B, G, K, D, page, M = s["batch"], s["heads"] // s["kv"], s["kv"], s["dim"], s["page"], s["max_q"]
    # In 64 bits: which pages are kept goes by the order of near values.
    q = s["q"].double().view(-1, K, G, D)
    q = torch.cat([q.clamp_max(0).sum(2), q.clamp_min(0).sum(2)], -1)
    q, there = _spread(s, q)
    bounds = s["bounds"].flatten(2)[s["table"].long()].double()
    score = (q.transpose(1, 2) @ bounds.permute(0, 2, 3, 1)).transpose(1, 2)[there]
    row, pos = _places(s)
    at, every = pos // page, torch.arange(score.shape[-1], device=q.device)
    forced = (every < s["first"]) | (every > at.view(-1, 1, 1) - s["recent"])
    return _best(score.masked_fill(forced, math.inf), at, s["keep"])


def _sparse(s):
    N, G, K, D, page = s["N"], s["heads"] // s["kv"], s["kv"], s["dim"], s["page"]
    row, pos = _places(s)
    blocks = s["blocks"].long()
    pages = s["table"][row[:, None, None], blocks.clamp_min(0)].long()
    head = torch.arange(K, device=row.device)[:, None]
    at = blocks[..., None] * page + torch.arange(page, device=row.device)
    hidden = ((blocks < 0)[..., None] | (at > pos.view(N, 1, 1, 1))).flatten(2)
    k = s["k_pages"][pages, head].float().flatten(2, 3)
    x = s["q"].float().view(N, K, G, D) @ k.transpose(-1, -2) * (1 / math.sqrt(D))
    x = _softmax(x.masked_fill(hidden[:, :, None], -math.inf))
    v = s["v_pages"][pages, head].float().flatten(2, 3).masked_fill(hidden[..., None], 0)
    return (x @ v).view(N, K * G, D).to(s["q"].dtype)


def exact(case, seed):
    s = prepare(case, seed)
    ctx, new = _lengths(case)
    D, G, page = s["dim"], s["heads"] // s["kv"], s["page"]
    if s["op"] == "select":
        return None
    if s["op"] == "append":
        q, bounds = torch.zeros_like(s["q_out"], dtype=torch.float64), s["bounds"].double()
        k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
    else:
        out = torch.zeros_like(s["q"], dtype=torch.float64)
    start = 0
    for b, (a, n) in enumerate(zip(ctx, new)):
        here, keys = slice(start, start + n), torch.arange(a + n, device=s["table"].device)
        start += n
        pages, slots = s["table"][b].long()[keys // page], keys % page
        if s["op"] == "append":
            x = s["qkv"][here].double()
            turn = torch.complex(s["cos"][a: a + n, : D // 2].double(), s["sin"][a: a + n, : D // 2].double())[:, None]

            def placed(x, weight):
                x = x * weight.double() / torch.sqrt((x * x).sum(-1, keepdim=True) / D + 1e-6)
                x = torch.complex(x[..., : D // 2].contiguous(), x[..., D // 2:].contiguous()) * turn
                return torch.cat([x.real, x.imag], -1)

            q[here] = placed(x[:, : s["heads"]], s["q_weight"])
            k_pages[pages[a:], :, slots[a:]] = placed(x[:, s["heads"]: s["heads"] + s["kv"]], s["k_weight"])
            v_pages[pages[a:], :, slots[a:]] = x[:, s["heads"] + s["kv"]:]
            for p in range(a // page, (a + n - 1) // page + 1):
                to = int(s["table"][b, p])
                held = k_pages[to, :, : min(page, a + n - p * page)]
                bounds[to] = torch.stack([held.amin(1), held.amax(1)], 1)
            continue
        k, v = (s[x][pages, :, slots].double() for x in ("k_pages", "v_pages"))  # [keys, kv, D]
        q = s["q"][here].double()
        for h in range(s["heads"]):
            for i in range(0, n, 2048):
                x = q[i: i + 2048, h] @ k[:, h // G].T / math.sqrt(D)
                pos = a + i + torch.arange(x.shape[0], device=x.device)[:, None]
                seen = keys <= pos
                if s["op"] == "sparse":
                    kept = torch.zeros(x.shape[0], s["table"].shape[1] + 1, dtype=torch.bool, device=x.device)
                    kept.scatter_(1, s["blocks"][here][i: i + 2048, h // G].long() % kept.shape[1], True)
                    seen &= kept[:, keys // page]
                out[here][i: i + 2048, h] = x.masked_fill(~seen, -math.inf).softmax(-1) @ v[:, h // G]
    return (q, k_pages, v_pages, bounds) if s["op"] == "append" else out
