"""The operators of a paged key and value cache, as cases that can be timed and compared.

A case is one pass through one of three operators: "append" (new keys and values rotated to their positions and put into
their pages, queries rotated beside them), "paged" (attention of the new tokens over their sequences' pages) and "prefix"
(the same for a batch whose sequences all continue one long prefix). A batch is packed: the tokens of a sequence follow one
another, and sequences differ in length.

With `own` false a pass is plain torch in 32 bits; with it true, the calls of `limn_b200.paged`.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

TORCH = {"float16": torch.float16, "bfloat16": torch.bfloat16}


def _case(op, dtype, batch, heads, kv_heads, hd, page_size, new, context, *, pages="token", prefix=0, rotated=None,
          pairing="halves", first=0):
    """`new`, `context`: shortest and longest number of new tokens and of earlier ones over the batch. `pages`: whether a
    page holds its tokens one after the other ("token": page, slot, head) or its heads ("head": page, head, slot).
    `prefix`: shared keys in front of every sequence. `rotated`: columns that turn with the position; `first`: the
    position of a sequence's first slot."""
    return {"op": op, "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads, "hd": hd, "page_size": page_size,
            "new_low": new[0], "new_high": new[1], "context_low": context[0], "context_high": context[1], "pages": pages,
            "prefix": prefix, "rotated": hd if rotated is None else rotated, "pairing": pairing, "first": first}


def listed() -> list[dict]:
    named = {
        # generation for a single user: one token enters the cache of every layer
        "append_one_token": _case("append", "bfloat16", 1, 32, 8, 128, 16, (1, 1), (1999, 1999)),
        # a captured step of a batch in which some sequences check drafted tokens; partly rotated heads of an odd width
        "append_drafts": _case("append", "float16", 200, 12, 12, 80, 48, (1, 5), (0, 3000), pages="head", rotated=32, pairing="neighbours"),
        # prompts of a batch enter the cache
        "append_prompts": _case("append", "bfloat16", 12, 32, 8, 128, 64, (100, 4000), (0, 500)),
        # generation for a single user, small heads, short cache
        "decode_one": _case("paged", "bfloat16", 1, 8, 8, 64, 16, (1, 1), (1998, 1998)),
        # batched generation, sequences of very different age, grouped heads
        "decode_batch": _case("paged", "bfloat16", 64, 32, 8, 128, 16, (1, 1), (500, 8191)),
        # generation over two very long documents
        "decode_long": _case("paged", "bfloat16", 2, 32, 8, 128, 64, (1, 1), (100000, 131071), pages="head"),
        # drafted tokens checked at once, one key head to every query head, pages of an odd size
        "decode_drafts": _case("paged", "float16", 24, 12, 12, 80, 48, (1, 5), (0, 3000), pages="head"),
        # pieces of prompts behind what is cached already, single tokens of other sequences among them
        "prompt_pieces": _case("paged", "bfloat16", 8, 32, 8, 128, 16, (1, 1000), (0, 7000)),
        # a whole long prompt
        "prompt_8k": _case("paged", "bfloat16", 1, 32, 8, 128, 64, (8192, 8192), (0, 0)),
        # a few answers to one short instruction
        "prefix_few": _case("prefix", "float16", 4, 8, 8, 64, 16, (1, 1), (0, 60), prefix=1000),
        # a batch of requests behind one long instruction, a token each
        "prefix_batch": _case("prefix", "bfloat16", 64, 32, 8, 128, 16, (1, 1), (15, 511), prefix=8192),
        # questions about one document, read in at once
        "prefix_questions": _case("prefix", "bfloat16", 16, 32, 4, 128, 64, (20, 150), (0, 0), prefix=4113, pages="head"),
    }
    return [{"name": name, **case} for name, case in named.items()]


def _spread(low, high, n, turn) -> list[int]:
    """n whole numbers from low to high, in no order, the same every time; one alone is the highest."""
    if n == 1:
        return [high]
    at = [((i + 1) * turn) % 1.0 for i in range(n)]
    top, bottom = max(at), min(at)
    return [low + int(round((high - low) * (x - bottom) / (top - bottom))) for x in at]


def _lengths(case):
    """New tokens and keys in the own pages (new ones among them), by sequence."""
    new = _spread(case["new_low"], case["new_high"], case["batch"], 0.6180339887)
    context = _spread(case["context_low"], case["context_high"], case["batch"], 0.7548776662)
    return new, [c + n for c, n in zip(context, new)]


def _seen(case) -> int:
    """(token, key) pairs that the batch attends to."""
    new, keys = _lengths(case)
    return sum(n * (k - n) + n * (n + 1) // 2 + n * case["prefix"] for n, k in zip(new, keys))


def work(case):
    e, (new, keys) = 2, _lengths(case)
    tokens, h, hk, hd = sum(new), case["heads"], case["kv_heads"], case["hd"]
    tables = 4 * sum(-(-k // case["page_size"]) for k in keys) + 8 * case["batch"]
    if case["op"] == "append":
        return {"bytes": 2.0 * tokens * (h + 2 * hk) * hd * e + tables + 4 * case["rotated"],
                "flops": 3.0 * tokens * (h + hk) * case["rotated"]}
    kv = 2.0 * hk * hd * e * (sum(keys) + case["prefix"])
    return {"bytes": kv + 2.0 * tokens * h * hd * e + 4 * tokens * h + tables, "flops": 4.0 * h * hd * _seen(case)}


_MOST_FLOPS, _MOST_BYTES = 5.0e11, 1.1e9  # below the largest listed prompt's, the largest listed generation step's
_MOST_SCORES = 2**31  # of the plain form, which pads


def draw(rng) -> dict:
    def between(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    while True:
        op = rng.choice(["append", "paged", "paged", "paged", "prefix", "prefix"])
        kv_heads = rng.choice([1, 2, 4, 5, 8, 12])
        heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 4, 7, 8, 16])
        hd = rng.choice([32, 64, 64, 80, 96, 128, 128, 128])
        page_size = rng.choice([8, 16, 16, 24, 32, 48, 64, 128, 256])
        batch = between(1, 256)
        kind = rng.choice(["token", "token", "drafts", "pieces", "prompts"])
        high = {"token": 1, "drafts": rng.randint(2, 8), "pieces": between(16, 2000), "prompts": between(16, 8000)}[kind]
        new = (1 if kind != "prompts" else between(1, high), high)
        low = 0 if kind == "prompts" else between(1, 4000) - 1
        context = (low, low if kind == "prompts" else between(low + 1, 100000))
        case = _case(op, rng.choice(["bfloat16", "bfloat16", "float16"]), batch, heads, kv_heads, hd, page_size, new, context,
                     pages=rng.choice(["token", "head"]), prefix=between(64, 30000) if op == "prefix" else 0,
                     rotated=rng.choice([hd, hd, 32, 16]), pairing=rng.choice(["halves", "neighbours"]),
                     first=rng.choice([0, 0, between(1, 1000000)]))
        amount, (_, keys) = work(case), _lengths(case)
        scores = batch * heads * high * (max(keys) + case["prefix"])
        padded = batch * max(keys) * kv_heads * hd
        if amount["flops"] <= _MOST_FLOPS and amount["bytes"] <= _MOST_BYTES and scores <= _MOST_SCORES and padded <= 2**30:
            return case


def _pages_like(case, shape, gen, device):
    """A tensor of pages, seen as (page, slot, head, column) whatever its order in memory."""
    pages, size, heads, width = shape
    in_memory = shape if case["pages"] == "token" else (pages, heads, size, width)
    held = torch.randn(in_memory, generator=gen, device=device, dtype=TORCH[case["dtype"]])  # empty slots hold what earlier sequences left
    return held if case["pages"] == "token" else held.transpose(1, 2)


def prepare(case, seed):
    """What a serving loop has in hand: the cache's pages, the step's page table, offsets and lengths, and the projections'
    output (append) or the rotated queries (attention), with room for the results."""
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(int(seed))
    dtype = TORCH[case["dtype"]]
    h, hk, hd, size, batch, prefix = (case[k] for k in ("heads", "kv_heads", "hd", "page_size", "batch", "prefix"))
    new, keys = _lengths(case)
    tokens, max_pages, prefix_pages = sum(new), max(1, -(-max(keys) // size)), -(-prefix // size)
    used = [-(-k // size) for k in keys]
    pages = sum(used) + prefix_pages + 3
    s = {"case": case, "tokens": tokens, "max_new": max(new), "max_keys": max(keys), "max_pages": max_pages, "pages": pages}
    s["k_cache"] = _pages_like(case, (pages, size, hk, hd), gen, device)
    s["v_cache"] = _pages_like(case, (pages, size, hk, hd), gen, device)
    free = torch.randperm(pages, generator=gen, device=device).to(torch.int32)
    s["prefix_table"] = free[:prefix_pages].contiguous()
    first = np.cumsum([prefix_pages] + used)
    at = np.zeros((batch, max_pages), dtype=np.int64)  # places past a sequence's pages repeat its table's first entry
    for b in range(batch):
        at[b] = first[b]
        at[b, : used[b]] = np.arange(first[b], first[b] + used[b])
    s["page_table"] = free[torch.from_numpy(np.minimum(at, pages - 1)).to(device)].contiguous()
    s["q_start"] = torch.tensor([0, *np.cumsum(new)], dtype=torch.int32, device=device)
    s["kv_lens"] = torch.tensor(keys, dtype=torch.int32, device=device)
    if case["op"] == "append":
        projected = torch.randn((tokens, (h + 2 * hk) * hd), generator=gen, device=device, dtype=dtype)
        s["q"] = projected[:, : h * hd].unflatten(1, (h, hd))
        s["k"] = projected[:, h * hd : (h + hk) * hd].unflatten(1, (hk, hd))
        s["v"] = projected[:, (h + hk) * hd :].unflatten(1, (hk, hd))
        s["q_out"] = torch.empty((tokens, h, hd), device=device, dtype=dtype)
        pairs = case["rotated"] // 2
        s["frequencies"] = 10000.0 ** (-torch.arange(pairs, dtype=torch.float64, device=device) / pairs)
    else:
        s["q"] = torch.randn((tokens, h, hd), generator=gen, device=device, dtype=dtype)
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty((tokens, h), device=device, dtype=torch.float32)
    if own:  # the handles that the loop keeps for its cache and its batch
        from limn_b200.paged import PagedBatch, PagedCache

        k, v = s["k_cache"], s["v_cache"]
        order = (0, 2, 1)  # page, head, slot
        cache = PagedCache(k, v, dtype=case["dtype"], pages=pages, page_size=size, kv_heads=hk, hd=hd,
                           k_strides=[k.stride(i) for i in order], v_strides=[v.stride(i) for i in order])
        s["step"] = PagedBatch(cache, heads=h, batch=batch, tokens=tokens, max_t_q=max(new), page_table=s["page_table"],
                               max_pages=max_pages, q_start=s["q_start"], kv_lens=s["kv_lens"],
                               first_position=case["first"] + prefix)
    return s


def run(s):
    op = s["case"]["op"]
    if op == "append":
        return _append(s)
    return _attention(s)


def _append(s):
    case = s["case"]
    if own:
        row = s["q"].stride(0)
        s["step"].append(s["k"], s["v"], q=s["q"], q_out=s["q_out"], q_strides=(row, case["hd"]), k_strides=(row, case["hd"]),
                         v_strides=(row, case["hd"]), frequencies=s["frequencies"], rotated=case["rotated"],
                         pairing=case["pairing"], stream=torch.cuda.current_stream().cuda_stream)
        return s["q_out"], s["k_cache"], s["v_cache"]
    sequence, slot = _places(s)
    page = s["page_table"][sequence, slot // case["page_size"]].long()
    within = slot % case["page_size"]
    turns = (slot + case["first"] + case["prefix"]).double()[:, None] * s["frequencies"]
    cos, sin = turns.cos().float()[:, None], turns.sin().float()[:, None]
    s["q_out"].copy_(_rotated(s["q"], cos, sin, case))
    s["k_cache"][page, within] = _rotated(s["k"], cos, sin, case)
    s["v_cache"][page, within] = s["v"]
    return s["q_out"], s["k_cache"], s["v_cache"]


def _places(s):
    """Sequence of every token, and its slot there."""
    token = torch.arange(s["tokens"], device=s["q_start"].device)
    sequence = torch.searchsorted(s["q_start"], token, right=True) - 1
    return sequence, s["kv_lens"][sequence].long() - s["q_start"][sequence + 1] + token


def _rotated(x, cos, sin, case):
    r = case["rotated"]
    wide = x.float()
    if case["pairing"] == "halves":
        a, b = wide[..., : r // 2], wide[..., r // 2 : r]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = wide[..., 0:r:2], wide[..., 1:r:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([turned, wide[..., r:]], -1).to(x.dtype)


def _attention(s):
    case = s["case"]
    h, hk, hd, batch = case["heads"], case["kv_heads"], case["hd"], case["batch"]
    scale = hd**-0.5
    if own:
        stream = torch.cuda.current_stream().cuda_stream
        if case["prefix"]:
            s["step"].attention_with_prefix(s["q"], s["out"], s["lse"], prefix_table=s["prefix_table"], prefix_len=case["prefix"],
                                            causal=True, scale=scale, stream=stream)
        else:
            s["step"].attention(s["q"], s["out"], s["lse"], causal=True, scale=scale, stream=stream)
        return s["out"], s["lse"]
    group, new, longest = h // hk, s["max_new"], s["max_keys"]
    sequence, slot = _places(s)
    within = torch.arange(s["tokens"], device=slot.device) - s["q_start"][sequence]
    # queries padded to (sequence, key head, token and head of its group, column)
    q = torch.zeros((batch, new, h, hd), device=slot.device)
    q[sequence, within] = s["q"].float()
    q = q.view(batch, new, hk, group, hd).permute(0, 2, 1, 3, 4).reshape(batch, hk, new * group, hd)
    k = s["k_cache"][s["page_table"].long()].flatten(1, 2)[:, :longest].float().permute(0, 2, 3, 1)
    v = s["v_cache"][s["page_table"].long()].flatten(1, 2)[:, :longest].float().transpose(1, 2)
    scores = (q @ k).mul_(scale)
    last = s["kv_lens"].long()[:, None] - (s["q_start"][1:] - s["q_start"][:-1]).long()[:, None] + torch.arange(new, device=slot.device)
    key = torch.arange(longest, device=slot.device)
    hidden = (key > last[..., None]) | (key >= s["kv_lens"][:, None, None])
    scores.view(batch, hk, new, group, longest).masked_fill_(hidden[:, None, :, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    if case["prefix"]:
        pk = s["k_cache"][s["prefix_table"].long()].flatten(0, 1)[: case["prefix"]].float().permute(1, 2, 0)
        pv = s["v_cache"][s["prefix_table"].long()].flatten(0, 1)[: case["prefix"]].float().transpose(0, 1)
        in_front = (q @ pk).mul_(scale)
        top = torch.maximum(top, in_front.amax(-1, keepdim=True))
        in_front.sub_(top).exp_()
    scores.sub_(top).exp_()
    total = scores.sum(-1, keepdim=True)
    o = scores @ v
    if case["prefix"]:
        total += in_front.sum(-1, keepdim=True)
        o += in_front @ pv
    o = (o / total).view(batch, hk, new, group, hd).transpose(1, 2).reshape(batch, new, h, hd)
    lse = (top + total.log()).view(batch, hk, new, group).transpose(1, 2).reshape(batch, new, h)
    s["out"].copy_(o[sequence, within])
    s["lse"].copy_(lse[sequence, within])
    return s["out"], s["lse"]


def exact(case, seed):
    """From the definitions, in 64 bits, a sequence and a key head at a time."""
    s = prepare(case, seed)
    new, keys = _lengths(case)
    size, h, hk, hd, p = case["page_size"], case["heads"], case["kv_heads"], case["hd"], case["prefix"]
    group = h // hk
    start = np.cumsum([0] + new)
    table = s["page_table"].cpu().numpy()
    if case["op"] == "append":
        q_out, kc, vc = s["q"].double(), s["k_cache"].double(), s["v_cache"].double()
        r = case["rotated"]
        for b, (n, length) in enumerate(zip(new, keys)):
            here = slice(int(start[b]), int(start[b + 1]))
            slots = np.arange(length - n, length)
            position = torch.from_numpy(slots + case["first"] + p).to(q_out.device, torch.float64)
            turn = torch.polar(torch.ones((), dtype=torch.float64, device=q_out.device), torch.outer(position, s["frequencies"]))[:, None]
            where = (torch.from_numpy(table[b][slots // size].astype(np.int64)), torch.from_numpy(slots % size))

            def turned(x):
                x = x.double().clone()
                if case["pairing"] == "halves":
                    z = torch.complex(x[..., : r // 2], x[..., r // 2 : r]) * turn
                    x[..., :r] = torch.cat([z.real, z.imag], -1)
                else:
                    z = torch.view_as_complex(x[..., :r].unflatten(-1, (r // 2, 2)).contiguous()) * turn
                    x[..., :r] = torch.view_as_real(z).flatten(-2)
                return x

            q_out[here] = turned(s["q"][here])
            kc[where] = turned(s["k"][here])
            vc[where] = s["v"][here].double()
        return q_out, kc, vc
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    lse = torch.empty(out.shape[:2], dtype=torch.float64, device=out.device)
    in_front = s["prefix_table"].long()
    for b, (n, length) in enumerate(zip(new, keys)):
        of = torch.from_numpy(table[b][: -(-length // size)].astype(np.int64)).to(out.device)
        here = slice(int(start[b]), int(start[b + 1]))
        seen = torch.ones((n, p + length), dtype=torch.bool, device=out.device).tril(p + length - n)[:, None]
        for head in range(hk):
            of_group = slice(head * group, (head + 1) * group)
            k, v = (torch.cat([c[in_front, :, head].flatten(0, 1)[:p], c[of, :, head].flatten(0, 1)[:length]]).double()
                    for c in (s["k_cache"], s["v_cache"]))
            x = torch.einsum("tgd,kd->tgk", s["q"][here, of_group].double(), k) / math.sqrt(hd)
            x = x.where(seen, -math.inf)
            total = torch.logsumexp(x, -1)
            lse[here, of_group] = total
            out[here, of_group] = torch.einsum("tgk,kd->tgd", torch.exp(x - total[..., None]), v)
    return out, lse
