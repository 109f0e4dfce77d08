"""Workloads of the paged key-value cache: appending to it, attention of new tokens over it, and the same over the pages
that a cheap score selects.

A cache holds ``[pages, kv_heads, page_size, head_dim]`` keys and values; row ``i`` of ``block_table`` names the pages of a
sequence in order, ``lengths[i]`` how many of its positions are held.  Each case is a dict of plain values; ``prepare`` makes
the tensors that a decoding program has in hand, ``run`` is one pass.  With ``own`` false it computes the operators from
elementary torch operations in 32 bits (selection scores in 64, as they stand next to a border), with ``own`` true through
this package.  ``exact`` computes them from their definition in 64 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}

# the largest listed cases, in bytes of keys and values; drawn ones stay below
DECODE_BYTES = 2 * 131071 * 8 * 128 * 4
SPARSE_BYTES = 16 * 32768 * 8 * 128 * 4
APPEND_VALUES = 4096 * (32 + 2 * 8) * 128


def listed():
    return [
        # the next token of one sequence, heads of a LLaMA-7B-shaped layer: latency
        dict(name="append-one", kind="append", dtype="f16", batch=1, tokens=1, longest=500, heads=32, kv_heads=32, dim=128,
             page=64, rotary=128, interleaved=False, padded=0),
        # one decoding step of a serving batch
        dict(name="append-decode", kind="append", dtype="f16", batch=64, tokens=1, longest=500, heads=32, kv_heads=32, dim=128,
             page=64, rotary=128, interleaved=False, padded=0),
        # prompts of a serving batch, grouped heads, behind what earlier turns left in the cache
        dict(name="append-prompts", kind="append", dtype="bf16", batch=8, tokens=512, longest=2048, heads=32, kv_heads=8,
             dim=128, page=64, rotary=128, interleaved=False, padded=0),
        # ragged pieces of prompts in a batch that is padded, small pages, a part of each head rotated in pairs
        dict(name="append-odd", kind="append", dtype="f16", batch=5, tokens=201, longest=1003, heads=6, kv_heads=6, dim=80,
             page=16, rotary=48, interleaved=True, padded=37),
        # one token against one short sequence: latency
        dict(name="decode-one", kind="decode", dtype="f16", batch=1, longest=500, heads=32, kv_heads=32, dim=128, page=64),
        # a serving batch of uneven lengths, four query heads to a key head
        dict(name="decode-batch", kind="decode", dtype="bf16", batch=64, longest=4096, heads=32, kv_heads=8, dim=128, page=64),
        # two long documents: the work is along the cache
        dict(name="decode-long", kind="decode", dtype="f16", batch=2, longest=131071, heads=32, kv_heads=8, dim=128, page=128),
        # small pages, a head width that is no power of two, rows with nothing in them
        dict(name="decode-odd", kind="decode", dtype="f16", batch=37, longest=1003, heads=24, kv_heads=24, dim=80, page=16),
        # one token against the selected pages of one long sequence: latency
        dict(name="sparse-one", kind="sparse", dtype="f16", batch=1, longest=32768, heads=32, kv_heads=8, dim=128, page=64,
             count=32, queries=1),
        # a serving batch of long sequences, a sixteenth of each read
        dict(name="sparse-batch", kind="sparse", dtype="bf16", batch=16, longest=32768, heads=32, kv_heads=8, dim=128, page=64,
             count=32, queries=1),
        # a piece of a prompt against the cache of one sequence: every query has pages of its own
        dict(name="sparse-queries", kind="sparse", dtype="bf16", batch=1, longest=16384, heads=32, kv_heads=8, dim=128, page=64,
             count=16, queries=256),
        # small pages, few and narrow heads, uneven lengths, some shorter than what is selected
        dict(name="sparse-odd", kind="sparse", dtype="f16", batch=11, longest=4096, heads=12, kv_heads=4, dim=64, page=16,
             count=33, queries=1),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "decode", "decode", "sparse", "sparse"])
    while True:
        kv_heads = rng.choice([1, 2, 4, 6, 8, 12, 24, 32])
        heads = kv_heads * rng.choice([1, 1, 2, 4, 5, 8, 16])
        case = dict(kind=kind, dtype=rng.choice(["f16", "bf16"]), batch=_log_int(rng, 1, 64), heads=heads, kv_heads=kv_heads,
                    dim=rng.choice([32, 64, 80, 96, 128]), page=rng.choice([16, 32, 64, 128]))
        if heads > 64:
            continue
        if kind == "append":
            case.update(tokens=_log_int(rng, 1, 512), longest=_log_int(rng, 512, 4096), padded=rng.choice([0, 0, 5, 64]))
            case.update(rotary=rng.choice([case["dim"], case["dim"], case["dim"] // 2]), interleaved=rng.random() < 0.3)
            if (case["batch"] * case["tokens"] * (heads + 2 * kv_heads) * case["dim"] <= APPEND_VALUES
                    and case["batch"] * case["longest"] * kv_heads * case["dim"] <= 1 << 27):
                return case
            continue
        case.update(longest=_log_int(rng, 16, 131072) if kind == "decode" else _log_int(rng, 1024, 65536))
        size = case["batch"] * case["longest"] * kv_heads * case["dim"] * 4
        if kind == "decode":
            if size <= DECODE_BYTES:
                return case
            continue
        case.update(count=_log_int(rng, 2, 64), queries=rng.choice([1, 1, 1, _log_int(rng, 2, 256)]))
        rows = case["batch"] * case["queries"]
        if size > SPARSE_BYTES or rows > 256 or rows * _pages(case, case["longest"]) * kv_heads * case["dim"] > 1 << 26:
            continue
        if case["batch"] * case["queries"] * kv_heads * case["count"] * case["page"] * case["dim"] * 4 <= SPARSE_BYTES // 2:
            return case


def _lengths(case):
    """Positions held for each sequence, what is appended included: the longest, a few short ones, the rest in between."""
    rng = random.Random("%(batch)d %(longest)d %(heads)d %(page)d" % case)
    longest, batch = case["longest"], case["batch"]
    got = [longest] + [rng.randint(max(1, longest // 8), longest) for _ in range(batch - 1)]
    if batch >= 4:
        got[2] = 1
    if batch >= 5:
        got[3] = 0
    return got


def _new_tokens(case):
    """Tokens appended to each sequence: all of ``tokens`` for the first, then uneven, none where nothing is held."""
    rng = random.Random("%(batch)d %(tokens)d" % case)
    most = case["tokens"]
    got = [most] + [rng.randint(max(1, most // 2), most) for _ in range(case["batch"] - 1)]
    return [min(n, length) for n, length in zip(got, _lengths(case))]


def _query_lengths(case):
    """Positions that each query row sees: a sequence's last queries each see one position more."""
    return [max(0, n - case["queries"] + 1 + j) if n else 0 for n in _lengths(case) for j in range(case["queries"])]


def _pages(case, n):
    return (n + case["page"] - 1) // case["page"]


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype, batch, page = DTYPES[case["dtype"]], case["batch"], case["page"]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]

    def randn(*shape, std=1.0):
        return (torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float16) * std).to(dtype)

    lengths = _lengths(case)
    width = max(1, max(_pages(case, n) for n in lengths))
    used = sum(_pages(case, n) for n in lengths)
    total = used + 3  # some pages belong to nobody
    order = torch.randperm(total, generator=gen, device=DEVICE, dtype=torch.int32)[:used]
    # every sequence's pages in order, the rest of its row of the table empty
    counts = torch.tensor([_pages(case, n) for n in lengths], device=DEVICE)
    table = torch.zeros(batch, width, dtype=torch.int32, device=DEVICE)
    held_pages = torch.arange(width, device=DEVICE) < counts[:, None]
    table[held_pages] = order
    k_cache = randn(total, kv_heads, page, dim)
    k_cache += randn(total, kv_heads, 1, dim, std=0.5)  # keys of neighbouring positions resemble each other
    state = dict(case=case, k_cache=k_cache, v_cache=randn(total, kv_heads, page, dim))
    held = torch.tensor(lengths, device=DEVICE)

    def boxes():
        """The smallest and largest key of each page in each dimension, over the positions that are held."""
        fill = torch.zeros(total, dtype=torch.int64, device=DEVICE)
        fill[table[held_pages].long()] = (held[:, None] - torch.arange(width, device=DEVICE) * page).clamp(0, page)[held_pages]
        out = (torch.arange(page, device=DEVICE) >= fill[:, None])[:, None, :, None]
        lo = k_cache.masked_fill(out, math.inf).amin(2)
        hi = k_cache.masked_fill(out, -math.inf).amax(2)
        empty = (fill == 0)[:, None, None]
        return torch.stack([lo.masked_fill(empty, 0), hi.masked_fill(empty, 0)], 2).contiguous()

    if case["kind"] == "append":
        tokens = _new_tokens(case)
        rows = sum(tokens) + case["padded"]
        fused = randn(rows, (heads + 2 * kv_heads) * dim)  # a qkv projection's output
        state["q"] = fused[:, :heads * dim].view(rows, heads, dim)
        state["k"] = fused[:, heads * dim:(heads + kv_heads) * dim].view(rows, kv_heads, dim)
        state["v"] = fused[:, (heads + kv_heads) * dim:].view(rows, kv_heads, dim)
        state["cu_tokens"] = torch.tensor([0] + [sum(tokens[:i + 1]) for i in range(batch)], dtype=torch.int32, device=DEVICE)
        half = case["rotary"] // 2
        angle = (torch.arange(case["longest"], device=DEVICE, dtype=torch.float64)[:, None]
                 * 10000.0 ** (-torch.arange(half, device=DEVICE, dtype=torch.float64) / half))
        state["rope"] = (angle.cos().float(), angle.sin().float())
        state["boxes"] = boxes()
    else:
        queries = case.get("queries", 1)
        state["q"] = randn(batch * queries, heads, dim)
        if case["kind"] == "sparse":
            state["boxes"] = boxes()
            table = table.repeat_interleave(queries, 0)
            held = torch.tensor(_query_lengths(case), device=DEVICE)
    state["block_table"], state["lengths"] = table, held.int()
    return state


# --------------------------------------------------------------------------------------------- the plain forms

def _rotate(x, cos, sin, interleaved):
    """``x`` [rows, heads, dim] fp32 with its first 2 * cos.size(1) elements rotated in pairs."""
    half = cos.size(1)
    turn, rest = x[..., :2 * half], x[..., 2 * half:]
    cos, sin = cos[:, None], sin[:, None]
    if interleaved:
        a, b = turn[..., 0::2], turn[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = turn[..., :half], turn[..., half:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, rest], -1)


def _plain_append(state):
    q, k, v, cu = state["q"], state["k"], state["v"], state["cu_tokens"].long()
    k_cache, v_cache, boxes, table = state["k_cache"], state["v_cache"], state["boxes"], state["block_table"].long()
    lengths, page, (cos, sin) = state["lengths"].long(), state["case"]["page"], state["rope"]
    row = torch.arange(q.size(0), device=q.device)
    seq = torch.searchsorted(cu, row, right=True) - 1
    real = seq < lengths.numel()
    seq = seq.clamp(max=lengths.numel() - 1)
    at = lengths[seq] - (cu[seq + 1] - row)
    real &= at >= 0
    at = at.clamp(min=0)
    c, s, interleaved = cos[at], sin[at], state["case"]["interleaved"]
    q_out = (_rotate(q.float(), c, s, interleaved) * real[:, None, None]).to(q.dtype)
    live = real.nonzero().flatten()
    k_new = _rotate(k.float(), c, s, interleaved).to(k.dtype)[live]
    seq, at = seq[live], at[live]
    to = table[seq, at // page]
    k_cache[to, :, at % page] = k_new
    v_cache[to, :, at % page] = v[live]
    touched = torch.unique(seq * table.size(1) + at // page)
    seq, nth = touched // table.size(1), touched % table.size(1)
    to = table[seq, nth]
    out = (torch.arange(page, device=q.device) >= (lengths[seq] - nth * page)[:, None])[:, None, :, None]
    keys = k_cache[to].float()
    boxes[to] = torch.stack([keys.masked_fill(out, math.inf).amin(2), keys.masked_fill(out, -math.inf).amax(2)], 2).to(k.dtype)
    return q_out, k_cache, v_cache, boxes


def _softmax_product(q, k, v, seen):
    """``q`` [n, g, d] against ``k``, ``v`` [n, s, d] in fp32, over the positions that ``seen`` [n, s] marks; 0 where none is."""
    scores = torch.matmul(q.float(), k.float().transpose(1, 2)) * (1.0 / math.sqrt(q.size(-1)))
    scores = scores.masked_fill(~seen[:, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = (scores - top.masked_fill(top == -math.inf, 0)).exp()
    total = weights.sum(-1, keepdim=True)
    v = v.float().masked_fill(~seen[..., None], 0)
    return (torch.matmul(weights, v) / total.masked_fill(total == 0, 1)).to(q.dtype)


def _plain_decode(state):
    q, k_cache, v_cache = state["q"], state["k_cache"], state["v_cache"]
    table, lengths = state["block_table"].long(), state["lengths"].long()
    rows, heads, dim = q.shape
    kv_heads, span = k_cache.size(1), table.size(1) * k_cache.size(2)
    k = k_cache[table].transpose(1, 2).reshape(rows * kv_heads, span, dim)
    v = v_cache[table].transpose(1, 2).reshape(rows * kv_heads, span, dim)
    seen = torch.arange(span, device=q.device) < lengths[:, None]
    out = _softmax_product(q.reshape(rows * kv_heads, heads // kv_heads, dim), k, v, seen.repeat_interleave(kv_heads, 0))
    return out.reshape(rows, heads, dim)


def _plain_select(q, boxes, table, lengths, page, count):
    """The ``count`` pages of each row and key head whose box can give the largest scores, first and last page always."""
    rows, heads, dim = q.shape
    kv_heads = boxes.size(1)
    grouped = q.double().reshape(rows, kv_heads, heads // kv_heads, dim)
    up, down = grouped.clamp(min=0).sum(2), grouped.clamp(max=0).sum(2)
    box = boxes[table].double()  # [rows, width, kv_heads, 2, dim]
    scores = ((box[..., 1, :] * up[:, None]).sum(-1) + (box[..., 0, :] * down[:, None]).sum(-1)).transpose(1, 2)
    held = ((lengths + page - 1) // page)[:, None, None]
    nth = torch.arange(table.size(1), device=q.device)
    scores = scores.masked_fill((nth == 0) | (nth == held - 1), math.inf).masked_fill(nth >= held, -math.inf)
    chosen = scores.sort(dim=-1, descending=True, stable=True).indices[..., :count]
    chosen = chosen.masked_fill(chosen >= held, table.size(1)).sort(dim=-1).values
    chosen = torch.nn.functional.pad(chosen, (0, count - chosen.size(-1)), value=table.size(1))
    return chosen.masked_fill(chosen == table.size(1), -1)


def _plain_sparse(state):
    q, k_cache, v_cache, page = state["q"], state["k_cache"], state["v_cache"], state["case"]["page"]
    table, lengths = state["block_table"].long(), state["lengths"].long()
    rows, heads, dim = q.shape
    kv_heads, count = k_cache.size(1), state["case"]["count"]
    pages = _plain_select(q, state["boxes"], table, lengths, page, count)
    nth = pages.clamp(min=0)
    at = table[torch.arange(rows, device=q.device)[:, None, None], nth]
    head = torch.arange(kv_heads, device=q.device)[None, :, None]
    position = nth[..., None] * page + torch.arange(page, device=q.device)
    seen = (position < lengths[:, None, None, None]) & (pages >= 0)[..., None]
    n = rows * kv_heads
    out = _softmax_product(q.reshape(n, heads // kv_heads, dim), k_cache[at, head].reshape(n, count * page, dim),
                           v_cache[at, head].reshape(n, count * page, dim), seen.reshape(n, count * page))
    return out.reshape(rows, heads, dim), pages.int()


def run(state):
    case = state["case"]
    if own:
        from intrasm_engine_b200.pytorch import paged_attention as paged
        if case["kind"] == "append":
            q = paged.paged_append(state["q"], state["k"], state["v"], state["k_cache"], state["v_cache"], state["block_table"],
                                   state["lengths"], cu_tokens=state["cu_tokens"], rope=state["rope"],
                                   interleaved=case["interleaved"], boxes=state["boxes"])
            return q, state["k_cache"], state["v_cache"], state["boxes"]
        if case["kind"] == "decode":
            return paged.paged_attention(state["q"], state["k_cache"], state["v_cache"], state["block_table"], state["lengths"])
        pages = paged.paged_select(state["q"], state["boxes"], state["block_table"], state["lengths"], case["page"],
                                   case["count"], first=1, last=1)
        return paged.paged_attention(state["q"], state["k_cache"], state["v_cache"], state["block_table"], state["lengths"],
                                     pages=pages), pages
    return {"append": _plain_append, "decode": _plain_decode, "sparse": _plain_sparse}[case["kind"]](state)


# --------------------------------------------------------------------------------------------------- measures

def work(case):
    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    if case["kind"] == "append":
        tokens = sum(_new_tokens(case))
        # q, k, v in, q and the cache's rows out, the angles once; the boxes of the pages that are written
        touched = sum(_pages(case, n) - (n - new) // page for n, new in zip(_lengths(case), _new_tokens(case)) if new)
        return {"bytes": 2 * tokens * (2 * heads + 4 * kv_heads) * dim + tokens * case["rotary"] * 4 + touched * kv_heads * dim * 4,
                "flops": 3.0 * tokens * (heads + kv_heads) * case["rotary"]}
    if case["kind"] == "decode":
        held = sum(_lengths(case))
        return {"bytes": held * kv_heads * dim * 4 + case["batch"] * heads * dim * 4, "flops": 4.0 * held * heads * dim}
    seen = _query_lengths(case)
    read = sum(min(n, case["count"] * page) for n in seen)  # positions of a key head that some row attends to
    stored = min(read, sum(_lengths(case)))
    boxes = sum(_pages(case, n) for n in _lengths(case) if _pages(case, n) > case["count"])
    scored = sum(_pages(case, n) for n in seen if _pages(case, n) > case["count"])
    return {"bytes": (stored + boxes) * kv_heads * dim * 4 + len(seen) * (heads * dim * 4 + kv_heads * case["count"] * 4),
            "flops": 4.0 * read * heads * dim + 4.0 * scored * kv_heads * dim}


def _exact_rows(q, k, v):
    """Attention of ``q`` [g, d] over ``k``, ``v`` [s, d], in 64 bits."""
    if k.size(0) == 0:
        return torch.zeros_like(q)
    return torch.softmax((q @ k.T) / math.sqrt(q.size(-1)), -1) @ v


def exact(case, seed):
    state = prepare(case, seed)
    q, k_cache, v_cache, page = state["q"].double(), state["k_cache"], state["v_cache"], case["page"]
    table, lengths = state["block_table"].tolist(), state["lengths"].tolist()
    group = case["heads"] // case["kv_heads"]
    if case["kind"] == "append":
        cos, sin = (t.double() for t in state["rope"])
        half, q_out = cos.size(1), torch.zeros_like(q)
        k_out, v_out, box_out = k_cache.double(), v_cache.double(), state["boxes"].double()
        cu = state["cu_tokens"].tolist()

        def turn(x, at):
            z = x.double().clone()
            one, two = ((slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if case["interleaved"] else
                        (slice(0, half), slice(half, 2 * half)))
            z[..., one] = x[..., one].double() * cos[at][:, None] - x[..., two].double() * sin[at][:, None]
            z[..., two] = x[..., two].double() * cos[at][:, None] + x[..., one].double() * sin[at][:, None]
            return z

        for i, length in enumerate(lengths):
            new = cu[i + 1] - cu[i]
            if not new:
                continue
            rows, at = slice(cu[i], cu[i + 1]), torch.arange(length - new, length, device=DEVICE)
            q_out[rows] = turn(state["q"][rows], at)
            to = torch.tensor(table[i], device=DEVICE)[at // page]
            k_out[to, :, at % page] = turn(state["k"][rows], at)
            v_out[to, :, at % page] = state["v"][rows].double()
            for nth in range((length - new) // page, _pages(case, length)):
                keys = k_out[table[i][nth], :, :min(page, length - nth * page)]
                box_out[table[i][nth]] = torch.stack([keys.amin(1), keys.amax(1)], 1)
        return q_out, k_out, v_out, box_out
    out = torch.zeros_like(q)
    if case["kind"] == "decode":
        for i, length in enumerate(lengths):
            pages = torch.tensor(table[i][:_pages(case, length)], device=DEVICE, dtype=torch.long)
            for h in range(case["kv_heads"]):
                keys, values = (t[pages, h].reshape(-1, case["dim"])[:length].double() for t in (k_cache, v_cache))
                out[i, h * group:(h + 1) * group] = _exact_rows(q[i, h * group:(h + 1) * group], keys, values)
        return out
    count = case["count"]
    chosen = torch.full((len(lengths), case["kv_heads"], count), -1, dtype=torch.int32)
    slots = torch.arange(page, device=DEVICE)
    for i, length in enumerate(lengths):
        held = _pages(case, length)
        if not held:
            continue
        at = torch.tensor(table[i][:held], device=DEVICE, dtype=torch.long)
        lo, hi = state["boxes"][at].double().unbind(2)  # [held, kv_heads, dim]
        mine = q[i].reshape(1, case["kv_heads"], group, case["dim"])
        # what any key inside the box could give at most, over the query heads of a key head
        scores = torch.maximum(mine * lo[:, :, None], mine * hi[:, :, None]).sum((2, 3)).cpu()
        for h in range(case["kv_heads"]):
            rank = sorted(range(held), key=lambda p: (p not in (0, held - 1), -float(scores[p, h]), p))
            nth = torch.tensor(sorted(rank[:count]))
            chosen[i, h, :len(nth)] = nth.int()
            nth = nth.to(DEVICE)
            seen = ((nth[:, None] * page + slots) < length).flatten()
            keys, values = (t[at[nth], h].reshape(-1, case["dim"])[seen].double() for t in (k_cache, v_cache))
            out[i, h * group:(h + 1) * group] = _exact_rows(q[i, h * group:(h + 1) * group], keys, values)
    return out, chosen
