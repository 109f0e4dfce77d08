"""Definitions of the paged cache's operators in 64 bits, row by row, and random caches to run them on."""
import math

import torch

DEV = "cuda:0"
DTYPES = [torch.float16, torch.bfloat16]


def unit(dtype):
    """Half a step, relative to the value."""
    return torch.finfo(dtype).eps / 2


def make_cache(gen, lengths, kv_heads, dim, page, dtype, spare=2, dev=DEV, fill=float("nan")):
    """k, v, table: every sequence on pages of its own in random order; what no sequence holds is `fill`, as are entries of
    the table behind the pages that a row needs."""
    pages = [(n + page - 1) // page for n in lengths]
    total, width = sum(pages) + spare, max([1] + pages)
    order = torch.randperm(total, generator=gen)[:sum(pages)].to(torch.int32)
    k = torch.full((total, kv_heads, page, dim), fill, dtype=dtype)
    v = torch.full_like(k, fill)
    table = torch.full((len(lengths), width), 2 ** 30, dtype=torch.int32)
    at = 0
    for i, n in enumerate(lengths):
        mine = order[at:at + pages[i]]
        at += pages[i]
        table[i, :pages[i]] = mine
        for j, p in enumerate(mine.tolist()):
            here = min(page, n - j * page)
            k[p, :, :here] = torch.randn(kv_heads, here, dim, generator=gen).to(dtype)
            v[p, :, :here] = torch.randn(kv_heads, here, dim, generator=gen).to(dtype)
    return k.to(dev), v.to(dev), table.to(dev)


def positions_of(i, h, length, table, page, num_pages, pages):
    """(page of the cache, place in it) of every position that row i and key head h attend to, in order."""
    length = max(0, min(length, table.size(1) * page))
    held = (length + page - 1) // page
    listed = range(held) if pages is None else pages[i, h, :min(pages.size(2), held)].tolist()
    got = []
    for nth in listed:
        if not 0 <= nth < held:
            continue
        at = int(table[i, nth])
        if 0 <= at < num_pages:
            got += [(at, slot) for slot in range(min(page, length - nth * page))]
    return got


def attention(q, k, v, table, lengths, pages=None, scale=None):
    """(out, bound) in 64 bits on the CPU: bound is what |got - out| may be.

    Beside the output's rounding: a score is a sum of dim products in fp32 (an error of at most dim + 3 steps of 2^-23 of the terms,
    tensor cores truncating), twice as much with the factor and log2 e, and as an exponent a relative error of its weight, above the
    line and below; weights are kept to 2^-16 or better in the
    second product and summed in fp32 (a step of 2^-23 for every position, in the worst order)."""
    q, k, v, table = q.cpu().double(), k.cpu().double(), v.cpu().double(), table.cpu()
    pages = pages.cpu() if pages is not None else None
    rows, heads, dim = q.shape
    group, page = heads // k.size(1), k.size(2)
    scale = 1 / math.sqrt(dim) if scale is None else scale
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    for i in range(rows):
        for h in range(k.size(1)):
            at = positions_of(i, h, int(lengths[i]), table, page, k.size(0), pages)
            if not at:
                continue
            where, slot = torch.tensor(at).T
            keys, values = k[where, h, slot], v[where, h, slot]
            mine = q[i, h * group:(h + 1) * group]
            scores = mine @ keys.T * scale
            weights = torch.softmax(scores, -1)
            size = mine.abs() @ keys.abs().T * abs(scale)
            loss = weights * torch.expm1((2 * (dim + 3) * 2.0 ** -23 * size).clamp(max=30))
            mine_out = weights @ values
            out[i, h * group:(h + 1) * group] = mine_out
            bound[i, h * group:(h + 1) * group] = (loss @ values.abs() + loss.sum(-1, keepdim=True) * mine_out.abs()
                                                   + (2.0 ** -16 + len(at) * 2.0 ** -23) * (weights @ values.abs()))
    return out, bound


def check_attention(got, q, k, v, table, lengths, pages=None, scale=None):
    ref, bound = attention(q, k, v, table, lengths, pages, scale)
    got, dtype = got.cpu().double(), got.dtype
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    bound = bound + unit(dtype) * (ref.abs() + bound) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    off = (got - ref).abs()
    good = (off <= bound) | torch.isnan(ref)
    assert good.all(), f"off by {float((off / bound)[~good].max())} of what is allowed, {int((~good).sum())} of {good.numel()}"


def select(q, boxes, table, lengths, page, count, first, last):
    q, boxes, table = q.cpu().double(), boxes.cpu().double(), table.cpu()
    rows, heads, _ = q.shape
    kv_heads = boxes.size(1)
    group = heads // kv_heads
    chosen = torch.full((rows, kv_heads, count), -1, dtype=torch.int32)
    for i in range(rows):
        length = max(0, min(int(lengths[i]), table.size(1) * page))
        held = (length + page - 1) // page
        for h in range(kv_heads):
            mine = q[i, h * group:(h + 1) * group]
            up, down = mine.clamp(min=0).sum(0), mine.clamp(max=0).sum(0)
            keyed = []
            for nth in range(held):
                at = int(table[i, nth])
                if nth < first or nth >= held - last:
                    rank = (0, 0.0)
                elif not 0 <= at < boxes.size(0):
                    rank = (3, 0.0)
                else:
                    score = float((boxes[at, h, 1] * up + boxes[at, h, 0] * down).sum())
                    rank = (1, 0.0) if math.isnan(score) else (2, -score)
                keyed.append((rank, nth))
            nth = sorted(n for _, n in sorted(keyed)[:count])
            chosen[i, h, :len(nth)] = torch.tensor(nth, dtype=torch.int32)
    return chosen


def boxes_of(k, table, lengths, page):
    """Boxes of what the sequences hold; zero for pages that nobody holds."""
    boxes = torch.zeros(k.size(0), k.size(1), 2, k.size(3), dtype=k.dtype, device=k.device)
    for i, n in enumerate(lengths):
        for nth in range((n + page - 1) // page):
            at = int(table[i, nth])
            keys = k[at, :, :min(page, n - nth * page)]
            boxes[at] = torch.stack([keys.amin(1), keys.amax(1)], 1)
    return boxes


def turned(x, cos, sin, interleaved):
    """(x', bound) of x [tokens, heads, dim] in 64 bits with cos, sin [tokens, half]: two products and a sum in fp32."""
    x, cos, sin = x.double(), cos.double()[:, None], sin.double()[:, None]
    half = cos.size(-1)
    one, two = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    out, size = x.clone(), torch.zeros_like(x)
    out[..., one] = x[..., one] * cos - x[..., two] * sin
    out[..., two] = x[..., two] * cos + x[..., one] * sin
    size[..., one] = (x[..., one] * cos).abs() + (x[..., two] * sin).abs()
    size[..., two] = (x[..., two] * cos).abs() + (x[..., one] * sin).abs()
    return out, 3 * 2.0 ** -24 * size


def check_turned(got, x, cos, sin, interleaved):
    ref, bound = turned(x, cos, sin, interleaved)
    bound = bound + unit(got.dtype) * (ref.abs() + bound) + torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    assert ((got.double() - ref).abs() <= bound).all()
