"""A paged key-value cache for decoding, and attention of new tokens over it.

The layers of this package that a decoding model runs between its projections' inputs and outputs (``SparseLinear``,
``ReluSparseDownProj``) leave attention to the caller; ``SparseAttentionChain`` has one fixed mask and no softmax.  Here are the
operators of a decoding step, on a cache whose pages are handed out by the caller:

    q = paged_append(q, k, v, k_cache, v_cache, block_table, lengths, rope=rope, boxes=boxes)
    out = paged_attention(q, k_cache, v_cache, block_table, lengths)

or, reading ``count`` pages of each sequence only, chosen for every row and key head by a cheap score,

    pages = paged_select(q, boxes, block_table, lengths, page_size, count)
    out = paged_attention(q, k_cache, v_cache, block_table, lengths, pages=pages)

``k_cache`` and ``v_cache`` are ``[pages, kv_heads, page_size, head_dim]``, float16 or bfloat16, ``page_size`` 16, 32, 64, 128 or
256, ``head_dim`` a multiple of 8 up to 128; each page is contiguous, pages may lie at any distance (``cache[:, 0]`` and
``cache[:, 1]`` of one ``[pages, 2, ...]`` tensor will do).  ``block_table`` int32 ``[rows, width]`` names each sequence's pages in order (what lies
behind the pages it needs may be anything), ``lengths`` int32 ``[rows]`` how many positions it holds, new tokens included; a row of
length 0 is idle.  Heads are grouped: query heads ``h * heads / kv_heads`` and the following read key head ``h``.

The operators run on the current stream, read nothing back and can be captured into a CUDA graph.  They have no backward
pass and no forward derivatives: operands that require a gradient or have a tangent are refused.  ``PagedKVCache`` owns the tensors and passes them along.
"""
from __future__ import annotations

import torch

from .. import ops


def rope_table(positions: int, rotary_dim: int, base: float = 10000.0, device="cuda"):
    """``(cos, sin)``, each float32 ``[positions, rotary_dim / 2]``: the angles ``p * base^(-2 i / rotary_dim)`` of rotary position
    embedding, computed in 64 bits (in 32, those of far positions are off by 1e-2)."""
    if positions < 0 or rotary_dim < 0 or rotary_dim % 2:
        raise RuntimeError(f"rope_table expects a number of positions and an even width, got {positions} and {rotary_dim}")
    half = rotary_dim // 2
    exponent = torch.arange(half, device=device, dtype=torch.float64) / max(half, 1)
    angle = torch.arange(positions, device=device, dtype=torch.float64)[:, None] * float(base) ** -exponent
    return angle.cos().float(), angle.sin().float()


def paged_append(q, k, v, k_cache, v_cache, block_table, lengths, cu_tokens=None, rope=None, interleaved: bool = False,
                 boxes=None) -> torch.Tensor:
    """Writes the keys and values of new tokens into the cache and returns the queries, both turned by their positions.

    ``q`` ``[tokens, heads, head_dim]``, ``k`` and ``v`` ``[tokens, kv_heads, head_dim]`` (slices of a fused projection are read as they
    lie).  Sequence ``i`` has the rows ``cu_tokens[i]`` to ``cu_tokens[i + 1]`` (int32 ``[sequences + 1]``, ascending from 0), or without it
    row ``i``; its last one takes position ``lengths[i] - 1``.  ``rope`` is ``(cos, sin)`` as ``rope_table`` makes them: the first
    ``2 * cos.size(1)`` elements of a head are turned, element ``i`` with ``i + cos.size(1)``, or ``2 i`` with ``2 i + 1`` if ``interleaved``.
    ``boxes`` ``[pages, kv_heads, 2, head_dim]`` keeps the smallest and largest key of each page in each dimension: those of the pages that
    are written to are formed from all positions of the page up to the last new one (also where a sequence was cut back).

    Rows behind the last sequence, and tokens that have no place (position below 0, behind the table or behind ``rope``, a page that
    is not one of the cache's), come back as zeros and leave the cache as it is.  A page that is written belongs to one sequence of the call."""
    cos, sin = rope if rope is not None else (None, None)
    out = ops.native.paged_append(q, k, v, k_cache, v_cache, block_table, lengths, cu_tokens, cos, sin, interleaved, boxes)
    if out is None:
        out = torch.ops.iex_ops.paged_append(q, k, v, k_cache, v_cache, block_table, lengths, cu_tokens, cos, sin, interleaved,
                                             boxes)
    return out


def paged_attention(q, k_cache, v_cache, block_table, lengths, pages=None, scale: float | None = None) -> torch.Tensor:
    """``softmax(scale * q k^T) v`` of every row of ``q`` ``[rows, heads, head_dim]`` over the positions of its own row of
    ``block_table``; ``scale`` is ``head_dim ** -0.5`` by default.  Zeros for a row that holds nothing.
    Scores are held in 32 bits, times ``log2(e)``; a ``scale`` that leaves their range is refused.

    A piece of a prompt is several rows with the same row of the table, each with the length that it sees; every row reads its keys
    for itself, and the table has a row for each (8 times 512 tokens behind up to 2048 positions take 1.7 ms).  ``pages`` int32
    ``[rows, kv_heads, count]`` restricts a row to these places of its row of the table, as ``paged_select`` returns them: of
    the first ``min(count, pages held)`` entries those that are held (one that is there twice counts twice)."""
    out = ops.native.paged_attention(q, k_cache, v_cache, block_table, lengths, pages, scale)
    if out is None:
        out = torch.ops.iex_ops.paged_attention(q, k_cache, v_cache, block_table, lengths, pages, scale)
    return out


def paged_select(q, boxes, block_table, lengths, page_size: int, count: int, first: int = 1, last: int = 1) -> torch.Tensor:
    """The ``count`` pages that each row of ``q`` attends to, int32 ``[rows, kv_heads, count]``: places in its row of ``block_table``,
    ascending, -1 behind them.

    The ``first`` first and ``last`` last pages held are always taken, the others by the most that a key inside a page's box could give,
    ``sum_d hi_d max(q_d, 0) + lo_d min(q_d, 0)`` summed over the query heads of the key head, in 64 bits; NaN counts as the
    largest, ties go to the lower page.  An infinite ``lo_d`` or ``hi_d`` with a factor of 0 makes NaN, so that a page with a key that
    overflowed is taken.  A row that holds no more than ``count`` pages takes all of them."""
    out = ops.native.paged_select(q, boxes, block_table, lengths, page_size, count, first, last)
    if out is None:
        out = torch.ops.iex_ops.paged_select(q, boxes, block_table, lengths, page_size, count, first, last)
    return out


class PagedKVCache:
    """The tensors of one layer's cache, and the operators above on them.

    ``k`` and ``v`` ``[pages, kv_heads, page_size, head_dim]``, ``boxes`` ``[pages, kv_heads, 2, head_dim]`` (``boxes=False`` leaves it out:
    ``select`` is then an error).  Which page belongs to which sequence is the caller's."""

    def __init__(self, pages: int, kv_heads: int, head_dim: int, page_size: int = 64, dtype=torch.float16, device="cuda",
                 boxes: bool = True):
        if dtype not in (torch.float16, torch.bfloat16):
            raise RuntimeError(f"PagedKVCache holds float16 or bfloat16, not {dtype}")
        if page_size not in (16, 32, 64, 128, 256) or head_dim % 8 or not 0 < head_dim <= 128 or kv_heads < 1 or pages < 0:
            raise RuntimeError("PagedKVCache: page_size 16, 32, 64, 128 or 256, head_dim a multiple of 8 up to 128, "
                               f"kv_heads positive; got {page_size}, {head_dim} and {kv_heads}")
        self.page_size = page_size
        self.k = torch.zeros(pages, kv_heads, page_size, head_dim, dtype=dtype, device=device)
        self.v = torch.zeros_like(self.k)
        self.boxes = torch.zeros(pages, kv_heads, 2, head_dim, dtype=dtype, device=device) if boxes else None

    def append(self, q, k, v, block_table, lengths, cu_tokens=None, rope=None, interleaved: bool = False) -> torch.Tensor:
        return paged_append(q, k, v, self.k, self.v, block_table, lengths, cu_tokens, rope, interleaved, self.boxes)

    def attend(self, q, block_table, lengths, pages=None, scale: float | None = None) -> torch.Tensor:
        return paged_attention(q, self.k, self.v, block_table, lengths, pages, scale)

    def select(self, q, block_table, lengths, count: int, first: int = 1, last: int = 1) -> torch.Tensor:
        if self.boxes is None:
            raise RuntimeError("PagedKVCache.select needs the boxes that this cache was made without")
        return paged_select(q, self.boxes, block_table, lengths, self.page_size, count, first, last)

    def attend_selected(self, q, block_table, lengths, count: int, first: int = 1, last: int = 1, scale: float | None = None):
        """``(out, pages)``: attention over the ``count`` pages that ``select`` chooses."""
        pages = self.select(q, block_table, lengths, count, first, last)
        return self.attend(q, block_table, lengths, pages, scale), pages
