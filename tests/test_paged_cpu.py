"""CPU: what the paged cache's operators refuse before any launch, the angles' table, and the operators' schemas."""
import math

import pytest
import torch

from intrasm_engine_b200 import _lib, ops
from intrasm_engine_b200.pytorch import paged_attention as paged


def test_rope_table_holds_the_angles_of_far_positions():
    cos, sin = paged.rope_table(200001, 64, 10000.0, device="cpu")
    assert cos.shape == sin.shape == (200001, 32) and cos.dtype == sin.dtype == torch.float32
    for p in (0, 1, 77777, 200000):
        for i in (0, 1, 17, 31):
            angle = p * 10000.0 ** (-2 * i / 64)
            # the table's rounding, and that of the power and the product in 64 bits
            assert abs(float(cos[p, i]) - math.cos(angle)) <= 2.0 ** -24 + 4 * angle * 2.0 ** -53
            assert abs(float(sin[p, i]) - math.sin(angle)) <= 2.0 ** -24 + 4 * angle * 2.0 ** -53
    assert paged.rope_table(3, 0, device="cpu")[0].shape == (3, 0)
    for bad in ((4, 5), (-1, 4), (4, -2)):
        with pytest.raises(RuntimeError):
            paged.rope_table(*bad, device="cpu")


def test_cache_refuses_what_the_kernels_do_not_take():
    cache = paged.PagedKVCache(3, 2, 80, 16, torch.bfloat16, device="cpu")
    assert cache.k.shape == cache.v.shape == (3, 2, 16, 80) and cache.boxes.shape == (3, 2, 2, 80)
    assert paged.PagedKVCache(3, 2, 80, device="cpu", boxes=False).boxes is None
    for kwargs in (dict(page_size=48), dict(page_size=8), dict(page_size=512), dict(head_dim=84), dict(head_dim=136),
                   dict(head_dim=0), dict(kv_heads=0), dict(pages=-1), dict(dtype=torch.float32)):
        with pytest.raises(RuntimeError):
            paged.PagedKVCache(**{**dict(pages=3, kv_heads=2, head_dim=64, device="cpu"), **kwargs})
    with pytest.raises(RuntimeError):
        paged.PagedKVCache(3, 2, 80, device="cpu", boxes=False).select(None, None, None, 4)


def test_cpu_tensors_reach_no_implementation():
    cache = paged.PagedKVCache(3, 2, 64, 16, device="cpu")
    q = torch.zeros(1, 2, 64, dtype=torch.float16)
    table, lengths = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for call in (lambda: cache.append(q, q, q, table, lengths), lambda: cache.attend(q, table, lengths),
                 lambda: cache.select(q, table, lengths, 2)):
        with pytest.raises((NotImplementedError, RuntimeError)):
            call()


def test_derivatives_are_refused_ahead_of_any_implementation():
    """Calls through the dispatcher, function transforms among them: no output without a gradient or a tangent."""
    from torch.autograd import forward_ad
    q = torch.ones(1, 2, 64, dtype=torch.float16)
    cache = torch.zeros(3, 2, 16, 64, dtype=torch.float16)
    boxes = torch.zeros(3, 2, 2, 64, dtype=torch.float16)
    table, lengths = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    calls = (lambda q: torch.ops.iex_ops.paged_append(q, q.detach(), q.detach(), cache, cache.clone(), table, lengths),
             lambda q: torch.ops.iex_ops.paged_attention(q, cache, cache, table, lengths),
             lambda q: torch.ops.iex_ops.paged_select(q, boxes, table, lengths, 16, 2).float())
    for call in calls:
        with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="q has a tangent"):
            call(forward_ad.make_dual(q, torch.ones_like(q)))
        with pytest.raises(NotImplementedError, match="q has a tangent"):
            torch.func.jvp(call, (q,), (torch.ones_like(q),))
        with pytest.raises(RuntimeError, match="q requires a gradient"):
            torch.func.grad(lambda x: call(x).sum())(q)
        with pytest.raises(RuntimeError, match="q requires a gradient"):
            call(q.clone().requires_grad_(True))


def test_schemas_name_what_is_written():
    text = str(torch.ops.iex_ops.paged_append.default._schema)
    assert "Tensor(a!) k_cache" in text and "Tensor(b!) v_cache" in text and "Tensor(c!)? boxes" in text
    assert "!" not in str(torch.ops.iex_ops.paged_attention.default._schema)
    assert {"paged_append", "paged_attention", "paged_select"} <= set(ops.OP_NAMES)


def test_attention_refuses_scales_that_overflow_as_exponents_of_two():
    """The kernels' factor is scale * log2(e) in fp32: finite up to 2.3586e38.  Refused before any launch."""
    x = 4096  # an aligned address that nothing reads
    def attention(scale, rows):
        return _lib.lib.iex_paged_attention(rows, 4, 2, 64, 0, x, 256, 64, x, 2048, x, 2048, 3, 16, x, 2, x, None, 0, scale, x, None, 0,
                                            None)
    for rows in (0, 1):
        for scale in (3e38, -3e38, 2.36e38, 3.4028e38, float("inf"), float("nan")):
            assert attention(scale, rows) == -1, scale
    for scale in (2.35e38, -2.35e38, 0.0, 0.125):
        assert attention(scale, 0) == 0, scale


def test_entry_points_check_their_arguments():
    """The C ABI returns a status before any launch: nothing here needs a device."""
    lib, bad, unsupported, too_large = _lib.lib, -1, -2, -3
    assert lib.iex_paged_attention_supported(32, 8, 128, 64) == 1
    for args in ((32, 8, 132, 64), (32, 8, 136, 64), (32, 8, 128, 48), (30, 8, 128, 64), (0, 8, 128, 64), (8, 0, 128, 64)):
        assert lib.iex_paged_attention_supported(*args) == 0

    x = 4096  # an aligned address that nothing reads
    def attention(rows=1, heads=4, kv=2, dim=64, q=x, q_row=256, q_head=64, cache=x, stride=2048, num=3, page=16, table=x,
                  width=2, lengths=x, pages=None, count=0, out=x, ws=None, ws_bytes=0):
        return lib.iex_paged_attention(rows, heads, kv, dim, 0, q, q_row, q_head, cache, stride, cache, stride, num, page, table,
                                       width, lengths, pages, count, 1.0, out, ws, ws_bytes, None)
    assert attention(rows=0) == 0
    for kwargs in (dict(rows=-1), dict(num=-1), dict(width=-1), dict(count=-1), dict(q=None), dict(out=None),
                   dict(lengths=None), dict(table=None), dict(cache=None)):
        assert attention(**kwargs) == bad, kwargs
    for kwargs in (dict(dim=60), dict(page=24), dict(heads=3), dict(q_row=260), dict(q_head=4), dict(stride=2049), dict(q=x + 8),
                   dict(out=x + 2), dict(cache=x + 4)):
        assert attention(**kwargs) == unsupported, kwargs

    for width, page in ((2 ** 23, 256), (2 ** 27, 16), (2 ** 31 - 1, 256)):
        assert attention(width=width, page=page) == too_large
    assert attention(heads=2 ** 24, kv=1) == unsupported

    def select(rows=1, heads=4, kv=2, dim=64, q=x, q_row=256, boxes=x, num=3, page=16, table=x, width=2, lengths=x, count=2,
               first=1, last=1, pages=x):
        return lib.iex_paged_select(rows, heads, kv, dim, 0, q, q_row, 64, boxes, num, page, table, width, lengths, count, first,
                                    last, pages, None)
    assert select(rows=0) == 0
    for kwargs in (dict(rows=-1), dict(count=0), dict(first=-1), dict(last=-1), dict(first=2), dict(first=2 ** 31 - 1, last=2 ** 31 - 1),
                   dict(q=None), dict(pages=None), dict(boxes=None), dict(lengths=None), dict(table=None)):
        assert select(**kwargs) == bad, kwargs
    for kwargs in (dict(dim=60), dict(page=24), dict(heads=3), dict(q_row=260), dict(boxes=x + 8)):
        assert select(**kwargs) == unsupported, kwargs
    assert select(width=lib.iex_paged_select_max_pages() + 1) == too_large

    def append(tokens=2, batch=2, heads=4, kv=2, dim=64, q=x, q_row=256, k=x, cos=x, sin=x, rope_rows=9, rotary=64, out=x,
               cache=x, stride=2048, boxes=x, num=3, page=16, table=x, width=2, lengths=x, cu=None):
        return lib.iex_paged_append(tokens, batch, heads, kv, dim, 0, q, q_row, 64, k, 128, 64, k, 128, 64, cos, sin, rope_rows,
                                    rotary, 0, out, cache, stride, cache, stride, boxes, num, page, table, width, lengths, cu, None)
    assert append(tokens=0, batch=0) == 0
    for kwargs in (dict(tokens=-1), dict(batch=-1), dict(num=-1), dict(width=-1), dict(rope_rows=-1), dict(rotary=-2), dict(q=None),
                   dict(k=None), dict(cos=None), dict(sin=None), dict(out=None), dict(cache=None), dict(table=None),
                   dict(lengths=None), dict(tokens=3)):
        assert append(**kwargs) == bad, kwargs
    for kwargs in (dict(dim=60), dict(page=24), dict(heads=3), dict(rotary=31), dict(rotary=66), dict(q_row=260), dict(boxes=x + 8),
                   dict(k=x + 4), dict(stride=2052)):
        assert append(**kwargs) == unsupported, kwargs
    for width, page in ((2 ** 23, 256), (2 ** 27, 16), (2 ** 31 - 1, 256)):
        assert append(width=width, page=page) == too_large


# of the cases of test_paged_gpu.SHARED, in order: whether pages are read once for many rows
SHARED_PATHS = [True, True, True, True, True, False, False, True, False, True]


def test_scratch_of_shared_pages_is_bounded():
    """By its size alone, whatever the number of entries; sizes whose products leave 64 bits take none."""
    def need(rows, count, heads=1, dim=64, width=1 << 20):
        return _lib.lib.iex_paged_attention_workspace_bytes(rows, heads, heads, dim, 900, 64, width, 1, count)
    assert 60 << 20 < need(8192, 30) < 80 << 20 and 80 << 20 < need(8192, 40) < 100 << 20  # 2^18 entries are in between
    assert 500 << 20 < need(1 << 15, 58) <= 512 << 20
    for rows, count in ((1 << 15, 64), (1 << 20, 1 << 20), (2 ** 31 - 1, 1 << 20)):
        assert need(rows, count) < 1 << 20


def test_cases_of_shared_pages_take_the_path_that_they_stand_for():
    from .test_paged_gpu import SHARED
    assert len(SHARED) == len(SHARED_PATHS)
    for (rows, heads, kv_heads, dim, page, longest, count), shared in zip(SHARED, SHARED_PATHS):
        width = (longest + page - 1) // page
        def need(pages):
            return _lib.lib.iex_paged_attention_workspace_bytes(rows, heads, kv_heads, dim, pages, page, width, 1, count)
        # of a cache with more pages than are ever sorted, rows read their pages one by one
        assert (need(width + 2) != need(1 << 20)) == shared, (rows, heads, kv_heads, dim, page, longest, count)
