"""GPU: the paged cache's operators called by several host threads at once, through the C ABI, which holds no lock."""
import threading

import pytest
import torch

from intrasm_engine_b200 import _lib

from .paged_util import DEV

pytestmark = pytest.mark.gpu


def at_once(calls, turns):
    """Every call `turns` times by a thread of its own; the statuses that were not 0."""
    gate, failed = threading.Barrier(len(calls)), []

    def work(call):
        gate.wait()
        failed.extend(status for status in (call() for _ in range(turns)) if status != 0)

    threads = [threading.Thread(target=work, args=(call,)) for call in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    return failed


def test_selection_from_a_wide_and_from_a_narrow_table():
    """What one call needs of shared memory is no bound for another that is under way."""
    rows, dim, count, pages = 1, 64, 9, 100
    boxes = torch.randn(pages, 1, 2, dim, device=DEV).sort(2).values.half()
    q = torch.randn(rows, 2, dim, device=DEV).half()
    calls, outs = [], []
    for width in (16384, 3000, 9000, 2800):
        table = torch.randint(0, pages, (rows, width), device=DEV, dtype=torch.int32)
        held = torch.tensor([width * 16], device=DEV, dtype=torch.int32)
        out = torch.empty(rows, 1, count, device=DEV, dtype=torch.int32)
        stream = torch.cuda.Stream()
        outs.append((table, held, out, stream))
        calls.append(lambda width=width, table=table, held=held, out=out, stream=stream: _lib.lib.iex_paged_select(
            rows, 2, 1, dim, 0, q.data_ptr(), 2 * dim, dim, boxes.data_ptr(), pages, 16, table.data_ptr(), width,
            held.data_ptr(), count, 1, 1, out.data_ptr(), stream.cuda_stream))
    torch.cuda.synchronize()
    for call in calls:
        assert call() == 0
    torch.cuda.synchronize()
    alone = [out.clone() for _, _, out, _ in outs]
    for _, _, out, _ in outs:
        out.fill_(-9)
    torch.cuda.synchronize()
    assert at_once(calls, 4000) == []
    assert all(torch.equal(a, out) for a, (_, _, out, _) in zip(alone, outs))


def test_listed_pages_of_a_large_and_of_a_small_cache():
    rows, count, dim, page, width = 4096, 16, 8, 256, 32
    q = torch.randn(rows, 1, dim, device=DEV).half()
    held = torch.full((rows,), width * page, device=DEV, dtype=torch.int32)
    pages = torch.rand(rows, 1, width, device=DEV).argsort(-1)[..., :count].int().contiguous()
    calls, outs = [], []
    for total in (6000, 3500, 5000, 3450):
        k, v = (torch.randn(total, 1, page, dim, device=DEV).half() for _ in range(2))
        table = torch.randint(0, total, (1, width), device=DEV, dtype=torch.int32).expand(rows, -1).contiguous()
        need = _lib.lib.iex_paged_attention_workspace_bytes(rows, 1, 1, dim, total, page, width, 1, count)
        assert need > 2 << 20  # by page; row by row needs less
        out, ws = torch.empty_like(q), torch.empty(need, device=DEV, dtype=torch.uint8)
        stream = torch.cuda.Stream()
        outs.append((out, ws, k, v, table, stream))
        calls.append(lambda total=total, k=k, v=v, table=table, out=out, ws=ws, stream=stream: _lib.lib.iex_paged_attention(
            rows, 1, 1, dim, 0, q.data_ptr(), dim, dim, k.data_ptr(), page * dim, v.data_ptr(), page * dim, total, page,
            table.data_ptr(), width, held.data_ptr(), pages.data_ptr(), count, 0.125, out.data_ptr(), ws.data_ptr(),
            ws.numel(), stream.cuda_stream))
    torch.cuda.synchronize()
    for call in calls:
        assert call() == 0
    torch.cuda.synchronize()
    alone = [o[0].clone() for o in outs]
    for o in outs:
        o[0].fill_(float("nan"))
    torch.cuda.synchronize()
    assert at_once(calls, 400) == []
    assert all(torch.equal(a, o[0]) for a, o in zip(alone, outs))
