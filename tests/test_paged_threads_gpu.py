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
