"""GPU: the paged cache's operators against their definitions in 64 bits (paged_util.py)."""
import pytest
import torch

from intrasm_engine_b200.pytorch import paged_attention as paged

from . import paged_util as U
from .paged_util import DEV

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def case(lengths, heads, kv_heads, dim, page, dtype, seed=0, std=1.0, **kwargs):
    gen = torch.Generator().manual_seed(seed)
    k, v, table = U.make_cache(gen, lengths, kv_heads, dim, page, dtype, **kwargs)
    q = (torch.randn(len(lengths), heads, dim, generator=gen) * std).to(dtype).to(DEV)
    return q, k, v, table, ints(lengths)


# ------------------------------------------------------------------------------------------------- attention

SHAPES = [
    # lengths, heads, kv_heads, dim, page
    ([1], 1, 1, 8, 16),
    ([0, 1, 2, 15, 16, 17, 0, 31, 33], 4, 2, 64, 16),
    ([63, 64, 65, 127, 128, 129, 0], 8, 1, 128, 64),
    ([500], 32, 32, 128, 64),
    ([1003, 1, 700, 0, 333], 6, 6, 80, 16),
    ([257, 4096, 5], 10, 2, 96, 256),
    ([3000, 40], 16, 1, 128, 32),
    ([100, 2000, 31], 24, 1, 64, 128),
    ([777], 33, 1, 40, 16),
    ([0, 0, 0], 2, 2, 32, 16),
    ([50] * 70, 12, 4, 64, 32),
    ([9000, 10], 4, 4, 128, 64),
    ([200, 900], 5, 1, 104, 64),
    ([1500], 48, 2, 120, 64),
]


@pytest.mark.parametrize("dtype", U.DTYPES)
@pytest.mark.parametrize("lengths,heads,kv_heads,dim,page", SHAPES)
def test_attention(lengths, heads, kv_heads, dim, page, dtype):
    # what nobody holds is NaN, entries of the table behind a row's pages lie outside the cache
    q, k, v, table, held = case(lengths, heads, kv_heads, dim, page, dtype)
    got = paged.paged_attention(q, k, v, table, held)
    assert got.shape == q.shape and got.dtype == dtype and got.is_contiguous()
    U.check_attention(got, q, k, v, table, lengths)
    for i, n in enumerate(lengths):
        if n == 0:
            assert not got[i].any()


@pytest.mark.parametrize("dtype", U.DTYPES)
def test_attention_of_large_and_small_scores(dtype):
    for seed, std in enumerate((0.0, 0.01, 8.0, 40.0)):
        q, k, v, table, held = case([700, 90], 8, 2, 64, 32, dtype, seed=seed, std=std)
        U.check_attention(paged.paged_attention(q, k, v, table, held), q, k, v, table, [700, 90])
    for scale in (0.0, -0.3, 2.5):
        got = paged.paged_attention(q, k, v, table, held, scale=scale)
        U.check_attention(got, q, k, v, table, [700, 90], scale=scale)


@pytest.mark.parametrize("dtype", U.DTYPES)
def test_attention_follows_a_rising_maximum(dtype):
    """Scores that grow with the position, and ones that fall: the running maximum changes all the time, or never."""
    for sign in (1.0, -1.0):
        q, k, v, table, held = case([2500], 4, 1, 64, 64, dtype)
        q.fill_(0.0)
        q[..., 0] = sign
        for j in range((2500 + 63) // 64):
            k[int(table[0, j]), 0, :, 0] = (torch.arange(64, device=DEV) + 64 * j).to(dtype) * 0.25
        U.check_attention(paged.paged_attention(q, k, v, table, held), q, k, v, table, [2500])


def test_what_is_not_finite_reaches_the_rows_that_hold_it():
    lengths = [300, 200, 64]
    q, k, v, table, held = case(lengths, 4, 2, 64, 32, F16)
    k[int(table[0, 3]), 1, 7, 5] = float("nan")   # row 0, key head 1
    v[int(table[1, 2]), 0, 3, 9] = float("inf")   # row 1, key head 0, one element
    q[2, 3, 0] = float("nan")
    got = paged.paged_attention(q, k, v, table, held)
    clean = torch.isfinite(got)
    assert not clean[0, 2:].any() and clean[0, :2].all()
    assert clean[1, 2:].all() and (got[1, :2, 9] == float("inf")).all() and clean[1, :2].sum() == 2 * 63
    assert clean[2, :3].all() and not clean[2, 3].any()


@pytest.mark.parametrize("dtype", U.DTYPES)
def test_infinite_values_among_many_rows(dtype):
    """More segments than there are blocks; what is infinite is at the largest score, at a small one, and twice of opposite signs."""
    lengths = [300] * 30 + [17] * 30
    q, k, v, table, held = case(lengths, 8, 8, 64, 32, dtype)
    ref, bound = U.attention(q, k, v, table, lengths)
    scores = torch.stack([k[table[7].long()[:10], 2].reshape(-1, 64)[:300].float() @ q[7, 2].float()])[0]
    best, worst = int(scores.argmax()), int(scores.argmin())
    def put(row, head, position, element, value):
        v[int(table[row, position // 32]), head, position % 32, element] = value
    put(7, 2, best, 5, float("inf"))
    put(7, 2, worst, 6, float("-inf"))
    put(40, 1, 3, 0, float("inf"))
    put(40, 1, 16, 0, float("-inf"))
    put(40, 1, 16, 1, float("-inf"))
    got = paged.paged_attention(q, k, v, table, held).cpu().double()
    assert got[7, 2, 5] == float("inf") and got[7, 2, 6] == float("-inf")
    assert torch.isnan(got[40, 1, 0]) and got[40, 1, 1] == float("-inf")
    keep = torch.isfinite(got)
    assert int((~keep).sum()) == 4
    bound = bound + U.unit(dtype) * (ref.abs() + bound) + 1e-7
    assert ((got - ref).abs() <= bound)[keep].all()


def with_large_values(v, seed=0):
    """v with values whose sums leave fp32 and whose averages do not: of 8 elements of a head two all positive, two of both signs, two
    as they were, two small ones.  What nobody holds stays NaN."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    large = v.clone()
    size = (torch.rand(v.shape, generator=gen, device=DEV) * 0.8 + 2.5) * 1e38
    sign = torch.where(torch.rand(v.shape, generator=gen, device=DEV) < 0.5, -1.0, 1.0)
    large[..., 0::8] = size[..., 0::8].to(v.dtype)
    large[..., 1::8] = (size * sign)[..., 1::8].to(v.dtype)
    large[..., 4::8] = size[..., 4::8].to(v.dtype)
    large[..., 5::8] = (size * sign)[..., 5::8].to(v.dtype)
    large[..., 3::8] *= 1e-36
    large[..., 7::8] *= 1e-37
    return torch.where(torch.isnan(v), v, large)


def check_large(got, q, k, v, table, lengths, pages=None):
    """Infinite and NaN elements as the definition has them, finite ones within its bound."""
    ref, bound = U.attention(q, k, v, table, lengths, pages)
    got = got.cpu().double()
    plain = torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)) and torch.equal(torch.isinf(got), torch.isinf(ref))
    assert torch.equal(got[torch.isinf(ref)], ref[torch.isinf(ref)])
    tiny = torch.finfo(BF16).smallest_normal * torch.finfo(BF16).eps
    bound = bound + U.unit(BF16) * (ref.abs() + bound) + tiny
    assert ((got - ref).abs() <= bound)[plain].all()
    return plain


@pytest.mark.parametrize("lengths,heads,kv_heads,dim,page", [
    ([700, 0, 90], 4, 2, 64, 32),          # clusters of several blocks
    ([40, 17, 300] * 20, 8, 2, 128, 16),   # of one block
    ([300, 16] * 40, 8, 8, 64, 32),        # shares of warps
    ([3000, 200, 5] * 12, 24, 2, 128, 64),  # segments of several blocks, 16 query heads each
    ([20000] * 20, 8, 8, 128, 256),
    ([6000, 4000], 1, 1, 72, 16),
])
def test_values_whose_sums_leave_the_range_of_32_bits(lengths, heads, kv_heads, dim, page):
    """bfloat16 reaches as far as fp32: an average of its largest values is a number, their sum is not."""
    q, k, v, table, held = case(lengths, heads, kv_heads, dim, page, BF16)
    v = with_large_values(v)
    got = paged.paged_attention(q, k, v, table, held)
    assert check_large(got, q, k, v, table, lengths).all()
    # with infinite and NaN elements among them
    row = 0
    def put(head, position, element, value):
        v[int(table[row, position // page]), head, position % page, element] = value
    put(0, 5, 0, float("inf"))
    put(0, 7, 1, float("nan"))
    put(0, lengths[0] - 1, 2, float("-inf"))
    put(0, 11, 4, float("inf"))
    put(0, 12, 4, float("-inf"))
    plain = check_large(paged.paged_attention(q, k, v, table, held), q, k, v, table, lengths)
    assert int((~plain).sum()) == 4 * (heads // kv_heads)


def test_shared_pages_with_values_whose_sums_leave_the_range_of_32_bits():
    for args in ((128, 16, 4, 128, 64, 40 * 64 - 5, 8), (300, 16, 2, 104, 256, 12 * 256 - 200, 5)):
        q, k, v, table, lengths, lists = shared_case(*args, BF16, seed=4)
        assert takes_shared_pages(q, k, table, lists)
        v = with_large_values(v)
        got = paged.paged_attention(q, k, v, table, ints(lengths), pages=lists.to(DEV))
        assert check_large(got, q, k, v, table, lengths, lists).all()
        page = k.size(2)
        v[int(table[0, 1]), 0, 5, 0] = float("inf")
        v[int(table[0, 1]), 1, page - 1, 1] = float("nan")
        plain = check_large(paged.paged_attention(q, k, v, table, ints(lengths), pages=lists.to(DEV)), q, k, v, table, lengths, lists)
        assert not plain.all()


def test_scores_of_minus_infinity_weigh_nothing():
    q, k, v, table, held = case([150, 40], 2, 1, 64, 16, BF16)
    q.fill_(1.0)
    for j in range(1, 10):  # all of row 0 behind its first page
        k[int(table[0, j]), 0, :, 3] = float("-inf")
    for j in range(3):      # all of row 1
        k[int(table[1, j]), 0, :, 3] = float("-inf")
    got = paged.paged_attention(q, k, v, table, held)
    U.check_attention(got, q, k, v, table, [16, 0])


def test_the_lowest_values_of_the_type_are_scores_like_others():
    for dtype in U.DTYPES:
        q, k, v, table, held = case([150], 2, 1, 64, 16, dtype)
        q.fill_(0.0)
        q[..., 0] = 1.0
        k[..., 0] = 0.0
        k[int(table[0, 2]), 0, 5:, 0] = torch.finfo(dtype).min
        U.check_attention(paged.paged_attention(q, k, v, table, held, scale=1.0), q, k, v, table, [150], scale=1.0)


def test_lengths_and_tables_are_bounded_by_the_kernel():
    lengths = [100, 64, 30, 10]
    q, k, v, table, held = case(lengths, 4, 2, 64, 16, F16)
    # longer than the table: as long as the table; the entries of row 1 behind its 4 pages are not the cache's
    wild = [2 ** 31 - 1, 2 ** 31 - 1, -5, 10]
    got = paged.paged_attention(q, k, v, table, ints(wild))
    U.check_attention(got, q, k, v, table, wild)
    assert torch.isnan(got[0]).all() and not torch.isnan(got[1:]).any() and not got[2].any()
    holes = table.clone()
    holes[0, 2], holes[1, 0], holes[2, :] = -1, k.size(0), -2 ** 31
    got = paged.paged_attention(q, k, v, holes, held)
    U.check_attention(got, q, k, v, holes, lengths)
    assert not got[2].any()
    assert not paged.paged_attention(q, k[:0], v[:0], table, held).any()
    assert not paged.paged_attention(q, k, v, table[:, :0].contiguous(), held).any()
    assert paged.paged_attention(q[:0], k, v, table[:0], held[:0]).shape == (0, 4, 64)


def test_rows_of_q_and_pages_of_the_cache_at_other_distances():
    lengths, dim = [130, 77, 500], 64
    q, k, v, table, held = case(lengths, 8, 2, dim, 32, F16)
    ref = paged.paged_attention(q, k, v, table, held)
    fused = torch.randn(3, 8 * dim + 128, device=DEV).half()
    fused[:, 64:64 + 8 * dim] = q.reshape(3, -1)
    view = fused[:, 64:64 + 8 * dim].view(3, 8, dim)
    assert not view.is_contiguous() and torch.equal(paged.paged_attention(view, k, v, table, held), ref)
    odd = torch.zeros(3, 8, dim + 1, device=DEV).half()  # rows that are not on 16-byte boundaries
    odd[..., 1:] = q
    assert torch.equal(paged.paged_attention(odd[..., 1:], k, v, table, held), ref)
    assert torch.equal(paged.paged_attention(q.transpose(0, 1).contiguous().transpose(0, 1), k, v, table, held), ref)
    kv = torch.stack([k, v], 1)
    assert torch.equal(paged.paged_attention(q, kv[:, 0], kv[:, 1], table, held), ref)


@pytest.mark.parametrize("dtype", U.DTYPES)
def test_places_behind_two_to_the_32_bytes(dtype):
    """Pages 2^31 elements and more from the cache's start."""
    lengths, page, dim, far = [100], 16, 64, (1 << 31) + 1024
    q, k, v, table, held = case(lengths, 4, 2, dim, page, dtype)
    room = torch.empty(2 * far + 4096, dtype=dtype, device=DEV)
    wide = room.as_strided((3, 2, page, dim), (far, page * dim, dim, 1))
    to = [0, 2, 1]
    for j in range(3):
        wide[to[j]] = k[int(table[0, j])]
    near_v = torch.stack([v[int(table[0, j])] for j in (0, 2, 1)])
    got = paged.paged_attention(q, wide, near_v, ints([to]), ints([48]))
    U.check_attention(got, q, torch.stack([wide[j] for j in range(3)]), near_v, ints([to]), [48])


@pytest.mark.parametrize("dtype", U.DTYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(8, 2, 128, 64), (6, 6, 80, 16), (20, 1, 64, 32)])
def test_attention_over_listed_pages(heads, kv_heads, dim, page, dtype):
    lengths = [1000, 3 * page + 1, page, 0, 5]
    q, k, v, table, held = case(lengths, heads, kv_heads, dim, page, dtype)
    gen = torch.Generator().manual_seed(4)
    count = 7
    lists = torch.full((len(lengths), kv_heads, count), -1, dtype=torch.int32)
    for i, n in enumerate(lengths):
        pages = (n + page - 1) // page
        for h in range(kv_heads):
            some = torch.randperm(pages, generator=gen)[:count].sort().values
            lists[i, h, :len(some)] = some.int()
    got = paged.paged_attention(q, k, v, table, held, pages=lists.to(DEV))
    U.check_attention(got, q, k, v, table, lengths, pages=lists)
    # any order, one page twice, entries that are no page, and behind what the row holds nothing is read
    rough = lists.clone()
    rough[0, 0] = torch.tensor([5, 2, 2, 2 ** 31 - 1, 0, -9, 1000 // page])
    rough[1, 0] = torch.tensor([3, 0, 3, 1, 2, 1, 0])
    rough[2, 0] = torch.tensor([0, 0, 0, 0, 0, 0, 0])
    got = paged.paged_attention(q, k, v, table, held, pages=rough.to(DEV))
    U.check_attention(got, q, k, v, table, lengths, pages=rough)
    none = torch.zeros(len(lengths), kv_heads, 0, dtype=torch.int32, device=DEV)
    assert not paged.paged_attention(q, k, v, table, held, pages=none).any()
    every = torch.arange(table.size(1), dtype=torch.int32, device=DEV).expand(len(lengths), kv_heads, -1).contiguous()
    U.check_attention(paged.paged_attention(q, k, v, table, held, pages=every), q, k, v, table, lengths)


@pytest.mark.parametrize("rows,kv_heads,group,dim,dtype", [(700, 1, 1, 64, F16), (1500, 3, 2, 128, BF16), (9000, 32, 1, 64, F16), (900, 2, 9, 72, BF16)])
def test_attention_of_many_rows_that_share_a_table(rows, kv_heads, group, dim, dtype):
    """More rows than a block has threads, and, in the third case, more work than 32 bits of products hold."""
    gen = torch.Generator(device=DEV).manual_seed(rows)
    page, width = 16, 9
    k, v = (torch.randn(width + 2, kv_heads, page, dim, device=DEV, generator=gen).to(dtype) for _ in range(2))
    pages = torch.randperm(width + 2, device=DEV, generator=gen)[:width].to(torch.int32)
    table = pages.expand(rows, width).contiguous()
    held = torch.randint(0, width * page + 1, (rows,), device=DEV, generator=gen).to(torch.int32)
    held[::7] = 0
    q = torch.randn(rows, kv_heads * group, dim, device=DEV, generator=gen).to(dtype)
    got = paged.paged_attention(q, k, v, table, held).double()
    keys, values = (t[pages.long()].transpose(0, 1).reshape(kv_heads, width * page, dim).double() for t in (k, v))
    scores = torch.einsum("rhgd,hsd->rhgs", q.double().view(rows, kv_heads, group, dim), keys) * dim ** -0.5
    seen = (torch.arange(width * page, device=DEV) < held[:, None])[:, None, None]
    weights = torch.softmax(scores.masked_fill(~seen, -1e30), -1) * seen
    ref = torch.einsum("rhgs,hsd->rhgd", weights, values).reshape(q.shape)
    size = torch.einsum("rhgs,hsd->rhgd", weights, values.abs()).reshape(q.shape)
    # scores below 40 without their signs: exponents off by 2 (dim + 3) 2^-23 40, above the line and below (paged_util.attention)
    loss = 2 * (2 * (dim + 3) * 2.0 ** -23 * 40) + 2.0 ** -16 + width * page * 2.0 ** -23
    assert float(torch.einsum("rhgd,hsd->rhgs", q.double().abs().view(rows, kv_heads, group, dim), keys.abs()).max()) * dim ** -0.5 < 40
    assert ((got - ref).abs() <= loss * size + U.unit(dtype) * (ref.abs() + loss * size) + 1e-7).all()
    assert not got[held == 0].any()


# rows that list pages of one sequence: where enough of them do, a page is read once for many
SHARED = [
    # rows, heads, kv_heads, dim, page, longest, count
    (300, 36, 4, 80, 128, 31 * 128 - 9, 9),
    (300, 16, 2, 104, 256, 12 * 256 - 200, 5),
    (400, 32, 32, 64, 16, 60 * 16, 16),
    (512, 32, 2, 128, 256, 20 * 256 - 1, 8),
    (128, 16, 4, 128, 64, 40 * 64 - 5, 8),
    (400, 4, 4, 64, 16, 60 * 16, 16),
    (150, 27, 3, 80, 64, 30 * 64 + 1, 9),
    (140, 10, 2, 128, 128, 20 * 128 - 70, 6),
    (90, 32, 2, 104, 256, 12 * 256 - 200, 5),
    (300, 8, 8, 40, 32, 33 * 32 + 7, 20),
]


def shared_case(rows, heads, kv_heads, dim, page, longest, count, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    k, v, table = U.make_cache(gen, [longest], kv_heads, dim, page, dtype)
    table = table.expand(rows, -1).contiguous()
    q = torch.randn(rows, heads, dim, generator=gen).to(dtype).to(DEV)
    # a piece of a prompt at the end, rows anywhere, and idle ones
    lengths = [longest - rows // 2 + 1 + i for i in range(rows // 2)]
    lengths += [int(torch.randint(0, longest + 1, (1,), generator=gen)) for _ in range(rows - len(lengths))]
    lengths[-1], lengths[rows // 2], lengths[3] = 0, 1, longest
    lists = torch.full((rows, kv_heads, count), -1, dtype=torch.int32)
    for i, n in enumerate(lengths):
        held = (n + page - 1) // page
        for h in range(kv_heads):
            some = torch.randperm(held, generator=gen)[:count].sort().values
            lists[i, h, :len(some)] = some.int()
    return q, k, v, table, lengths, lists


def takes_shared_pages(q, k, table, lists):
    from intrasm_engine_b200 import _lib
    need = _lib.lib.iex_paged_attention_workspace_bytes(q.size(0), q.size(1), k.size(1), q.size(2), k.size(0), k.size(2), table.size(1), 1,
                                                        lists.size(2))
    return need > 4 << 20  # the other kernels need less


@pytest.mark.parametrize("dtype", U.DTYPES)
@pytest.mark.parametrize("rows,heads,kv_heads,dim,page,longest,count", SHARED)
def test_attention_over_pages_that_rows_share(rows, heads, kv_heads, dim, page, longest, count, dtype):
    q, k, v, table, lengths, lists = shared_case(rows, heads, kv_heads, dim, page, longest, count, dtype)
    assert rows * heads < 8192 or takes_shared_pages(q, k, table, lists)
    got = paged.paged_attention(q, k, v, table, ints(lengths), pages=lists.to(DEV))
    U.check_attention(got, q, k, v, table, lengths, pages=lists)
    assert not got[-1].any()
    # any order, a page twice, entries that are no page, lengths and tables that are none
    rough = lists.clone()
    rough[0, 0] = rough[0, 0].flip(0)
    rough[1, :, 1] = rough[1, :, 0]
    rough[2, 0, 0], rough[2, 0, 1] = -7, 2 ** 31 - 1
    rough[4] = rough[4, :, :1]
    wild, holes = list(lengths), table.clone()
    wild[6] = -3
    holes[7, 0], holes[8, :] = -1, k.size(0)
    got = paged.paged_attention(q, k, v, holes, ints(wild), pages=rough.to(DEV))
    U.check_attention(got, q, k, v, holes, wild, pages=rough)
    assert torch.equal(got, paged.paged_attention(q, k, v, holes, ints(wild), pages=rough.to(DEV)))


@pytest.mark.parametrize("dtype", U.DTYPES)
def test_shared_pages_keep_what_is_not_finite_to_the_rows_that_see_it(dtype):
    q, k, v, table, lengths, lists = shared_case(128, 16, 4, 128, 64, 40 * 64 - 5, 8, dtype, seed=3)
    assert takes_shared_pages(q, k, table, lists)
    ref, bound = U.attention(q, k, v, table, lengths, pages=lists)
    last = (lengths[3] - 1) // 64
    lists[:64, :, 0] = last  # the piece of a prompt: all rows list the last page, of which they see more and more
    lists[:64] = lists[:64].sort(-1).values
    for i in range(64):
        for h in range(4):
            seen = torch.unique(lists[i, h])
            seen = torch.cat([seen, torch.full((8 - len(seen),), -1, dtype=torch.int32)])
            lists[i, h] = seen
    ref, bound = U.attention(q, k, v, table, lengths, pages=lists)
    spot = lengths[3] - 1 - last * 64 - 20            # seen by rows from some on
    v[int(table[0, last]), 1, spot, 9] = float("inf")
    k[int(table[0, last]), 2, spot, 5] = float("nan")
    got = paged.paged_attention(q, k, v, table, ints(lengths), pages=lists.to(DEV)).cpu().double()
    expected = torch.isfinite(got)
    sees = torch.tensor([any(int(x) == last for x in lists[i, 1]) and n > last * 64 + spot for i, n in enumerate(lengths)])
    assert (got[sees][:, 4:8, 9] == float("inf")).all() and torch.isnan(got[sees][:, 8:12]).all() and 10 < int(sees.sum()) < 64
    expected[sees, 4:8, 9] = True
    expected[sees, 8:12] = True
    assert expected.all()
    keep = torch.isfinite(got)
    bound = bound + U.unit(dtype) * (ref.abs() + bound) + 1e-7
    assert ((got - ref).abs() <= bound)[keep].all()


def test_shared_pages_in_graphs_and_whatever_scratch_memory_held():
    cases = [shared_case(128, 16, 4, 128, 64, 40 * 64 - 5, 8, F16, seed=s) for s in (5, 6)]
    expected, graphs = [], []
    for q, k, v, table, lengths, lists in cases:
        assert takes_shared_pages(q, k, table, lists)
        held, listed = ints(lengths), lists.to(DEV)
        expected.append(paged.paged_attention(q, k, v, table, held, pages=listed))
        U.check_attention(expected[-1], q, k, v, table, lengths, pages=lists)
        for value in (float("nan"), float("inf"), 0.0):
            junk = torch.full((1 << 24,), value, device=DEV)
            del junk
            assert torch.equal(expected[-1], paged.paged_attention(q, k, v, table, held, pages=listed))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = paged.paged_attention(q, k, v, table, held, pages=listed)
            out = paged.paged_attention(out, k, v, table, held, pages=listed)
        graphs.append((graph, out, q, held, listed, paged.paged_attention(expected[-1], k, v, table, held, pages=listed)))
    for _ in range(3):
        for graph, out, *_, twice in graphs:
            out.fill_(float("nan"))
            graph.replay()
            assert torch.equal(out, twice)
    # two streams at once
    streams, outs = [torch.cuda.Stream() for _ in cases], [[], []]
    torch.cuda.synchronize()
    for _ in range(8):
        for i, (q, k, v, table, _, _) in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                outs[i].append(paged.paged_attention(q, k, v, table, graphs[i][3], pages=graphs[i][4]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, expected[i]) for o in outs[i])


def check_listed(got, q, k, v, table, lengths, lists):
    """As U.check_attention, for many rows: in 64 bits on the GPU, some rows at a time."""
    (rows, heads, dim), kv_heads, page = q.shape, k.size(1), k.size(2)
    group, width, slots = heads // kv_heads, table.size(1), torch.arange(k.size(2), device=DEV)
    count, heads_of = lists.size(2), torch.arange(kv_heads, device=DEV)[:, None]
    for at in range(0, rows, 64):
        some = slice(at, min(at + 64, rows))
        held = lengths[some].long().clamp(0, width * page)[:, None, None]
        pages, nth = (held + page - 1) // page, lists[some].long()
        real = (torch.arange(count, device=DEV) < pages) & (nth >= 0) & (nth < pages)
        nth = torch.where(real, nth, 0)
        where = table[some].long()[:, None].expand(-1, kv_heads, -1).gather(2, nth)
        real &= (where >= 0) & (where < k.size(0))
        where = torch.where(real, where, 0)
        seen = (real[..., None] & (nth[..., None] * page + slots < held[..., None])).flatten(2)  # [rows, kv_heads, positions]
        keys, values = (t[where, heads_of].flatten(2, 3).double().masked_fill(~seen[..., None], 0) for t in (k, v))
        mine = q[some].double().view(-1, kv_heads, group, dim)
        scores = torch.einsum("rhgd,rhsd->rhgs", mine, keys) * dim ** -0.5
        weights = torch.softmax(scores.masked_fill(~seen[:, :, None], -1e30), -1) * seen[:, :, None]
        ref = torch.einsum("rhgs,rhsd->rhgd", weights, values)
        size = torch.einsum("rhgd,rhsd->rhgs", mine.abs(), keys.abs()) * dim ** -0.5
        loss = weights * torch.expm1((2 * (dim + 3) * 2.0 ** -23 * size).clamp(max=30))
        bound = (torch.einsum("rhgs,rhsd->rhgd", loss, values.abs()) + loss.sum(-1, keepdim=True) * ref.abs()
                 + (2.0 ** -16 + count * page * 2.0 ** -23) * torch.einsum("rhgs,rhsd->rhgd", weights, values.abs()))
        bound = bound + U.unit(got.dtype) * (ref.abs() + bound) + torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
        assert ((got[some].double().view_as(ref) - ref).abs() <= bound).all(), at


@pytest.mark.parametrize("dtype", U.DTYPES)
@pytest.mark.parametrize("rows,heads,kv_heads,dim,page,total,width,count", [
    (4096, 1, 1, 128, 128, 4000, 32, 16),    # counters of more than 40 KB; more entries than a block takes in one turn
    (4096, 2, 1, 16, 256, 16384, 24, 16),    # the largest cache that is sorted
    (3000, 3, 3, 64, 128, 1100, 40, 24),     # two pages to a thread
    (1500, 6, 6, 40, 128, 2000, 33, 30),
    (8192, 1, 1, 64, 64, 900, 60, 40),       # more than 2^18 entries
])
def test_shared_pages_of_large_caches(rows, heads, kv_heads, dim, page, total, width, count, dtype):
    gen = torch.Generator(device=DEV).manual_seed(total)
    k, v = (torch.randn(total, kv_heads, page, dim, device=DEV, generator=gen).to(dtype) for _ in range(2))
    q = torch.randn(rows, heads, dim, device=DEV, generator=gen).to(dtype)
    table = torch.randint(0, total, (rows, width), device=DEV, generator=gen, dtype=torch.int32)
    lengths = torch.randint(0, width * page + 1, (rows,), device=DEV, generator=gen, dtype=torch.int32)
    lengths[:4] = ints([width * page, 0, 1, 2 ** 31 - 1])
    lists = torch.rand(rows, kv_heads, width, device=DEV, generator=gen).argsort(-1)[..., :count].int().contiguous()
    lists[5, :, 1], lists[6, 0, 0], lists[7] = lists[5, :, 0], -7, 2 ** 31 - 1
    table[8, ::2], table[9, ::3] = -1, total
    table[-1] = total - 1  # the last page
    assert takes_shared_pages(q, k, table, lists)
    got = paged.paged_attention(q, k, v, table, lengths, pages=lists)
    check_listed(got, q, k, v, table, lengths, lists)
    assert not got[1].any() and not got[7].any()


def test_attention_refuses_scales_that_are_not_finite_in_32_bits():
    q, k, v, table, held = case([50, 20], 4, 2, 64, 16, F16)
    for scale in (1e300, -1e39, float("nan")):
        with pytest.raises(RuntimeError):
            paged.paged_attention(q, k, v, table, held, scale=scale)


def test_attention_refuses_scales_whose_product_with_log2_e_overflows():
    q, k, v, table, held = case([50, 20], 4, 2, 64, 16, F16)
    for scale in (3e38, -3e38, 2.36e38):
        with pytest.raises(RuntimeError, match="scale"):
            paged.paged_attention(q, k, v, table, held, scale=scale)
    q[...] = 0.0  # scores of 0, whatever the scale
    for scale in (2.35e38, -2.35e38):
        U.check_attention(paged.paged_attention(q, k, v, table, held, scale=scale), q, k, v, table, [50, 20], scale=scale)


def test_attention_of_sequences_with_a_common_beginning():
    lengths = [100, 77, 64]
    q, k, v, table, held = case(lengths, 4, 2, 64, 16, F16)
    table[1, :3] = table[0, :3]
    table[2, :4] = table[0, :4]
    U.check_attention(paged.paged_attention(q, k, v, table, held), q, k, v, table, lengths)


def test_attention_does_not_depend_on_what_scratch_memory_held():
    for lengths, heads, kv_heads in (([3000, 200, 0, 1500], 16, 4), ([200] * 200, 8, 8), ([500], 32, 32)):
        q, k, v, table, held = case(lengths, heads, kv_heads, 128, 64, BF16)
        ref = paged.paged_attention(q, k, v, table, held)
        for value in (float("nan"), float("inf"), -1.0):
            junk = [torch.full((1 << 18,), value, device=DEV) for _ in range(24)]
            del junk
            assert torch.equal(paged.paged_attention(q, k, v, table, held), ref)


def test_operators_on_another_device_than_the_current_one():
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    lengths = [700, 90]
    q, k, v, table, held = case(lengths, 8, 2, 64, 32, F16)
    boxes = U.boxes_of(k, table, lengths, 32)
    one = paged.paged_attention(q, k, v, table, held), paged.paged_select(q, boxes, table, held, 32, 4)
    other = [t.to("cuda:1") for t in (q, k, v, table, held, boxes)]
    two = paged.paged_attention(*other[:5]), paged.paged_select(other[0], other[5], other[3], other[4], 32, 4)
    assert all(torch.equal(a, b.to(DEV)) for a, b in zip(one, two))
    with pytest.raises(RuntimeError):
        paged.paged_attention(q, *other[1:5])


def test_attention_refuses():
    q, k, v, table, held = case([50, 20], 4, 2, 64, 16, F16)
    def refused(q=q, k=k, v=v, table=table, held=held, **kwargs):
        with pytest.raises(RuntimeError):
            paged.paged_attention(q, k, v, table, held, **kwargs)
    refused(q=q.float())
    refused(q=q.bfloat16())
    refused(q=q[:, :3])
    refused(q=q[..., :32])
    refused(q=q[:1])
    refused(q=q[0])
    refused(q=q.clone().requires_grad_(True))
    refused(k=k.clone().requires_grad_(True))
    refused(k=k[:, :1])
    refused(k=k.transpose(2, 3).contiguous().transpose(2, 3))
    refused(k=k[:1].expand(k.shape))
    refused(v=v.bfloat16())
    refused(v=v[:1])
    refused(k=k[:, :, :8].contiguous(), v=v[:, :, :8].contiguous())
    refused(table=table.long())
    refused(table=table[:1])
    refused(table=torch.cat([table, table], 1)[:, ::2])
    refused(table=table.cpu())
    refused(held=held.long())
    refused(held=held.cpu())
    refused(scale=float("inf"))
    refused(pages=torch.zeros(2, 4, 3, dtype=torch.int32, device=DEV))
    refused(pages=torch.zeros(2, 2, 3, device=DEV))
    refused(pages=torch.zeros(2, 2, 3, dtype=torch.int32))
    with torch.no_grad():
        paged.paged_attention(q.clone().requires_grad_(True), k, v, table, held)


# ------------------------------------------------------------------------------------------------- selection

@pytest.mark.parametrize("dtype", U.DTYPES)
@pytest.mark.parametrize("lengths,heads,kv_heads,dim,page,count,first,last", [
    ([1000, 64, 65, 0, 1, 16], 8, 2, 128, 16, 4, 1, 1),
    ([4096, 3000], 6, 6, 80, 16, 33, 1, 1),
    ([5000], 16, 1, 64, 32, 1, 0, 0),
    ([5000], 16, 1, 64, 32, 1, 1, 0),
    ([700, 699], 5, 1, 8, 16, 40, 3, 5),
    ([2000, 100], 32, 32, 96, 64, 16, 8, 8),
    ([30000, 17], 4, 2, 32, 16, 200, 0, 2),
    ([70000], 4, 1, 128, 16, 64, 1, 1),
])
def test_selection(lengths, heads, kv_heads, dim, page, count, first, last, dtype):
    q, k, v, table, held = case(lengths, heads, kv_heads, dim, page, dtype)
    boxes = U.boxes_of(k, table, lengths, page)
    got = paged.paged_select(q, boxes, table, held, page, count, first, last)
    assert torch.equal(got.cpu(), U.select(q, boxes, table, lengths, page, count, first, last))


@pytest.mark.parametrize("rows,heads,kv_heads,dim,longest,count", [
    (300, 4, 1, 128, 40 * 16, 9),      # more blocks than two an SM
    (150, 6, 3, 64, 300 * 16, 33),
    (310, 1, 1, 24, 2500 * 16, 64),    # and more scores than leave room for six
    (9, 64, 32, 128, 70 * 16 + 1, 70),
])
def test_selection_of_many_rows_that_share_a_table(rows, heads, kv_heads, dim, longest, count):
    gen = torch.Generator().manual_seed(rows)
    pages = (longest + 15) // 16
    boxes = torch.randn(pages + 2, kv_heads, 2, dim, generator=gen).sort(2).values.half().to(DEV)
    table = (torch.randperm(pages + 2, generator=gen)[:pages].int().to(DEV)).expand(rows, -1).contiguous()
    q = torch.randn(rows, heads, dim, generator=gen).half().to(DEV)
    lengths = torch.randint(0, longest + 1, (rows,), generator=gen)
    lengths[0], lengths[1], lengths[2] = longest, 0, 1
    got = paged.paged_select(q, boxes, table, ints(lengths.tolist()), 16, count)
    # the same, row by row, and a few of them by definition
    for i in range(0, rows, 37):
        one = paged.paged_select(q[i:i + 1], boxes, table[i:i + 1], ints([int(lengths[i])]), 16, count)
        assert torch.equal(got[i:i + 1], one), i
    some = [0, 1, 2, rows - 1]
    assert torch.equal(got[some].cpu(), U.select(q[some], boxes, table[some], [int(lengths[i]) for i in some], 16, count, 1, 1))


def test_selection_of_equal_scores_takes_the_lower_pages():
    lengths = [1600, 1600, 333]
    q, k, v, table, held = case(lengths, 4, 2, 64, 16, F16)
    boxes = U.boxes_of(k, table, lengths, 16)
    q[0] = 0.0                      # all scores are zero
    boxes[...] = (torch.randn(boxes.shape, device=DEV) * 2).round()
    q[1] = (q[1] * 2).round()       # small whole numbers: many scores are equal
    boxes[table[1, :100].long(), 0, :, 1:] = 0.0
    got = paged.paged_select(q, boxes, table, held, 16, 20, 1, 1)
    assert torch.equal(got.cpu(), U.select(q, boxes, table, lengths, 16, 20, 1, 1))
    assert got[0, 0].tolist() == list(range(19)) + [99]


@pytest.mark.parametrize("same", (2, 3, 31, 32, 33, 70))
def test_selection_with_some_equal_scores_at_the_border(same):
    """Few pages with the score at the border are compared with one another, more of them all over again; a part of them in pairs
    that 32 bits do not tell apart."""
    pages, page, above = 200, 16, 9
    gen = torch.Generator().manual_seed(same)
    q, k, v, table, held = case([pages * page] * 4, 8, 2, 128, page, F16)
    boxes = U.boxes_of(k, table, [pages * page] * 4, page)
    q[...] = 1.0
    for i in range(4):
        order = torch.randperm(pages - 2, generator=gen)[:above + same] + 1
        own = table[i].long()
        boxes[own] = 0.0
        boxes[own[order[:above].to(DEV)], :, 1] = 2.0
        boxes[own[order[above:].to(DEV)], :, 1] = 1.0
        if i >= 2:  # every other one adds up to 2^-38 more, beside a sum of some 500
            boxes[own[order[above::2].to(DEV)], :, 1, 5] += 2.0 ** -10
            boxes[own[order[above::2].to(DEV)], :, 1, 6] -= 2.0 ** -10
            boxes[own[order[above + 1::2].to(DEV)], :, 0, 7] = -(2.0 ** -24)
            q[i, :, 7] = 0.5
            q[i, ::4, 7] = -2.0 ** -14
    for taken in (1, same // 2, same - 1, same):
        count = above + taken + 2
        got = paged.paged_select(q, boxes, table, held, page, count)
        assert torch.equal(got.cpu(), U.select(q, boxes, table, [pages * page] * 4, page, count, 1, 1)), taken


def test_selection_where_pages_are_not_the_caches():
    lengths = [900, 30, 0, 1600, 1500]
    q, k, v, table, held = case(lengths, 4, 2, 40, 16, F16)
    boxes = U.boxes_of(k, table, lengths, 16)
    table[0, 3:20], table[0, 20:23], table[3, 1::2] = -1, 2 ** 31 - 1, k.size(0)
    table[4] = -2 ** 31
    for first in (0.0, float("inf"), float("nan"), 65504.0):  # what the cache's first page has is nothing to them
        boxes[0] = first
        table[table == 0] = 1
        for count in (2, 7, 60, 95):
            got = paged.paged_select(q, boxes, table, held, 16, count)
            assert torch.equal(got.cpu(), U.select(q, boxes, table, lengths, 16, count, 1, 1)), (first, count)
    for count, first, last in ((2, 1, 1), (9, 0, 3), (20, 4, 0), (95, 1, 1)):
        got = paged.paged_select(q, boxes[:0], table, held, 16, count, first, last)
        assert torch.equal(got.cpu(), U.select(q, boxes[:0], table, lengths, 16, count, first, last)), count


def test_selection_tells_scores_apart_that_are_equal_in_32_bits():
    """Two pages whose scores differ by 2^-40 of their size."""
    q, k, v, table, held = case([160], 1, 1, 64, 16, BF16)
    boxes = torch.zeros(k.size(0), 1, 2, 64, dtype=BF16, device=DEV)
    q.zero_()
    q[0, 0, 0], q[0, 0, 1] = 1.0, 2.0 ** -40
    for j in range(10):
        boxes[int(table[0, j]), 0, 1, 0] = 1.0
    for j in (7, 4):
        boxes[int(table[0, j]), 0, 1, 1] = 1.0
    assert paged.paged_select(q, boxes, table, held, 16, 2, 0, 0)[0, 0].tolist() == [4, 7]


def test_selection_of_scores_that_are_not_finite():
    lengths = [1600]
    q, k, v, table, held = case(lengths, 4, 1, 64, 16, BF16)
    boxes = U.boxes_of(k, table, lengths, 16)
    boxes[int(table[0, 40]), 0, 1, 3] = float("nan")
    boxes[int(table[0, 50]), 0, 1, :] = float("inf")
    boxes[int(table[0, 60]), 0, :, :] = torch.finfo(BF16).max
    boxes[int(table[0, 70]), 0, 0, :] = float("-inf")
    table[0, 80], table[0, 81] = -1, 10 ** 6  # not the cache's: behind all others
    for count in (1, 2, 3, 4, 5, 97, 98, 99):
        got = paged.paged_select(q, boxes, table, held, 16, count, 0, 0)
        assert torch.equal(got.cpu(), U.select(q, boxes, table, lengths, 16, count, 0, 0)), count


@pytest.mark.parametrize("value", (float("nan"), float("inf"), float("-inf")))
@pytest.mark.parametrize("dim,rows", ((128, 3), (8, 3), (40, 320)))
def test_selection_with_more_infinite_scores_than_are_wanted(dim, rows, value):
    """The border lies among scores that are not numbers, the largest keys that there are, beside ones of any size."""
    gen = torch.Generator().manual_seed(dim)
    pages = 150
    boxes = torch.randn(pages, 1, 2, dim, generator=gen).sort(2).values.half()
    strange = torch.randperm(pages, generator=gen)[:60]
    boxes[strange, :, int(value != float("-inf")), 3] = value
    boxes = boxes.to(DEV)
    table = torch.stack([torch.randperm(pages, generator=gen) for _ in range(rows)]).int().to(DEV)
    q = torch.randn(rows, 2, dim, generator=gen).half().to(DEV)
    lengths = [pages * 16 - 5 * i for i in range(rows)]
    some = list(range(0, rows, 45))
    for count in (1, 2, 3, 7, 30, 61, 62, 63, 100):
        first = min(1, count - 1)
        got = paged.paged_select(q, boxes, table, ints(lengths), 16, count, first, 0)
        assert torch.equal(got[some].cpu(), U.select(q[some], boxes, table[some], [lengths[i] for i in some], 16, count, first, 0)), count


def test_selection_takes_a_page_with_a_key_that_overflowed():
    """An infinite element of a box makes NaN where no query head has a factor for it, and an infinite score where one has."""
    q, k, v, table, held = case([1600], 2, 1, 64, 16, F16)
    boxes = U.boxes_of(k, table, [1600], 16)
    q[...] = q.abs()            # of lo no element has a factor
    q[0, :, 5] = torch.tensor([1.0, -1.0], device=DEV).half()
    lower, upper = int(table[0, 37]), int(table[0, 61])
    boxes[lower, 0, 0, 9] = float("-inf")
    boxes[upper, 0, 0, 5] = float("-inf")
    for count, expected in ((1, [37]), (2, [37, 61])):
        assert paged.paged_select(q, boxes, table, held, 16, count, 0, 0)[0, 0].tolist() == expected
        assert U.select(q, boxes, table, [1600], 16, count, 0, 0)[0, 0].tolist() == expected


def test_selection_by_queries_that_are_not_finite():
    lengths = [1600] * 4
    q, k, v, table, held = case(lengths, 4, 2, 64, 16, F16)
    boxes = U.boxes_of(k, table, lengths, 16)
    q[0, 0, 3] = float("nan")
    q[1, 3, 5] = float("inf")
    q[2, 1, :] = float("-inf")
    q[3] *= 20000.0
    for count in (2, 9, 99):
        got = paged.paged_select(q, boxes, table, held, 16, count)
        assert torch.equal(got.cpu(), U.select(q, boxes, table, lengths, 16, count, 1, 1)), count


@pytest.mark.parametrize("dtype", U.DTYPES)
def test_selection_of_whole_numbers(dtype):
    """Scores that are often equal, of both signs, at random sizes: the border is in the middle of equal ones."""
    import random
    rng = random.Random(21)
    for turn in range(25):
        kv_heads, group, dim = rng.choice([1, 2, 5]), rng.choice([1, 3, 4, 9]), 8 * rng.randint(1, 16)
        lengths = [rng.randint(0, 6000) for _ in range(rng.randint(1, 4))]
        q, k, v, table, held = case(lengths, kv_heads * group, kv_heads, dim, 16, dtype, seed=turn)
        boxes = (U.boxes_of(k, table, lengths, 16) * rng.choice([1.0, 2.0])).round()
        q = (q * rng.choice([0.0, 1.0, 2.0])).round()
        count, first = rng.randint(2, 60), rng.randint(0, 1)
        last = rng.randint(0, count - first)
        got = paged.paged_select(q, boxes, table, held, 16, count, first, last)
        assert torch.equal(got.cpu(), U.select(q, boxes, table, lengths, 16, count, first, last)), turn


def test_selection_is_bounded_and_refuses():
    q, k, v, table, held = case([500, 200], 4, 2, 64, 16, F16)
    boxes = U.boxes_of(k, table, [500, 200], 16)
    wide = paged.paged_select(q, boxes, table, ints([2 ** 31 - 1, -3]), 16, 8)
    assert torch.equal(wide.cpu(), U.select(q, boxes, table, [2 ** 31 - 1, -3], 16, 8, 1, 1)) and (wide[1] == -1).all()
    assert paged.paged_select(q[:0], boxes, table[:0], held[:0], 16, 8).shape == (0, 2, 8)
    assert (paged.paged_select(q, boxes, table[:, :0].contiguous(), held, 16, 8) == -1).all()
    def refused(q=q, boxes=boxes, table=table, held=held, page=16, count=8, first=1, last=1):
        with pytest.raises(RuntimeError):
            paged.paged_select(q, boxes, table, held, page, count, first, last)
    refused(count=0)
    refused(count=1)
    refused(first=-1)
    refused(last=8)
    refused(first=2 ** 62, last=2 ** 62)
    refused(page=24)
    refused(boxes=boxes.bfloat16())
    refused(boxes=boxes[:, :, :1])
    refused(boxes=boxes[::2])
    refused(q=q.clone().requires_grad_(True))
    refused(table=torch.zeros(2, 20000, dtype=torch.int32, device=DEV))
    refused(held=held[:1])


def test_sizes_are_not_read_by_their_lower_32_bits():
    q, k, v, table, held = case([500, 200], 4, 2, 64, 16, F16)
    boxes = U.boxes_of(k, table, [500, 200], 16)
    for page in (2 ** 32 + 16, -2 ** 32 + 16, 2 ** 31 + 16):
        with pytest.raises(RuntimeError):
            paged.paged_select(q, boxes, table, held, page, 8)
    none = k.new_zeros(1).expand(0, 1, 2 ** 32 + 16, 64)  # a cache without pages, and q without rows
    with pytest.raises(RuntimeError):
        paged.paged_attention(q[:0], none, none, table[:0], held[:0])
    with pytest.raises(RuntimeError):
        paged.paged_attention(q.new_zeros(1).expand(0, 2 ** 32 + 2, 64), k, v, table[:0], held[:0])


# ------------------------------------------------------------------------------------------------- appending

APPENDS = [
    # lengths, new tokens, heads, kv_heads, dim, page, rotary, interleaved, rows behind the last sequence
    ([1], [1], 1, 1, 8, 16, 8, False, 0),
    ([5, 16, 17, 1, 33], [1, 1, 1, 1, 1], 4, 2, 64, 16, 64, False, 0),
    ([500, 64, 65], [500, 64, 3], 8, 2, 128, 64, 128, False, 0),
    ([100, 0, 40, 7], [37, 0, 40, 7], 6, 6, 80, 16, 48, True, 5),
    ([300, 301], [200, 1], 4, 1, 96, 32, 20, False, 1),
    ([90], [90], 10, 2, 40, 16, 6, True, 0),
    ([70, 256, 20], [33, 255, 20], 16, 1, 120, 256, 0, False, 70),
    ([2000], [1999], 5, 5, 128, 64, 128, True, 0),
]


@pytest.mark.parametrize("dtype", U.DTYPES)
@pytest.mark.parametrize("lengths,new,heads,kv_heads,dim,page,rotary,interleaved,padded", APPENDS)
def test_append(lengths, new, heads, kv_heads, dim, page, rotary, interleaved, padded, dtype):
    gen = torch.Generator().manual_seed(1)
    old = [a - b for a, b in zip(lengths, new)]
    k_cache, v_cache, table = U.make_cache(gen, lengths, kv_heads, dim, page, dtype, fill=0.0)
    boxes = U.boxes_of(k_cache, table, old, page)
    before = k_cache.clone(), v_cache.clone(), boxes.clone()
    tokens = sum(new) + padded
    fused = torch.randn(tokens, (heads + 2 * kv_heads) * dim, generator=gen).to(dtype).to(DEV)
    q = fused[:, :heads * dim].view(tokens, heads, dim)
    k = fused[:, heads * dim:(heads + kv_heads) * dim].view(tokens, kv_heads, dim)
    v = fused[:, (heads + kv_heads) * dim:].view(tokens, kv_heads, dim)
    cos, sin = paged.rope_table(max(lengths) + 3, rotary, device=DEV)
    cu = [sum(new[:i]) for i in range(len(new) + 1)]
    got = paged.paged_append(q, k, v, k_cache, v_cache, table, ints(lengths), ints(cu), rope=(cos, sin), interleaved=interleaved,
                             boxes=boxes)
    assert got.shape == q.shape and not got[cu[-1]:].any()
    for i in range(len(lengths)):
        if new[i] == 0:
            continue
        at = torch.arange(old[i], lengths[i], device=DEV)
        rows = slice(cu[i], cu[i + 1])
        U.check_turned(got[rows], q[rows], cos[at], sin[at], interleaved)
        to = table[i].long()[at // page]
        U.check_turned(k_cache[to, :, at % page], k[rows], cos[at], sin[at], interleaved)
        assert torch.equal(v_cache[to, :, at % page], v[rows])
        before[0][to, :, at % page] = k_cache[to, :, at % page]
        before[1][to, :, at % page] = v[rows]
    assert torch.equal(before[0], k_cache) and torch.equal(before[1], v_cache)  # all else is as it was
    assert torch.equal(boxes, U.boxes_of(k_cache, table, lengths, page))
    # without boxes, again: the same
    again = paged.paged_append(q, k, v, k_cache, v_cache, table, ints(lengths), ints(cu), rope=(cos, sin), interleaved=interleaved)
    assert torch.equal(again, got) and torch.equal(before[0], k_cache)


def test_append_with_angles_off_16_bytes():
    gen = torch.Generator().manual_seed(6)
    k_cache, v_cache, table = U.make_cache(gen, [40], 2, 64, 16, F16, fill=0.0)
    boxes = torch.zeros(k_cache.size(0), 2, 2, 64, dtype=F16, device=DEV)
    cos, sin = paged.rope_table(40, 64, device=DEV)
    room = torch.zeros(2 * 40 * 32 + 2, device=DEV)
    off = [room[1:1 + 40 * 32].view(40, 32), room[2 + 40 * 32:2 + 80 * 32].view(40, 32)]
    off[0].copy_(cos), off[1].copy_(sin)
    q, k, v = (torch.randn(40, h, 64, generator=gen).half().to(DEV) for h in (4, 2, 2))
    out = paged.paged_append(q, k, v, k_cache, v_cache, table, ints([40]), ints([0, 40]), rope=tuple(off), boxes=boxes)
    kept = k_cache.clone(), boxes.clone()
    ref = paged.paged_append(q, k, v, k_cache, v_cache, table, ints([40]), ints([0, 40]), rope=(cos, sin), boxes=boxes)
    assert torch.equal(out, ref) and torch.equal(kept[0], k_cache) and torch.equal(kept[1], boxes)


@pytest.mark.parametrize("dtype", U.DTYPES)
def test_append_without_rotation_copies_bits(dtype):
    gen = torch.Generator().manual_seed(1)
    k_cache, v_cache, table = U.make_cache(gen, [40, 16], 2, 64, 16, dtype, fill=0.0)
    q, k, v = (torch.randint(-2 ** 15, 2 ** 15, (2, h, 64), generator=gen, dtype=torch.int16).view(dtype).to(DEV) for h in (4, 2, 2))
    out = paged.paged_append(q, k, v, k_cache, v_cache, table, ints([40, 16]))
    bits = lambda t: t.view(torch.int16)
    assert torch.equal(bits(out), bits(q))
    for i, (place, slot) in enumerate([(2, 7), (0, 15)]):
        assert torch.equal(bits(k_cache[int(table[i, place]), :, slot].contiguous()), bits(k[i]))
        assert torch.equal(bits(v_cache[int(table[i, place]), :, slot].contiguous()), bits(v[i]))


def test_append_one_token_each_equals_ragged():
    gen = torch.Generator().manual_seed(2)
    lengths = [1, 0, 64, 65, 200]
    k_cache, v_cache, table = U.make_cache(gen, lengths, 2, 128, 64, F16, fill=0.0)
    rope = paged.rope_table(300, 128, device=DEV)
    q, k, v = (torch.randn(5, h, 128, generator=gen).half().to(DEV) for h in (8, 2, 2))
    a, b = [t.clone() for t in (k_cache, v_cache)], [t.clone() for t in (k_cache, v_cache)]
    one = paged.paged_append(q, k, v, *a, table, ints(lengths), rope=rope)
    two = paged.paged_append(q, k, v, *b, table, ints(lengths), ints([0, 1, 2, 3, 4, 5]), rope=rope)
    assert torch.equal(one, two) and torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert not one[1].any() and one[0].any()  # an idle sequence


def test_boxes_propagate_nan_and_begin_anew():
    gen = torch.Generator().manual_seed(3)
    k_cache, v_cache, table = U.make_cache(gen, [32], 1, 64, 16, BF16, fill=0.0)
    boxes = torch.full((k_cache.size(0), 1, 2, 64), 99.0, dtype=BF16, device=DEV)
    def put(length, value):
        x = torch.full((1, 1, 64), value, dtype=BF16, device=DEV)
        paged.paged_append(x, x, x, k_cache, v_cache, table, ints([length]), boxes=boxes)
        return boxes[int(table[0, (length - 1) // 16]), 0, :, 0].tolist()
    assert put(1, 2.0) == [2.0, 2.0]          # what was there before the page's first position does not count
    assert put(2, -1.0) == [-1.0, 2.0]
    assert put(3, 0.5) == [-1.0, 2.0]
    assert all(x != x for x in put(4, float("nan")))
    assert all(x != x for x in put(5, 1.0))
    assert put(17, 3.0) == [3.0, 3.0]
    assert put(1, 7.0) == [7.0, 7.0]


def test_boxes_of_a_sequence_that_was_cut_back():
    """What a box said before does not count, nor do keys behind the last new one."""
    gen = torch.Generator().manual_seed(3)
    k_cache, v_cache, table = U.make_cache(gen, [60], 2, 64, 32, F16, fill=0.0)
    boxes = torch.full((k_cache.size(0), 2, 2, 64), 99.0, dtype=F16, device=DEV)
    x = torch.randn(3, 2, 64, generator=gen).half().to(DEV)
    paged.paged_append(x, x, x, k_cache, v_cache, table, ints([41]), ints([0, 3]), boxes=boxes)
    ref = U.boxes_of(k_cache, table, [41], 32)
    assert torch.equal(boxes[int(table[0, 1])], ref[int(table[0, 1])]) and (boxes[int(table[0, 0])] == 99.0).all()


def test_append_drops_tokens_without_a_place():
    gen = torch.Generator().manual_seed(4)
    k_cache, v_cache, table = U.make_cache(gen, [64, 64, 64], 2, 64, 16, F16, spare=0, fill=0.0)
    rope = paged.rope_table(60, 64, device=DEV)
    table[1, 2] = -1
    table[2, 0] = k_cache.size(0)
    before = k_cache.clone(), v_cache.clone()
    boxes = U.boxes_of(k_cache, table[:1], [64], 16)
    kept = boxes.clone()
    q, k, v = (torch.randn(3 * 50, h, 64, generator=gen).half().to(DEV) for h in (2, 2, 2))
    # sequence 0: positions 14 .. 63, angles for 60; 1: a page is missing; 2: begins 20 positions in front of 0, first page missing
    out = paged.paged_append(q, k, v, k_cache, v_cache, table, ints([64, 64, 30]), ints([0, 50, 100, 150]), rope=rope, boxes=boxes)
    written = [(0, p) for p in range(14, 60)] + [(1, p) for p in range(14, 60) if not 32 <= p < 48] + [(2, p) for p in range(16, 30)]
    start = [14, 14, -20]
    rows = {50 * i + p - start[i] for i, p in written}
    for r in range(150):
        assert bool(out[r].any()) == (r in rows), r
    for i, p in written:
        before[0][int(table[i, p // 16]), :, p % 16] = k_cache[int(table[i, p // 16]), :, p % 16]
        before[1][int(table[i, p // 16]), :, p % 16] = v[50 * i + p - start[i]]
    assert torch.equal(before[0], k_cache) and torch.equal(before[1], v_cache)
    touched = {int(table[i, p // 16]) for i, p in written}
    rest = [p for p in range(k_cache.size(0)) if p not in touched]
    assert torch.equal(boxes[rest], kept[rest])
    # behind the table
    out = paged.paged_append(q[:1], k[:1], v[:1], k_cache, v_cache, table[:1], ints([65]))
    assert not out.any() and torch.equal(before[0], k_cache)
    out = paged.paged_append(q[:2], k[:2], v[:2], k_cache, v_cache, table[:2], ints([2 ** 31 - 1, -2 ** 31]))
    assert not out.any() and torch.equal(before[0], k_cache)
    # no sequences at all: nothing but rows behind the last one
    assert not paged.paged_append(q, k, v, k_cache, v_cache, table[:0], ints([]), ints([0])).any()
    assert paged.paged_append(q[:0], k[:0], v[:0], k_cache, v_cache, table[:0], ints([])).shape == (0, 2, 64)
    assert torch.equal(before[0], k_cache) and torch.equal(before[1], v_cache)


def test_lengths_below_zero_leave_no_place():
    gen = torch.Generator().manual_seed(5)
    k_cache, v_cache, table = U.make_cache(gen, [64, 64], 2, 64, 16, F16, spare=0, fill=0.0)
    before = k_cache.clone(), v_cache.clone()
    q, k, v = (torch.randn(6, 2, 64, generator=gen).half().to(DEV) for _ in range(3))
    for n, cu in ((2, None), (6, ints([0, 4, 6]))):
        for low in (-2 ** 31, -2 ** 31 + 3, -1, 0):
            junk = [torch.full_like(q[:n], float("nan")) for _ in range(4)]  # what the output's memory holds, most likely
            del junk
            out = paged.paged_append(q[:n], k[:n], v[:n], k_cache, v_cache, table, ints([low, low]), cu)
            assert torch.equal(out, torch.zeros_like(out)), (n, low)
            assert torch.equal(before[0], k_cache) and torch.equal(before[1], v_cache)


def test_append_refuses():
    gen = torch.Generator().manual_seed(5)
    k_cache, v_cache, table = U.make_cache(gen, [20, 20], 2, 64, 16, F16, fill=0.0)
    held, rope = ints([20, 20]), paged.rope_table(64, 64, device=DEV)
    q, k, v = (torch.randn(2, h, 64, generator=gen).half().to(DEV) for h in (4, 2, 2))
    boxes = U.boxes_of(k_cache, table, [20, 20], 16)
    def refused(q=q, k=k, v=v, k_cache=k_cache, v_cache=v_cache, table=table, held=held, cu=None, rope=rope, boxes=boxes):
        with pytest.raises(RuntimeError):
            paged.paged_append(q, k, v, k_cache, v_cache, table, held, cu, rope, False, boxes)
    refused(k=k[:1])
    refused(v=v[:, :1])
    refused(k=k.bfloat16())
    refused(q=q.clone().requires_grad_(True))
    refused(k_cache=k_cache.bfloat16(), v_cache=v_cache.bfloat16())
    refused(v_cache=v_cache[:1])
    refused(q=torch.cat([q, q]), k=torch.cat([k, k]), v=torch.cat([v, v]))
    refused(cu=ints([0, 1]))
    refused(cu=torch.tensor([0, 1, 2], device=DEV))
    refused(rope=(rope[0], rope[1][:, :5]))
    refused(rope=(rope[0].double(), rope[1].double()))
    refused(rope=paged.rope_table(64, 128, device=DEV))
    refused(rope=(rope[0], None))
    refused(boxes=boxes[:1])
    refused(boxes=boxes.bfloat16())
    refused(held=held[:1])
    version = k_cache._version
    paged.paged_append(q, k, v, k_cache, v_cache, table, held)
    assert k_cache._version > version


# -------------------------------------------------------------------------------------------------- together

def _decode(cache, rope, steps, heads, kv_heads, dim, table, start, gen, count=None):
    """`steps` decoding steps of a batch; the outputs, and q, k, v as they came."""
    outs, seen = [], []
    lengths = list(start)
    for _ in range(steps):
        lengths = [n + 1 for n in lengths]
        held = ints(lengths)
        q, k, v = (torch.randn(len(start), h, dim, generator=gen).to(cache.k.dtype).to(DEV) for h in (heads, kv_heads, kv_heads))
        turned = cache.append(q, k, v, table, held, rope=rope)
        out = cache.attend(turned, table, held) if count is None else cache.attend_selected(turned, table, held, count)
        outs.append(out)
        seen.append((turned, lengths))
    return outs, seen


@pytest.mark.parametrize("dtype", U.DTYPES)
def test_a_prompt_and_decoding_steps(dtype):
    """Prompts of uneven lengths appended at once, then tokens one by one, with full and with selected attention."""
    heads, kv_heads, dim, page = 8, 2, 64, 16
    gen = torch.Generator().manual_seed(7)
    cache = paged.PagedKVCache(64, kv_heads, dim, page, dtype, device=DEV)
    rope = paged.rope_table(512, dim, device=DEV)
    table = torch.randperm(60, generator=gen)[:48].reshape(3, 16).to(torch.int32).to(DEV)
    prompt = [130, 1, 47]
    q, k, v = (torch.randn(sum(prompt), h, dim, generator=gen).to(dtype).to(DEV) for h in (heads, kv_heads, kv_heads))
    turned = cache.append(q, k, v, table, ints(prompt), ints([0, 130, 131, 178]), rope=rope)
    # the prompt's own attention, causal: a row for each token
    rows_table = torch.cat([table[i:i + 1].expand(n, -1) for i, n in enumerate(prompt)]).contiguous()
    sees = [j + 1 for n in prompt for j in range(n)]
    U.check_attention(cache.attend(turned, rows_table, ints(sees)), turned, cache.k, cache.v, rows_table, sees)
    outs, seen = _decode(cache, rope, 20, heads, kv_heads, dim, table, prompt, gen)
    U.check_attention(outs[-1], seen[-1][0], cache.k, cache.v, table, seen[-1][1])
    assert torch.equal(cache.boxes[table[0, :9].long()], U.boxes_of(cache.k, table, seen[-1][1], page)[table[0, :9].long()])
    outs, seen = _decode(cache, rope, 3, heads, kv_heads, dim, table, seen[-1][1], gen, count=4)
    out, pages = outs[-1]
    assert torch.equal(pages.cpu(), U.select(seen[-1][0], cache.boxes, table, seen[-1][1], page, 4, 1, 1))
    U.check_attention(out, seen[-1][0], cache.k, cache.v, table, seen[-1][1], pages=pages)


def test_steps_captured_into_two_graphs_and_replayed_in_turn():
    heads, kv_heads, dim, page = 8, 2, 128, 64
    gen = torch.Generator().manual_seed(8)
    rope = paged.rope_table(2048, dim, device=DEV)
    sets = []
    for lengths in ([900, 30], [100, 1500]):
        k, v, table = U.make_cache(gen, [n + 10 for n in lengths], kv_heads, dim, page, F16, fill=0.0)
        boxes = U.boxes_of(k, table, [n + 10 for n in lengths], page)
        held = ints(lengths)
        x = [torch.randn(2, h, dim, generator=gen).half().to(DEV) for h in (heads, kv_heads, kv_heads)]
        def step(k=k, v=v, table=table, boxes=boxes, held=held, x=x):
            q = paged.paged_append(*x, k, v, table, held, rope=rope, boxes=boxes)
            pages = paged.paged_select(q, boxes, table, held, page, 4)
            return q, paged.paged_attention(q, k, v, table, held), paged.paged_attention(q, k, v, table, held, pages=pages), pages
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        sets.append((graph, outs, step, held, x))
    for turn in range(3):
        for graph, outs, step, held, x in sets:
            held += 1
            for t in x:
                t.mul_(-0.9)
            graph.replay()
        torch.cuda.synchronize()
        for graph, outs, step, held, x in sets:
            for a, b in zip(outs, step()):
                assert torch.equal(a, b)


def test_two_streams_at_once_and_another_than_the_tensors_own():
    q, k, v, table, held = case([3000, 200, 0, 1500], 16, 4, 128, 64, BF16)
    boxes = U.boxes_of(k, table, [3000, 200, 0, 1500], 64)
    ref = paged.paged_attention(q, k, v, table, held)
    ref_pages = paged.paged_select(q, boxes, table, held, 64, 5)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                got.append((paged.paged_attention(q, k, v, table, held), paged.paged_select(q, boxes, table, held, 64, 5)))
    torch.cuda.synchronize()
    for out, pages in got:
        assert torch.equal(out, ref) and torch.equal(pages, ref_pages)


def test_chained_calls_read_what_the_one_in_front_has_written():
    """Launches overlap: nothing is read before the kernel in front is done."""
    gen = torch.Generator().manual_seed(9)
    k, v, table = U.make_cache(gen, [4000] * 4, 4, 128, 64, F16, fill=0.0)
    boxes = U.boxes_of(k, table, [4000] * 4, 64)
    rope = paged.rope_table(4096, 128, device=DEV)
    xs = [[torch.randn(4, h, 128, generator=gen).half().to(DEV) for h in (16, 4, 4)] for _ in range(20)]
    def walk(sync):
        kk, vv, bb, held, outs = k.clone(), v.clone(), boxes.clone(), ints([3900] * 4), []
        for x in xs:
            torch.add(held, 1, out=held)
            for call in range(3):
                if call == 0:
                    q = paged.paged_append(*x, kk, vv, table, held, rope=rope, boxes=bb)
                elif call == 1:
                    pages = paged.paged_select(q, bb, table, held, 64, 6)
                else:
                    outs.append(paged.paged_attention(q, kk, vv, table, held, pages=pages))
                    outs.append(paged.paged_attention(q, kk, vv, table, held))
                if sync:
                    torch.cuda.synchronize()
        torch.cuda.synchronize()
        return outs
    for a, b in zip(walk(True), walk(False)):
        assert torch.equal(a, b)


def test_random_calls():
    import random
    rng = random.Random(11)
    for _ in range(60):
        kv_heads = rng.choice([1, 2, 3, 8])
        heads, dim, page, dtype = kv_heads * rng.choice([1, 2, 3, 4, 7, 8, 9, 16, 17]), 8 * rng.randint(1, 16), rng.choice([16, 32, 64, 128, 256]), rng.choice(U.DTYPES)
        lengths = [rng.choice([0, 1, rng.randint(1, 64), rng.randint(1, 1500)]) for _ in range(rng.randint(1, 9))]
        q, k, v, table, held = case(lengths, heads, kv_heads, dim, page, dtype, seed=rng.randint(0, 99))
        U.check_attention(paged.paged_attention(q, k, v, table, held), q, k, v, table, lengths)
        first, last = rng.randint(0, 2), rng.randint(0, 2)
        count = max(1, first + last) + rng.randint(0, 6)
        boxes = U.boxes_of(k, table, lengths, page)
        pages = paged.paged_select(q, boxes, table, held, page, count, first, last)
        assert torch.equal(pages.cpu(), U.select(q, boxes, table, lengths, page, count, first, last))
        U.check_attention(paged.paged_attention(q, k, v, table, held, pages=pages), q, k, v, table, lengths, pages=pages)
