"""What the paged cache promises at its edges (include/mlops_paged.h): rows of no request, values that are not finite in tokens that a row does not see,
counts that do not agree with each other, rings and tables with numbers that mean no page. Plain forms in tests/paged_util.py; attention's bounds as in
tests/test_gpu_paged.py."""
import math

import pytest
import torch

from tests import paged_util as pu
from tests.test_gpu_paged import TYPES, generator, ints, paged_case, starts_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def paged():
    from mlops_b200.attention import paged
    return paged


def attend_into_marked(paged, q, cache, table, lengths, starts):
    """the C call into outputs that hold 77 everywhere before it"""
    tokens, heads, _ = q.shape
    out, lse = torch.full_like(q, 77.0), torch.full((tokens, heads), 77.0, device="cuda")
    call = paged._ATTEND.pack(lengths.numel(), tokens, heads, paged._TYPES[q.dtype], q.data_ptr(), q.stride(0), q.stride(1), out.data_ptr(), out.stride(0), out.stride(1),
                              lse.data_ptr(), table.data_ptr(), table.shape[1], table.shape[1], lengths.data_ptr(), starts.data_ptr(), 0.0)
    scratch = torch.zeros(paged._lib.mlops_paged_attend_scratch_bytes(call, cache.units.shape[1]), dtype=torch.uint8, device="cuda")
    status = paged._lib.mlops_paged_attend(call, paged._pool(cache)[0], scratch.data_ptr(), scratch.numel(), torch.cuda.current_stream().cuda_stream)
    assert status == 0, paged._lib.mlops_paged_last_error()
    return out, lse


def agree(out, lse, want, name):
    """(out, lse) within attention's bounds of `want`, what pu.attend gives"""
    value, weight, log = want
    assert bool(((out.double() - value).abs() <= 2.0 ** -10 * weight + TYPES[name][1] * value.abs() + 1e-7).all())
    empty = torch.isinf(log)
    assert torch.equal(torch.isneginf(lse), empty) and bool((out[empty] == 0).all())
    assert bool(((lse.double() - log)[~empty].abs() <= 2.0 ** -12 * (1 + log[~empty].abs() / 8)).all())


@pytest.mark.parametrize("group, counts, skipped", [(4, [1, 1, 1, 1], 2), (4, [5, 0, 3, 7], 1), (2, [70, 3, 200, 1], 1), (8, [9, 40], 1), (1, [2, 3, 4], 3), (16, [1, 300], 1)])
def test_rows_before_the_first_request_are_cleared(paged, group, counts, skipped):
    """a slice of a step's requests with all of its rows: those of the requests before the slice are rows of no request (the fifth: no request is left)"""
    lengths, heads, pad = [400 + 33 * i for i in range(len(counts))], 2, 3
    gen, table, cache = paged_case(paged, sum(counts) + group, lengths, heads, 32)
    q = torch.randn((sum(counts) + pad, heads * group, 128), generator=gen, device="cuda").to(torch.bfloat16)
    first, end = sum(counts[:skipped]), sum(counts)
    table = table[skipped:].contiguous()
    out, lse = attend_into_marked(paged, q, cache, table, ints(lengths[skipped:]), starts_of(counts)[skipped:].contiguous())
    for rows in (slice(0, first), slice(end, None)):
        assert bool((out[rows] == 0).all()) and bool(torch.isneginf(lse[rows]).all())
    agree(out[first:end], lse[first:end], pu.attend(q[first:end], cache.units, cache.k_scale, cache.v_scale, table, lengths[skipped:], counts[skipped:]), "bf16")


def test_rows_before_a_first_request_behind_the_last_row(paged):
    """starts[0] above the rows of q: all of them are cleared, nothing beside them is written"""
    gen, table, cache = paged_case(paged, 2, [50], 1, 16)
    q = torch.randn((8, 4, 128), generator=gen, device="cuda").to(torch.float16)
    out, lse = attend_into_marked(paged, q[:5], cache, table, ints([50]), ints([1000, 1001]))
    assert bool((out == 0).all()) and bool(torch.isneginf(lse).all())


def with_bad_values(cache, table, b, bad):
    """NaN scales of V at (position, KV head, block of 16 channels, byte) of request b; a copy of the pool in which these blocks are zeros"""
    zeroed, P = cache.units.clone(), cache.page_size
    for position, head, block, byte in bad:
        page, at = int(table[b, position // P]), position % P
        for units, value in ((cache.units, byte), (zeroed, 0)):
            pu.fields(units)[3][page, head, at // 16, at % 16, block] = value
    return zeroed


def check_bad_values(paged, name, q, cache, table, lengths, counts, b, bad, starts):
    """NaN in the 16 channels of the rows that see them, all else as if these blocks were zeros"""
    zeroed = with_bad_values(cache, table, b, bad)
    heads, group = zeroed.shape[1], q.shape[1] // zeroed.shape[1]
    first = sum(counts[:b])
    limit = torch.arange(lengths[b] - counts[b], lengths[b], device="cuda")
    nan = torch.zeros(q.shape, dtype=torch.bool, device="cuda")
    for position, head, block, _ in bad:
        if int(table[b, position // cache.page_size]) in range(cache.pages):
            nan[first : first + counts[b], head * group : (head + 1) * group, 16 * block : 16 * block + 16] |= (limit >= position)[:, None, None]
    out, lse = paged.attend(q, cache, table, ints(lengths), starts, return_lse=True)
    assert torch.equal(out.isnan(), nan)
    value, weight, log = pu.attend(q, zeroed, cache.k_scale, cache.v_scale, table, lengths, counts)
    agree(torch.where(nan, value.to(out.dtype), out), lse, (value, weight, log), name)


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("group, length, n", [(4, 200, 1), (4, 200, 2), (1, 200, 30), (4, 200, 8), (3, 77, 5), (4, 200, 20), (2, 200, 64), (4, 200, 60), (4, 333, 333), (8, 3000, 700), (1, 260, 260)])
def test_not_a_number_in_v_stays_behind_the_causal_limit(paged, name, group, length, n):
    """both kernels, rows of work of all widths; tokens that no row, some rows and all rows see, and the request beside it"""
    lengths, counts, heads = [150, length, 90], [min(n, 3), n, 2 if n > 1 else 1], 2
    gen, table, cache = paged_case(paged, length + n, lengths, heads, 64)
    q = torch.randn((sum(counts), heads * group, 128), generator=gen, device="cuda").to(TYPES[name][0])
    bad = [(length - 1, 1, 4, 0x7F), (length - 1 - n // 2, 0, 0, 0xFF), (length - 1 - n // 3, 1, 7, 0x7F), (length - max(n - 1, 1), 1, 5, 0xFF)]
    if n < length:
        bad.append((3, 0, 6, 0x7F))
    check_bad_values(paged, name, q, cache, table, lengths, counts, 1, bad, starts_of(counts) if max(counts) > 1 else None)


@pytest.mark.parametrize("n", [2, 7, 30, 100])
def test_rows_that_see_nothing_beside_not_a_number_in_v(paged, n):
    """more queries than tokens: the first rows see nothing and are zeros, whatever the tokens hold"""
    lengths, counts = [1 + n // 3], [n]
    gen, table, cache = paged_case(paged, n, lengths, 2, 16)
    q = torch.randn((n, 8, 128), generator=gen, device="cuda").to(torch.bfloat16)
    check_bad_values(paged, "bf16", q, cache, table, lengths, counts, 0, [(p, h, (3 * p + h) % 8, 0x7F) for p in range(lengths[0]) for h in range(2)], starts_of(counts))


@pytest.mark.parametrize("n", [3, 20, 90])
def test_not_a_number_in_v_of_a_page_that_is_not_there(paged, n):
    lengths, counts = [300], [n]
    gen, table, cache = paged_case(paged, n, lengths, 2, 32)
    q = torch.randn((n, 8, 128), generator=gen, device="cuda").to(torch.bfloat16)
    whole = table.clone()
    table[0, 4] = -1
    with_bad_values(cache, whole, 0, [(4 * 32 + 5, 0, 2, 0x7F)])
    check_bad_values(paged, "bf16", q, cache, table, lengths, counts, 0, [(299, 0, 3, 0x7F)], starts_of(counts))


@pytest.mark.parametrize("size, head, tail", [(0, 0, 3), (0, 5, 1 << 40), (4, 0, 100), (4, 3, 8), (7, -5, 2), (7, -20, -9), (3, 9, 9), (3, 9, 4), (5, (1 << 62) + 1, (1 << 62) + 4)])
def test_rings_of_every_size_and_cursor(paged, size, head, tail):
    """a ring holds at most its size, none where it has no places or its ends are crossed; cursors are taken modulo the size, negative ones too"""
    P, held, added = 16, [0, 10, 40], [20, 30, 16]  # two, two and one new pages
    table, ring = [[-1] * 5, [90] + [-1] * 4, [91, 92, 93, -1, -1]], [10 + i for i in range(size)]
    left = min(max(tail - head, 0), size)
    want = [ring[(head + i) % size] if i < left else -1 for i in range(5)]
    device_table = ints(table)
    step = paged.assign(device_table, ints(held), ints(added), ints(ring), torch.tensor([head, tail], dtype=torch.int64, device="cuda"), P, sum(added))
    table[0][:2], table[1][1:3], table[2][3] = want[:2], want[2:4], want[4]
    assert device_table.tolist() == table and step.cursor.tolist() == [head + min(left, 5), tail, 5 - min(left, 5)]
    slots = [table[b][p // P] * P + p % P if table[b][p // P] >= 0 else -1 for b, (h, n) in enumerate(zip(held, added)) for p in range(h, h + n)]
    assert step.slots.tolist() == slots


def test_pages_and_positions_that_pass_31_bits(paged):
    """a page number whose slots lie behind 2^31 gives no slot (not another page's, modulo 2^32); positions and lengths end at 2^31 - 1"""
    P, last = 64, 2 ** 31 - 1
    table = ints([[1 << 27, -1, -1], [(1 << 25) - 1, -1, -1], [7, 8, 9], [1 << 25, -1, -1]])
    held, added = [3, 60, last - 4, 64], [2, 3, 8, 1]
    ring = ints([1 << 26])
    step = paged.assign(table, ints(held), ints(added), ring, torch.tensor([0, 1], dtype=torch.int64, device="cuda"), P, sum(added))
    positions = [3, 4, 60, 61, 62] + [last - 4 + i for i in range(5)] + [-1, -1, -1] + [64]
    assert step.positions.tolist() == positions
    assert step.slots.tolist() == [-1, -1] + [((1 << 25) - 1) * P + i for i in (60, 61, 62)] + [-1] * 8 + [-1]
    assert step.lengths.tolist() == [5, 63, last, 65] and step.starts.tolist() == [0, 2, 5, 13, 14]
    assert table[3].tolist() == [1 << 25, 1 << 26, -1] and step.cursor.tolist() == [1, 1, 1]


def assign_cut(table, held, added, ring, head, tail, P, tokens):
    """page assignment by loops for the first `tokens` new tokens; `missing` counts for all of them"""
    width, need = len(table[0]), sum(-(-(h + n) // P) - -(-h // P) for h, n in zip(held, added))
    table, slots, positions, starts, lengths, taken = [list(r) for r in table], [], [], [0], [], 0
    for b, (h, n) in enumerate(zip(held, added)):
        n = min(n, tokens - starts[-1])
        for p in range(h, h + n):
            column = p // P
            if p % P == 0 and column < width:
                table[b][column] = ring[(head + taken) % len(ring)] if head + taken < tail else -1
                taken += head + taken < tail
            page = table[b][column] if column < width else -1
            slots.append(page * P + p % P if page >= 0 else -1)
            positions.append(p)
        starts.append(starts[-1] + n)
        lengths.append(h + n)
    return table, slots, positions, starts, lengths, [head + taken, tail, need - taken]


@pytest.mark.parametrize("held, added, tokens, free", [
    ([5, 16, 0, 30], [40, 1, 100, 3], 100, 40), ([5, 16, 0, 30], [40, 1, 100, 3], 41, 40), ([5, 16, 0, 30], [40, 1, 100, 3], 40, 40), ([5, 16, 0, 30], [40, 1, 100, 3], 0, 40),
    ([5, 16, 0, 30], [40, 1, 100, 3], 143, 40), ([5, 16, 0, 30], [40, 1, 100, 3], 100, 4), ([0] * 300, [33] * 300, 4321, 2000), ([7], [500], 300, 40), ([16] * 40, [16] * 40, 16 * 20, 100)])
def test_fewer_rows_than_new_tokens(paged, held, added, tokens, free):
    """tokens without a row of the step are not added: no page is taken for them, lengths and starts say what was"""
    P, width, batch = 16, 12, len(held)
    table, taken = [[-1] * width for _ in held], 0
    for b in range(batch):
        for c in range(-(-held[b] // P)):
            table[b][c], taken = taken, taken + 1
    ring = [taken + i for i in range(free)]
    device_table = ints(table)
    step = paged.assign(device_table, ints(held), ints(added), ints(ring), torch.tensor([0, free], dtype=torch.int64, device="cuda"), P, tokens)
    for got, want in zip((device_table, *step), assign_cut(table, held, added, ring, 0, free, P, tokens)):
        assert got.tolist() == want


@pytest.mark.parametrize("group, counts, rows", [(4, [3, 6], 5), (4, [1, 1, 8], 3), (2, [10, 90], 60), (8, [200], 33), (1, [5, 5], 4), (4, [300, 7], 150), (4, [2, 3], 2)])
def test_fewer_rows_than_the_requests_have(paged, group, counts, rows):
    """rows that are left out at the end move no other row: each sees what it sees in the whole call"""
    lengths, heads = [500 + 41 * i for i in range(len(counts))], 2
    gen, table, cache = paged_case(paged, rows, lengths, heads, 32)
    q = torch.randn((sum(counts), heads * group, 128), generator=gen, device="cuda").to(torch.bfloat16)
    out, lse = paged.attend(q[:rows], cache, table, ints(lengths), starts_of(counts), return_lse=True)
    want = pu.attend(q, cache.units, cache.k_scale, cache.v_scale, table, lengths, counts)
    agree(out, lse, [x[:rows] for x in want], "bf16")


@pytest.mark.parametrize("which", [slice(0, 1), slice(1, 2)])
def test_one_token_of_rows_of_any_width(paged, which):
    """a dimension of one element has no stride that matters: one row of an array whose rows are no multiple of 8 elements apart, one head of it"""
    heads, group, P = 2, 2, 16
    gen, table, cache = paged_case(paged, 4, [40], heads, P)
    rows = torch.randn((3, 1028), generator=gen, device="cuda").to(torch.bfloat16)
    q, k, v = (rows[:, at : at + n * 128].view(3, n, 128)[which] for at, n in ((0, heads * group), (512, heads), (768, heads)))
    assert q.stride(0) % 8 and q.is_contiguous()
    slots = (table[:, 2] * P + 7).to(torch.int32)
    other = paged.PagedCache(cache.units.clone(), cache.k_scale, cache.v_scale)
    paged.append(cache, k, v, slots)
    paged.append(other, *(torch.empty(x.shape, dtype=x.dtype, device="cuda").copy_(x) for x in (k, v)), slots)
    assert torch.equal(cache.units, other.units)
    out, lse = paged.attend(q, cache, table, ints([40]), return_lse=True)
    agree(out, lse, pu.attend(q, cache.units, cache.k_scale, cache.v_scale, table, [40], [1]), "bf16")
    # (one head: strides of heads that are no multiple of 8)
    one = rows.as_strided((2, 1, 128), (128, 1028, 1), which.start * 1028)
    pair = table.repeat(2, 1)
    single = paged.PagedCache(cache.units[:, :1], cache.k_scale[:1], cache.v_scale[:1])
    out, lse = paged.attend(one, single, pair, ints([40, 33]), return_lse=True)
    agree(out, lse, pu.attend(one, single.units, single.k_scale, single.v_scale, pair, [40, 33], [1, 1]), "bf16")


@pytest.mark.parametrize("counts", [[1], [6], [200]])
@pytest.mark.parametrize("at", [5, 39000])
def test_one_score_far_above_a_long_context(paged, counts, at):
    """Weights 2^-32 to 2^-24 of the largest, over 40 000 tokens, with V that is 0 in half of the channels of the loud token: these hold what the small weights leave.
    A weight P is held with its largest at 2^9 or more; in FP16 it is off by 2^-11 of itself, below 2^-14 by 2^-25, which is 2^-34 of the largest. So an element is off by
    at most 2^-10 sum p |v| / sum p (the bound of the other tests) and 2^-34 max |v| per token that is seen."""
    length, heads, group, P = 40000, 2, 4, 64
    gen, table, cache = paged_case(paged, 17, [length], heads, P)
    height = 6.0 * torch.rand((length, heads), generator=gen, device="cuda")
    height[at] = 24.0
    k = (height[..., None] * torch.ones(128, device="cuda")).to(torch.bfloat16)
    v = (1.0 + torch.rand((length, heads, 128), generator=gen, device="cuda")).to(torch.bfloat16)
    v[at, :, :64] = 0.0
    position = torch.arange(length, device="cuda")
    paged.append(cache, k, v, (table[0, position // P].long() * P + position % P).to(torch.int32))
    q = torch.ones((counts[0], heads * group, 128), dtype=torch.bfloat16, device="cuda")
    scale = 32.0 * math.log(2.0) / (24.0 * 128.0)
    out, lse = paged.attend(q, cache, table, ints([length]), starts_of(counts), scale=scale, return_lse=True)
    want, weight, want_lse = pu.attend(q, cache.units, cache.k_scale, cache.v_scale, table, [length], counts, scale)
    assert bool(((out.double() - want).abs() <= 2.0 ** -10 * weight + length * 2.0 ** -34 * 2.5 + TYPES["bf16"][1] * want.abs()).all())
    assert float(want[..., :64].min()) > 2.0 ** -16 and bool(((lse.double() - want_lse).abs() <= 2.0 ** -12 * (1 + want_lse.abs() / 8)).all())


@pytest.mark.parametrize("name", ["attend", "cross_attend", "attend_shared"])
def test_a_length_at_the_end_of_its_type(paged, name):
    """2^31 - 1 tokens, which a row of the table could name (`assign` ends there): those whose pages there are are seen"""
    from tests.test_gpu_paged import factors
    P, width, heads = 2048, 1 << 20, 1
    gen = generator(41)
    cache = paged.PagedCache(pu.random_units(gen, 3, heads, P), *factors(gen, heads))
    table = torch.full((2, width), -1, dtype=torch.int32, device="cuda")
    table[0, :2], table[1, 0] = ints([2, 0]), 1
    q = torch.randn((2, 4, 128), generator=gen, device="cuda").to(torch.bfloat16)
    more = (None, None, ints([0])) if name == "attend_shared" else (None,)
    out, lse = getattr(paged, name)(q, cache, table, ints([(1 << 31) - 1, 700]), *more, return_lse=True)
    agree(out, lse, pu.attend(q, cache.units, cache.k_scale, cache.v_scale, table[:, :2], [2 * P, 700], [1, 1]), "bf16")
