"""The paged 4-bit cache on the GPU against plain implementations (tests/paged_util.py): bytes and whole numbers equal, attention within what its
roundings allow.

Attention's bound, element by element: the weights p are rounded to 16 bits once (relative 2^-11), scores are FP32 sums of exact products (their error,
at most 2^-12 here, moves p by as much), so the sum is off by at most 2^-10 of sum p |v| / sum p; the output's own rounding adds 2^-8 (BF16) or 2^-11
(FP16) of the value. The log-sum-exp carries the scores' error alone."""
import math
import random

import pytest
import torch

from tests import paged_util as pu

pytestmark = pytest.mark.gpu
TYPES = {"bf16": (torch.bfloat16, 2.0 ** -8), "fp16": (torch.float16, 2.0 ** -11)}


@pytest.fixture(scope="module")
def paged():
    from mlops_b200.attention import paged
    return paged


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def factors(gen, heads):
    return torch.exp2(torch.randint(-2, 3, (heads,), generator=gen, device="cuda").float()), 0.05 + torch.rand((heads,), generator=gen, device="cuda")


# ---- append and read ---------------------------------------------------------------------------------------------------------
def check_append(paged, k, v, units, k_scale, v_scale, slots):
    cache = paged.PagedCache(units, k_scale, v_scale)
    before = units.clone()
    assert paged.append(cache, k, v, slots) is cache
    stored = [(f.cpu(), x) for f, x in zip(pu.at_slots(units, slots.clamp(min=0)), sum(zip(pu.quantise(k, k_scale), pu.quantise(v, v_scale)), ()))]
    # (K codes, V codes, K scales, V scales)
    there = (slots >= 0).cpu()
    for got, want in stored:
        assert torch.equal(got[there], want[there])
    P = units.shape[2] * 16
    rest = torch.ones(units.shape[0] * P, dtype=torch.bool, device="cuda")
    rest[slots[slots >= 0].long()] = False
    rest = rest.nonzero().view(-1).to(torch.int32)
    for got, want in zip(pu.at_slots(units, rest), pu.at_slots(before, rest)):
        assert torch.equal(got, want)  # nothing else was written


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("tokens, heads, page_size", [(1, 1, 16), (3, 8, 64), (257, 2, 32), (1000, 5, 48), (4097, 8, 256)])
def test_append_is_the_plain_quantiser(paged, name, tokens, heads, page_size):
    gen = generator(tokens + heads)
    pages = -(-tokens // page_size) + 2
    units = torch.full((pages, heads, page_size // 16, 2304), 0xA5, dtype=torch.uint8, device="cuda")
    k_scale, v_scale = factors(gen, heads)
    slots = torch.randperm(pages * page_size, generator=gen, device="cuda")[:tokens].to(torch.int32)
    if tokens > 2:
        slots[tokens // 2] = -1
    # slices of a fused projection; the blocks' sizes spread over the scales' whole range and beyond
    rows = torch.randn((tokens, 2 * heads + 3, 8, 16), generator=gen, device="cuda") * torch.exp2(torch.randint(-16, 13, (tokens, 2 * heads + 3, 8, 1), generator=gen, device="cuda").float())
    rows = rows.flatten(-2).clamp(-60000, 60000).to(TYPES[name][0])
    check_append(paged, rows[:, 3 : 3 + heads], rows[:, 3 + heads :], units, k_scale, v_scale, slots)


@pytest.mark.parametrize("name", ["bf16", "fp16"])
def test_append_halfway_cases_and_values_that_are_not_finite(paged, name):
    dtype = TYPES[name][0]
    levels = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 0.0, -0.0, 0.5, -0.25, -0.75, -5.0, 1e-3, -1e-3]
    rows = [[x * s for x in levels] for s in (1.0, 0.875, 0.013671875, 448.0, 1.75, 2.0 ** -9)]
    rows += [[0.0] * 16, [-0.0] * 16, [math.inf] + [1.0] * 15, [1.0] * 15 + [math.nan], [-math.inf, math.nan] + [0.5] * 14, [60000.0] * 16, [2.0 ** -14] * 16, [2.0 ** -12] * 16]
    # scales halfway between two E4M3 numbers: amax / 6 = 17/16, 19/16 ... of a power of two
    rows += [[6 * m / 16 * 2.0 ** e] + [0.1] * 15 for m in (17, 19, 21, 23, 25, 27, 29, 31) for e in (-5, 0, 3)]
    while len(rows) % 8:
        rows.append([1.0] * 16)
    x = torch.tensor(rows, dtype=torch.float32, device="cuda").to(dtype).view(-1, 1, 128)
    units = torch.zeros((2, 1, 1, 2304), dtype=torch.uint8, device="cuda")
    one = torch.ones(1, device="cuda")
    check_append(paged, x, x.flip(0).contiguous(), units, one, one, torch.arange(3, 3 + x.shape[0], dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("tokens, heads, page_size", [(1, 1, 16), (70, 3, 48), (3001, 8, 64)])
def test_read_rounds_the_stored_values_once(paged, name, tokens, heads, page_size):
    gen = generator(tokens)
    pages = tokens // page_size + 3
    units = pu.random_units(gen, pages, heads, page_size)
    units[0, :, :, 2048:] = torch.randint(0, 256, units[0, :, :, 2048:].shape, generator=gen, device="cuda", dtype=torch.uint8)  # (every scale, NaN too)
    k_scale, v_scale = factors(gen, heads)
    slots = torch.randint(0, pages * page_size, (tokens,), generator=gen, device="cuda").to(torch.int32)
    if tokens > 2:
        slots[1], slots[2] = -1, pages * page_size
    there = (slots >= 0) & (slots < pages * page_size)
    got = paged.read(paged.PagedCache(units, k_scale, v_scale), slots, TYPES[name][0])
    kc, vc, ks, vs = pu.at_slots(units, torch.where(there, slots, 0))
    for x, codes, scales, factor in ((got[0], kc, ks, k_scale), (got[1], vc, vs, v_scale)):
        want = pu.values(codes, scales, 1.0).float() * factor[:, None]  # code * scale is exact in FP32, its product with the factor rounded once
        want = torch.where(there[:, None, None], want, 0.0).to(TYPES[name][0])
        assert torch.equal(x.isnan(), want.isnan()) and torch.equal(x.nan_to_num(0.0), want.nan_to_num(0.0))


# ---- assign ---------------------------------------------------------------------------------------------------------------------
def assign_by_loops(table, held, added, ring, head, tail, P, tokens):
    table = [list(r) for r in table]
    slots, positions, starts, missing = [], [], [0], 0
    for b, (h, n) in enumerate(zip(held, added)):
        for c in range(-(-h // P), -(-(h + n) // P)):
            page = -1
            if c >= len(table[b]):
                missing += 1
                continue
            if head < tail:
                page = ring[head % len(ring)]
                head += 1
            else:
                missing += 1
            table[b][c] = page
        for p in range(h, h + n):
            page = table[b][p // P] if p // P < len(table[b]) else -1
            positions.append(p)
            slots.append(page * P + p % P if page >= 0 else -1)
        starts.append(starts[-1] + n)
    pad = tokens - len(slots)
    return table, (slots + [-1] * pad)[:tokens], (positions + [-1] * pad)[:tokens], starts, [h + n for h, n in zip(held, added)], [head, tail, missing]


@pytest.mark.parametrize("batch, held_hi, new_hi, P, free, narrow, pad", [
    (1, 0, 1, 16, 5, False, 0), (1, 100, 700, 32, 400, False, 5), (3, 65, 0, 16, 4, False, 2), (64, 5000, 1, 64, 80, False, 0), (255, 300, 40, 16, 2000, False, 0),
    (257, 300, 40, 48, 2000, False, 77), (700, 60, 3, 16, 100, False, 0), (40, 200, 100, 16, 60, True, 9), (2500, 900, 2, 128, 4000, False, 0), (9000, 20, 1, 16, 4000, False, 1)])
def test_assign_is_the_loop_over_requests(paged, batch, held_hi, new_hi, P, free, narrow, pad):
    rng = random.Random(batch)
    held, added = [rng.randint(0, held_hi) for _ in range(batch)], [rng.randint(0, new_hi) for _ in range(batch)]
    width = max(1, -(-(held_hi + new_hi) // P)) - (3 if narrow else 0)
    table, taken = [[-1] * width for _ in range(batch)], 0
    for b in range(batch):
        for c in range(min(width, -(-held[b] // P))):
            table[b][c], taken = taken, taken + 1
    size = free + 11
    head = (1 << 33) + size - min(3, free)  # (counted without end; the free pages wrap around the ring's end)
    ring = [-7] * size
    for i in range(free):
        ring[(head + i) % size] = taken + i
    tokens = sum(added) + pad
    device_table = torch.full((batch, width + 2), -9, dtype=torch.int32, device="cuda")[:, :width]  # (rows inside a wider array)
    device_table.copy_(ints(table))
    step = paged.assign(device_table, ints(held), ints(added), ints(ring), torch.tensor([head, head + free], dtype=torch.int64, device="cuda"), P, tokens)
    want = assign_by_loops(table, held, added, ring, head, head + free, P, tokens)
    for got, expected in zip((device_table, *step), want):
        assert got.tolist() == expected


def test_assign_steps_follow_each_other_in_a_graph(paged):
    """lengths and cursor of a step are the next one's; a captured step is replayed with the lengths it finds"""
    P, batch, steps = 16, 5, 40
    table, held, cursor = torch.full((batch, 8), -1, dtype=torch.int32, device="cuda"), ints([0, 3, 16, 31, 50]), torch.tensor([0, 60, 0], dtype=torch.int64, device="cuda")
    ring, added = ints(list(range(60))), ints([1] * batch)
    table[1, 0], table[2, 0], table[3, :2], table[4, :4] = 59, 58, ints([57, 56]), ints([55, 54, 53, 52])
    plain_table, plain_held, plain_head = table.tolist(), held.tolist(), 0
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step = paged.assign(table, held, added, ring, cursor, P, batch)
            held.copy_(step.lengths)
            cursor.copy_(step.cursor)
        for _ in range(steps):
            graph.replay()
            plain_table, slots, positions, _, plain_held, moved = assign_by_loops(plain_table, plain_held, [1] * batch, ring.tolist(), plain_head, 60, P, batch)
            plain_head = moved[0]
            assert step.slots.tolist() == slots and step.positions.tolist() == positions and table.tolist() == plain_table and cursor.tolist() == moved


# ---- attend ---------------------------------------------------------------------------------------------------------------------
def check_attend(paged, q, cache, table, lengths, counts, starts, name, scale=0.0, rows=None):
    out, lse = paged.attend(q, cache, table, ints(lengths), starts, scale=scale, return_lse=True)
    assert torch.equal(out, paged.attend(q, cache, table, ints(lengths), starts, scale=scale))  # (and twice the same)
    want, weight, want_lse = pu.attend(q, cache.units, cache.k_scale, cache.v_scale, table, lengths, counts, scale or None)
    bound = 2.0 ** -10 * weight + TYPES[name][1] * want.abs() + 1e-7
    off = (out.double() - want).abs()
    assert bool((off <= bound).all()), f"off by up to {(off / bound).max().item():.2f} of the bound"
    empty = torch.isinf(want_lse)
    assert torch.equal(torch.isinf(lse), empty) and bool((out[empty] == 0).all())
    assert bool(((lse.double() - want_lse)[~empty].abs() <= 2.0 ** -12 * (1 + want_lse[~empty].abs() / 8)).all())


def paged_case(paged, seed, lengths, heads, page_size, width=None):
    gen = generator(seed)
    table, pages = pu.tables(gen, lengths, page_size, width=width)
    units = pu.random_units(gen, pages, heads, page_size)
    pu.spoil_behind(units, table, lengths)
    return gen, table, paged.PagedCache(units, *factors(gen, heads))


def starts_of(counts):
    s = [0]
    for n in counts:
        s.append(s[-1] + n)
    return ints(s)


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("heads, group, page_size, lengths", [
    (1, 1, 16, [1]), (2, 1, 16, [0, 1, 2, 15, 16, 17, 33]), (8, 4, 64, [5000]), (8, 2, 64, [4096]), (4, 3, 48, [700, 0, 1, 64]), (2, 7, 32, [129, 31, 300]), (1, 16, 128, [1000, 77]),
    (3, 8, 16, [0, 0, 513]), (2, 24, 16, [40, 41]), (8, 4, 64, [0, 0]), (1, 5, 256, [20000]), (8, 4, 64, [300 + 37 * i for i in range(70)]), (2, 2, 64, [1 + 7 * i % 90 for i in range(300)])])
def test_decode(paged, name, heads, group, page_size, lengths):
    gen, table, cache = paged_case(paged, len(lengths) + heads, lengths, heads, page_size)
    q = torch.randn((len(lengths), heads * group, 128), generator=gen, device="cuda").to(TYPES[name][0])
    check_attend(paged, q, cache, table, lengths, [1] * len(lengths), None, name)


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("heads, group, page_size, lengths, counts", [
    (2, 4, 64, [300, 17, 900], [2, 3, 8]), (4, 1, 16, [50, 60, 70, 80], [5, 0, 1, 9]), (1, 2, 32, [100], [100]), (2, 4, 64, [129, 128, 127, 1], [129, 128, 127, 1]),
    (2, 3, 48, [1000, 555], [400, 33]), (1, 16, 64, [3000, 64], [70, 64]), (8, 4, 64, [2000, 1, 700, 300], [1, 1, 640, 5]), (1, 8, 128, [5000], [17]), (2, 5, 16, [260, 2000], [260, 31]),
    (2, 4, 64, [3, 0, 10], [7, 4, 40]), (1, 1, 16, [1500], [1500])])
def test_several_queries_per_request(paged, name, heads, group, page_size, lengths, counts):
    """chunks of prompts, drafted tokens, whole prompts; the last-but-one: more queries than tokens, whose first rows see nothing"""
    gen, table, cache = paged_case(paged, sum(counts), lengths, heads, page_size)
    q = torch.randn((sum(counts), heads * group, 128), generator=gen, device="cuda").to(TYPES[name][0])
    check_attend(paged, q, cache, table, lengths, counts, starts_of(counts), name)


@pytest.mark.parametrize("counts", [[1], [6], [200]])
@pytest.mark.parametrize("order", ["rising", "falling", "one", "flat"])
def test_scores_of_every_order(paged, order, counts):
    """scores that grow or fall along the sequence by hundreds, one that is far above the others, all the same"""
    lengths, heads, group, P = [1777], 2, 4, 64
    gen, table, cache = paged_case(paged, 3, lengths, heads, P)
    position = torch.arange(1777, device="cuda")
    height = {"rising": position / 100.0, "falling": (1777 - position) / 100.0, "one": torch.where(position == 900, 25.0, 0.02), "flat": torch.full((1777,), 0.5, device="cuda")}[order]
    k = (height[:, None, None] * torch.ones((1, heads, 128), device="cuda")).to(torch.bfloat16)
    v = torch.randn((1777, heads, 128), generator=gen, device="cuda").to(torch.bfloat16)
    slots = (table[0, position // P].long() * P + position % P).to(torch.int32)
    paged.append(cache, k, v, slots)
    q = (torch.rand((counts[0], heads * group, 128), generator=gen, device="cuda") + 0.5).to(torch.bfloat16)
    check_attend(paged, q, cache, table, lengths, counts, starts_of(counts), "bf16", scale=0.05)


def test_queries_of_every_size(paged):
    """rows of zeros, of numbers near the ends of the type's range, with a few large channels"""
    for name, tiny, huge in (("bf16", 1e-37, 1e30), ("fp16", 6e-8, 6e4)):
        gen, table, cache = paged_case(paged, 9, [300, 300, 300, 300], 2, 32)
        q = torch.randn((4, 8, 128), generator=gen, device="cuda")
        q[0], q[1] = 0.0, q[1].sign() * tiny
        q[2] *= huge / 1e4
        q[3, :, :3] *= 1000
        # (scores so large that FP32 sums of them are off by more than the bound of p are one-hot: the scale brings them down)
        check_attend(paged, q[[0, 1]].to(TYPES[name][0]), cache, table[:2], [300] * 2, [1] * 2, None, name)
        check_attend(paged, q[[2]].to(TYPES[name][0]), cache, table[:1], [300], [1], None, name, scale=1e4 / huge / 12)
        check_attend(paged, q[[3]].to(TYPES[name][0]), cache, table[:1], [300], [1], None, name, scale=1e-3)


@pytest.mark.parametrize("counts", [[1, 1, 1], [3, 1, 2], [150, 90, 1]])
def test_pages_that_are_not_there(paged, counts):
    """tokens of table entries outside the pool are not seen; a length beyond the table's width is cut"""
    lengths, P = [500, 333, 4 * 64 + 9], 64
    gen, table, cache = paged_case(paged, 5, [500, 333, 4 * 64], 2, P, width=8)
    table = table.clone()
    table[0, 2], table[0, 7], table[1, 5], table[1, 0] = -1, cache.pages, 1 << 30, -(1 << 31)
    table[2] = -1
    table[2, 3] = 0
    table = torch.cat((table, torch.full_like(table, 12345)), 1)[:, :8]
    q = torch.randn((sum(counts), 8, 128), generator=gen, device="cuda").to(torch.bfloat16)
    plain = torch.where((table >= 0) & (table < cache.pages), table, -1)
    lengths[2] = 8 * 64 + 100
    cache.units[0, :, :, 2048:] = 56
    out, lse = paged.attend(q, cache, table, ints(lengths), starts_of(counts), return_lse=True)
    want, weight, want_lse = pu.attend(q, cache.units, cache.k_scale, cache.v_scale, plain, lengths, counts)
    assert bool(((out.double() - want).abs() <= 2.0 ** -10 * weight + 2.0 ** -8 * want.abs() + 1e-7).all())
    assert torch.equal(torch.isinf(lse), torch.isinf(want_lse))


@pytest.mark.parametrize("counts", [[1, 1], [4, 3], [130, 77]])
def test_strides_rows_of_no_request_and_another_stream(paged, counts):
    """a pool that is one layer of a larger one, queries inside a fused projection's rows, rows behind the last request, a stream of its own"""
    lengths, heads, group, P, pad = [700, 222], 4, 4, 32, 5
    gen = generator(11)
    table, pages = pu.tables(gen, lengths, P)
    everything = pu.random_units(gen, pages * 3, heads + 1, P).view(pages, 3, heads + 1, P // 16, 2304)
    units = everything[:, 1, :heads]
    pu.spoil_behind(units, table, lengths)
    cache = paged.PagedCache(units, *factors(gen, heads))
    rows = torch.randn((sum(counts) + pad, heads * group + 7, 128), generator=gen, device="cuda").to(torch.bfloat16)
    q = rows[:, 3 : 3 + heads * group]
    wide = torch.cat((table, table), 1)[:, : table.shape[1]]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        out, lse = paged.attend(q, cache, wide, ints(lengths), starts_of(counts), return_lse=True)
        assert bool((out[sum(counts) :] == 0).all()) and bool(torch.isneginf(lse[sum(counts) :]).all())
        check_attend(paged, q[: sum(counts)], cache, wide, lengths, counts, starts_of(counts), "bf16")


@pytest.mark.parametrize("counts", [[1], [5], [140]])
def test_a_pool_of_more_than_4_gib(paged, counts):
    """pages far beyond 2^32 bytes from the pool's start"""
    heads, P, lengths = 8, 64, [500]
    big = torch.zeros((4, (5 << 30) // 4), dtype=torch.uint8, device="cuda")
    unit = P // 16 * 2304
    units = big.as_strided((4, heads, P // 16, 2304), (big.stride(0), unit, 2304, 1))
    gen = generator(12)
    small = pu.random_units(gen, 4, heads, P)
    units.copy_(small)
    # eight pages' tokens in four pages: the last ones twice
    table = ints([[3, 1, 2, 3, 0, 3, 2, 3]])
    cache = paged.PagedCache(units, *factors(gen, heads))
    q = torch.randn((counts[0], heads * 4, 128), generator=gen, device="cuda").to(torch.bfloat16)
    check_attend(paged, q, cache, table, lengths, counts, starts_of(counts), "bf16")
    k = torch.randn((3, heads, 128), generator=gen, device="cuda").to(torch.bfloat16)
    slots = ints([3 * P + 1, 3 * P + 63, 2 * P])
    paged.append(cache, k, k, slots)
    for got, (codes, scales) in zip((0, 1), (pu.quantise(k, cache.k_scale), pu.quantise(k, cache.v_scale))):
        stored = pu.at_slots(units, slots)
        assert torch.equal(stored[got].cpu(), codes) and torch.equal(stored[2 + got].cpu(), scales)


def test_not_a_number_is_not_hidden(paged):
    """a token with NaN in K makes the rows that see it NaN, and no others"""
    lengths, counts = [200], [60]
    gen, table, cache = paged_case(paged, 13, lengths, 2, 64)
    k = torch.randn((1, 2, 128), generator=gen, device="cuda").to(torch.bfloat16)
    bad = k.clone()
    bad[0, 1, 77] = math.nan
    paged.append(cache, bad, k, (table[0, 2] * 64 + 180 - 128).view(1).to(torch.int32))
    q = torch.randn((60, 4, 128), generator=gen, device="cuda").to(torch.bfloat16)
    for n in (60, 3, 1):
        out = paged.attend(q[:n], cache, table, ints(lengths), starts_of([n]))
        sees = torch.arange(200 - n, 200, device="cuda") >= 180
        assert torch.equal(out.isnan().all(-1)[:, 2:], sees[:, None].expand(-1, 2)) and not bool(out[:, :2].isnan().any())


def test_a_step_from_pages_to_attention(paged):
    """assign, append and attend as an engine runs them, against the same tokens kept densely"""
    heads, group, P, batch = 4, 2, 16, 3
    gen = generator(14)
    cache = paged.empty(40, heads, P, v_scale=torch.full((heads,), 0.25))
    table, lengths, cursor = torch.full((batch, 12), -1, dtype=torch.int32, device="cuda"), ints([0] * batch), torch.tensor([0, 40], dtype=torch.int64, device="cuda")
    ring = torch.randperm(40, generator=gen, device="cuda").to(torch.int32)
    kept = [[] for _ in range(batch)]
    for added in ([37, 0, 5], [1, 20, 1], [1, 1, 1], [4, 60, 0], [1, 1, 1]):
        n = sum(added)
        rows = torch.randn((n, heads * group + 2 * heads, 128), generator=gen, device="cuda").to(torch.bfloat16)
        q, k, v = rows.split([heads * group, heads, heads], 1)
        step = paged.assign(table, lengths, ints(added), ring, cursor, P, n)
        paged.append(cache, k, v, step.slots)
        out, lse = paged.attend(q, cache, table, step.lengths, step.starts, return_lse=True)
        lengths, cursor = step.lengths, step.cursor
        (kc, ks), (vc, vs) = pu.quantise(k, cache.k_scale), pu.quantise(v, cache.v_scale)
        kd, vd = pu.values(kc, ks, 1.0).cuda(), pu.values(vc, vs, 0.25).cuda()
        first = 0
        for b, m in enumerate(added):
            kept[b] += [(kd[first + i], vd[first + i]) for i in range(m)]
            for i in range(m):
                seen = kept[b][: len(kept[b]) - m + i + 1]
                for x in range(heads * group):
                    keys, vals = (torch.stack([t[j][x // group] for t in seen]) for j in (0, 1))
                    s = keys @ q[first + i, x].double() / math.sqrt(128)
                    p = (s - torch.logsumexp(s, 0)).exp()
                    bound = 2.0 ** -10 * (p @ vals.abs()) + 2.0 ** -8 * (p @ vals).abs() + 1e-7
                    assert bool(((out[first + i, x].double() - p @ vals).abs() <= bound).all())
            first += m
    assert cursor.tolist()[2] == 0


@pytest.mark.parametrize("heads, group, counts", [(2, 4, [8, 9, 1, 2]), (1, 8, [4, 5, 1]), (1, 16, [2, 3]), (1, 32, [1, 2]), (1, 40, [1, 1]), (4, 1, [31, 32, 33, 8]), (1, 33, [1])])
def test_on_both_sides_of_the_kernels_limits(paged, heads, group, counts):
    """8, 16, 32 columns and one more; groups that are streamed with and without `starts`"""
    lengths = [1200 + 77 * i for i in range(len(counts))]
    gen, table, cache = paged_case(paged, sum(counts) + group, lengths, heads, 32)
    q = torch.randn((sum(counts), heads * group, 128), generator=gen, device="cuda").to(torch.bfloat16)
    check_attend(paged, q, cache, table, lengths, counts, starts_of(counts), "bf16")
    if max(counts) == 1:
        check_attend(paged, q, cache, table, lengths, counts, None, "bf16")


@pytest.mark.parametrize("heads, group, counts", [(2, 4, [1] * 20 + [8, 9, 3]), (3, 8, [1, 1, 1, 0]), (2, 2, [4, 4]), (2, 2, [4, 5]), (1, 1, [1, 0, 30, 2, 7, 0, 1])])
def test_on_both_sides_of_the_average(paged, heads, group, counts):
    """up to 8 columns per request on average and more, with single requests of more than that"""
    lengths = [900 + 131 * i for i in range(len(counts))]
    gen, table, cache = paged_case(paged, sum(counts) + group, lengths, heads, 16)
    q = torch.randn((sum(counts), heads * group, 128), generator=gen, device="cuda").to(torch.float16)
    check_attend(paged, q, cache, table, lengths, counts, starts_of(counts), "fp16")


def test_long_runs_of_tiles(paged):
    """some seventy tiles of tokens per CTA, rows of work of one tile to fifty"""
    lengths, counts = [6144], [6144]
    gen, table, cache = paged_case(paged, 21, lengths, 2, 64)
    q = torch.randn((6144, 16, 128), generator=gen, device="cuda").to(torch.bfloat16)
    check_attend(paged, q, cache, table, lengths, counts, starts_of(counts), "bf16")


def test_calls_of_all_shapes_one_after_the_other(paged):
    """sixty calls on one stream without a wait between them, from one query to whole prompts: each leaves the scratch as the next one needs it"""
    rng, shapes = random.Random(5), []
    for i in range(12):
        batch = rng.randint(1, 9)
        counts = [rng.choice([1, 1, 2, 7, 40, 300]) for _ in range(batch)] if i % 3 else [1] * batch
        shapes.append(([n + rng.randint(0, 4000) for n in counts], counts, rng.choice([1, 2, 8]), rng.choice([1, 4, 6])))
    calls = []
    for seed, (lengths, counts, heads, group) in enumerate(shapes):
        gen, table, cache = paged_case(paged, 100 + seed, lengths, heads, 64)
        q = torch.randn((sum(counts), heads * group, 128), generator=gen, device="cuda").to(torch.bfloat16)
        calls.append((q, cache, table, ints(lengths), None if max(counts) == 1 else starts_of(counts)))
    torch.cuda.synchronize()
    results = [paged.attend(*c, return_lse=True) for _ in range(5) for c in calls]
    for i, (out, lse) in enumerate(results[12:]):
        assert torch.equal(out, results[i % 12][0]) and torch.equal(lse, results[i % 12][1])
    for (q, cache, table, lengths, _), (_, counts, _, _), (out, lse) in zip(calls, shapes, results):
        want, weight, want_lse = pu.attend(q, cache.units, cache.k_scale, cache.v_scale, table, lengths.tolist(), counts)
        assert bool(((out.double() - want).abs() <= 2.0 ** -10 * weight + 2.0 ** -8 * want.abs() + 1e-7).all())
        assert bool(((lse.double() - want_lse).abs() <= 2.0 ** -12 * (1 + want_lse.abs() / 8)).all())


def test_a_captured_step_follows_lengths_and_tables(paged):
    """append and attention captured once, replayed for a growing request: the tables, lengths and slots of the moment count; two streams at once"""
    heads, group, P, width = 2, 4, 16, 40
    gen = generator(31)
    table = torch.randperm(width, generator=gen, device="cuda").to(torch.int32).view(1, width)
    caches = [paged.empty(width, heads, P) for _ in range(2)]
    k, v, q = (torch.zeros((1, n, 128), dtype=torch.bfloat16, device="cuda") for n in (heads, heads, heads * group))
    slots, lengths = ints([0]), ints([1])
    streams, graphs, outs = [torch.cuda.Stream() for _ in range(2)], [], []
    for stream, cache in zip(streams, caches):
        with torch.cuda.stream(stream):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                paged.append(cache, k, v, slots)
                outs.append(paged.attend(q, cache, table, lengths))
            graphs.append(graph)
    torch.cuda.synchronize()
    for step in range(70):
        for x in (k, v, q):
            x.copy_(torch.randn(x.shape, generator=gen, device="cuda"))
        slots.copy_(table[0, step // P] * P + step % P)
        lengths.fill_(step + 1)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[1]) and torch.equal(caches[0].units, caches[1].units)
        if step % 23 == 0 or step == 69:
            want, weight, _ = pu.attend(q, caches[0].units, caches[0].k_scale, caches[0].v_scale, table, [step + 1], [1])
            assert bool(((outs[0].double() - want).abs() <= 2.0 ** -10 * weight + 2.0 ** -8 * want.abs() + 1e-7).all())


def test_the_serving_example(paged):
    """examples/paged_serving.py: lengths and finite outputs, the same again for the same numbers"""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "paged_serving.py")
    spec = importlib.util.spec_from_file_location("paged_serving", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    lengths, out, _ = example.serve(requests=3, steps=70, prompt=200)
    assert lengths == [1 + 200 * (i + 1) // 3 + 70 for i in range(3)] and bool(torch.isfinite(out).all())
    assert torch.equal(out, example.serve(requests=3, steps=70, prompt=200)[1])
