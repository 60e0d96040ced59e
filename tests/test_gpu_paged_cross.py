"""cross_attend against attention in 64 bits in which every query sees all of its request's tokens. Bounds as in tests/test_gpu_paged.py."""
import math

import pytest
import torch

from tests import paged_util as pu
from tests.test_gpu_paged import TYPES, factors, generator, ints, paged_case, starts_of
from tests.test_gpu_paged_edges import agree, with_bad_values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def paged():
    from mlops_b200.attention import paged
    return paged


def plain(q, units, k_scale, v_scale, table, lengths, counts, scale=None):
    """(out, weight, lse) in 64 bits, as pu.attend gives them"""
    parts, first = [[x[:0] for x in whole(q[:0], units, k_scale, v_scale, table[0], 0, scale)]], 0
    for b, n in enumerate(counts):
        parts.append(whole(q[first : first + n], units, k_scale, v_scale, table[b], lengths[b], scale))
        first += n
    return [torch.cat(x) for x in zip(*parts)]


def whole(q, units, k_scale, v_scale, entries, length, scale):
    """all rows of q see all of `length` tokens"""
    H, P = units.shape[1], units.shape[2] * 16
    group, n = q.shape[1] // H, min(length, entries.numel() * P)
    out, weight = (torch.zeros(q.shape, dtype=torch.float64, device="cuda") for _ in range(2))
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    if n <= 0:
        return out, weight, lse
    kc, vc, ks, vs = pu.fields(units)
    page = entries[: -(-n // P)].long()
    there = (page >= 0).repeat_interleave(P)[:n]
    page = page.clamp(min=0)
    for h in range(H):
        k, v = (torch.where(there[:, None], pu.values(c[page, h].reshape(-1, 64)[:n], s[page, h].reshape(-1, 8)[:n], g[h].double()), 0.0) for c, s, g in ((kc, ks, k_scale), (vc, vs, v_scale)))
        for x in range(h * group, (h + 1) * group):
            s = (q[:, x].double() @ k.T * (1 / math.sqrt(128) if scale is None else scale)).masked_fill(~there, -math.inf)
            lse[:, x] = torch.logsumexp(s, -1)
            p = torch.where(there, (s - lse[:, x, None]).exp(), 0.0)
            out[:, x], weight[:, x] = p @ v, p @ v.abs()
    return out, weight, lse


def check(paged, q, cache, table, lengths, counts, starts, name, scale=0.0):
    out, lse = paged.cross_attend(q, cache, table, ints(lengths), starts, scale=scale, return_lse=True)
    assert torch.equal(out, paged.cross_attend(q, cache, table, ints(lengths), starts, scale=scale))
    agree(out, lse, plain(q, cache.units, cache.k_scale, cache.v_scale, table, lengths, counts, scale or None), name)


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("heads, group, page_size, lengths", [
    (1, 1, 16, [1]), (2, 1, 16, [0, 1, 2, 15, 16, 17, 33]), (16, 1, 64, [1500]), (4, 3, 48, [700, 0, 1, 64]), (1, 16, 128, [1000, 77]), (2, 24, 16, [40, 41]), (8, 4, 64, [0, 0]),
    (1, 40, 32, [300, 5]), (8, 2, 64, [300 + 37 * i for i in range(40)]), (2, 2, 64, [1 + 7 * i % 90 for i in range(300)])])
def test_one_query_per_request(paged, name, heads, group, page_size, lengths):
    gen, table, cache = paged_case(paged, len(lengths) + heads, lengths, heads, page_size)
    q = torch.randn((len(lengths), heads * group, 128), generator=gen, device="cuda").to(TYPES[name][0])
    check(paged, q, cache, table, lengths, [1] * len(lengths), None, name)


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("heads, group, page_size, lengths, counts", [
    (2, 4, 64, [300, 17, 900], [2, 3, 8]), (4, 1, 16, [50, 60, 70, 80], [5, 0, 1, 9]), (1, 2, 32, [3], [100]), (2, 4, 64, [1, 128, 127, 129], [129, 128, 127, 1]), (2, 3, 48, [1000, 0], [400, 33]),
    (1, 16, 64, [3000, 64], [70, 64]), (8, 4, 64, [2000, 1, 700, 300], [1, 1, 640, 5]), (2, 2, 32, [1999, 300, 0, 512], [5, 5, 5, 5]), (1, 1, 16, [257], [1500]), (2, 4, 64, [700], [8]), (2, 4, 64, [700], [9])])
def test_several_queries_per_request(paged, name, heads, group, page_size, lengths, counts):
    """target texts, beams, more queries than states, no states"""
    gen, table, cache = paged_case(paged, sum(counts), lengths, heads, page_size)
    q = torch.randn((sum(counts), heads * group, 128), generator=gen, device="cuda").to(TYPES[name][0])
    check(paged, q, cache, table, lengths, counts, starts_of(counts), name)


@pytest.mark.parametrize("counts", [[1, 1, 1], [3, 1, 2], [150, 90, 1]])
def test_pages_that_are_not_there(paged, counts):
    """states of table entries outside the pool are not seen; a length beyond the table's width is cut"""
    lengths, P = [500, 333, 8 * 64 + 100], 64
    gen, table, cache = paged_case(paged, 5, [500, 333, 4 * 64], 2, P, width=8)
    table = table.clone()
    table[0, 2], table[0, 7], table[1, 5], table[1, 0] = -1, cache.pages, 1 << 30, -(1 << 31)
    table[2] = -1
    table[2, 3] = 0
    q = torch.randn((sum(counts), 8, 128), generator=gen, device="cuda").to(torch.bfloat16)
    cache.units[0, :, :, 2048:] = 56
    out, lse = paged.cross_attend(q, cache, table, ints(lengths), starts_of(counts), return_lse=True)
    agree(out, lse, plain(q, cache.units, cache.k_scale, cache.v_scale, torch.where((table >= 0) & (table < cache.pages), table, -1), lengths, counts), "bf16")


@pytest.mark.parametrize("group, counts", [(4, [2, 1, 3]), (2, [1, 9, 2]), (4, [1, 70, 20]), (1, [300, 1, 260])])
def test_not_a_number_in_v_and_in_k(paged, group, counts):
    """a state with a NaN block of V makes these 16 channels NaN in all rows of its request and KV head, one with NaN in K the rows; other requests are not touched"""
    lengths, heads = [150, 333, 90], 2
    gen, table, cache = paged_case(paged, sum(counts), lengths, heads, 64)
    q = torch.randn((sum(counts), heads * group, 128), generator=gen, device="cuda").to(torch.bfloat16)
    zeroed = with_bad_values(cache, table, 1, [(0, 1, 4, 0x7F), (332, 0, 0, 0xFF), (200, 1, 7, 0x7F)])
    nan = torch.zeros(q.shape, dtype=torch.bool, device="cuda")
    rows = slice(counts[0], counts[0] + counts[1])
    nan[rows, group:, 64:80] = nan[rows, group:, 112:] = nan[rows, :group, :16] = True
    out, lse = paged.cross_attend(q, cache, table, ints(lengths), starts_of(counts), return_lse=True)
    assert torch.equal(out.isnan(), nan)
    value, weight, log = plain(q, zeroed, cache.k_scale, cache.v_scale, table, lengths, counts)
    agree(torch.where(nan, value.to(out.dtype), out), lse, (value, weight, log), "bf16")
    pu.fields(cache.units)[2][int(table[2, 0]), 1, 2, 5, 3] = 0x7F
    out = paged.cross_attend(q, cache, table, ints(lengths), starts_of(counts))
    nan[counts[0] + counts[1] :, group:] = True
    assert torch.equal(out.isnan(), nan)


@pytest.mark.parametrize("counts, pad", [([1, 1], 0), ([4, 3], 5), ([130, 77], 5)])
def test_strides_rows_of_no_request_and_another_stream(paged, counts, pad):
    lengths, heads, group, P = [700, 222], 4, 4, 32
    gen = generator(11)
    table, pages = pu.tables(gen, lengths, P)
    units = pu.random_units(gen, pages * 3, heads + 1, P).view(pages, 3, heads + 1, P // 16, 2304)[:, 1, :heads]
    pu.spoil_behind(units, table, lengths)
    cache = paged.PagedCache(units, *factors(gen, heads))
    q = torch.randn((sum(counts) + pad, heads * group + 7, 128), generator=gen, device="cuda").to(torch.bfloat16)[:, 3 : 3 + heads * group]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        out, lse = paged.cross_attend(q, cache, table, ints(lengths), starts_of(counts), return_lse=True)
        assert bool((out[sum(counts) :] == 0).all()) and bool(torch.isneginf(lse[sum(counts) :]).all())
        check(paged, q[: sum(counts)], cache, table, lengths, counts, starts_of(counts), "bf16", scale=0.05)


def test_a_slice_of_the_requests(paged):
    """rows of the requests before the slice are cleared; rows that q does not have move no other"""
    lengths, counts = [300, 40, 500], [4, 90, 2]
    gen, table, cache = paged_case(paged, 6, lengths, 2, 32)
    q = torch.randn((sum(counts), 8, 128), generator=gen, device="cuda").to(torch.bfloat16)
    want = plain(q, cache.units, cache.k_scale, cache.v_scale, table, lengths, counts)
    out, lse = paged.cross_attend(q, cache, table[1:], ints(lengths)[1:], starts_of(counts)[1:], return_lse=True)
    assert bool((out[:4] == 0).all()) and bool(torch.isneginf(lse[:4]).all())
    agree(out[4:], lse[4:], [x[4:] for x in want], "bf16")
    out, lse = paged.cross_attend(q[:50], cache, table, ints(lengths), starts_of(counts), return_lse=True)
    agree(out, lse, [x[:50] for x in want], "bf16")


def test_a_captured_call_follows_lengths(paged):
    lengths, counts = [300, 40, 500], [5, 5, 5]
    gen, table, cache = paged_case(paged, 8, [500, 500, 500], 2, 32)
    q, held, starts = torch.randn((15, 8, 128), generator=gen, device="cuda").to(torch.bfloat16), ints(lengths), starts_of(counts)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out, lse = paged.cross_attend(q, cache, table, held, starts, return_lse=True)
        for lengths in ([300, 40, 500], [0, 1, 2], [500, 499, 17]):
            held.copy_(ints(lengths))
            graph.replay()
            agree(out, lse, plain(q, cache.units, cache.k_scale, cache.v_scale, table, lengths, counts), "bf16")
