"""attend_shared against causal attention in 64 bits of each request by itself (tests/paged_util.py). Bounds as in tests/test_gpu_paged.py: the two parts of a row are joined in FP32."""
import math
import random

import pytest
import torch

from tests import paged_util as pu
from tests.test_gpu_paged import TYPES, factors, generator, ints, starts_of
from tests.test_gpu_paged_edges import agree, with_bad_values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def paged():
    from mlops_b200.attention import paged
    return paged


def build(paged, seed, groups, lengths, heads, P, width=None, layers=1):
    """groups: (first request, end, common tokens). A table whose rows of a group name the same pages for the whole pages of these tokens (as far as a request reaches), the
    pool behind it, what no request uses spoilt"""
    gen = generator(seed)
    own = list(lengths)
    for first, end, common in groups:
        for b in range(first, end):
            own[b] = max(lengths[b] - common // P * P, 0)
    whole = [c // P for _, _, c in groups]
    table, pages = pu.tables(gen, own, P, spare=3 + sum(whole), width=width or max([-(-n // P) for n in lengths] + [1]))
    taken = set(table[table >= 0].tolist())
    rest = [p for p in torch.randperm(pages, generator=gen, device="cuda").tolist() if p not in taken]
    for (first, end, common), n in zip(groups, whole):
        pages_of, rest = rest[:n], rest[n:]
        for b in range(first, end):
            m = min(n, -(-lengths[b] // P))
            mine = table[b].clone()
            table[b] = -1
            table[b, :m] = ints(pages_of[:m])
            k = -(-own[b] // P)
            table[b, n : n + k] = mine[:k]
    units = pu.random_units(gen, pages, heads, P)
    pu.spoil_behind(units, table, lengths)
    return gen, table, paged.PagedCache(units, *factors(gen, heads))


def group_args(groups):
    cuts = [groups[0][0]] + [e for _, e, _ in groups]
    assert all(a[1] == b[0] for a, b in zip(groups, groups[1:]))
    return ints(cuts), ints([c for _, _, c in groups])


def check(paged, q, cache, table, lengths, counts, starts, groups, name, scale=0.0):
    cuts, common = group_args(groups)
    out, lse = paged.attend_shared(q, cache, table, ints(lengths), starts, cuts, common, scale=scale, return_lse=True)
    assert torch.equal(out, paged.attend_shared(q, cache, table, ints(lengths), starts, cuts, common, scale=scale))
    if len(groups) == 1 and groups[0][:2] == (0, len(lengths)):
        assert torch.equal(out, paged.attend_shared(q, cache, table, ints(lengths), starts, None, common, scale=scale))
    agree(out, lse, pu.attend(q, cache.units, cache.k_scale, cache.v_scale, table, lengths, counts, scale or None), name)
    return out


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("heads, group, P, groups, lengths", [
    (1, 1, 16, [(0, 2, 16)], [17, 18]), (2, 4, 64, [(0, 8, 640)], [700 + 13 * i for i in range(8)]), (2, 1, 16, [(0, 3, 40)], [41, 60, 48]), (8, 4, 64, [(0, 40, 2000)], [2001 + 7 * i for i in range(40)]),
    (2, 4, 32, [(0, 3, 500), (3, 4, 300), (4, 9, 64)], [501, 600, 777, 400, 65, 70, 66, 200, 90]), (1, 16, 128, [(0, 2, 3000)], [3100, 3333]), (1, 40, 16, [(0, 3, 100)], [101, 150, 120]),
    (2, 3, 48, [(1, 4, 200)], [90, 201, 230, 250, 40, 1]), (2, 4, 64, [(0, 5, 0), (5, 9, 63)], [1, 2, 3, 4, 5, 64, 65, 70, 300]), (4, 2, 16, [(0, 200, 333)], [340 + i % 50 for i in range(200)]),
    (1, 5, 256, [(0, 6, 20000)], [20001 + 300 * i for i in range(6)]), (2, 8, 16, [(0, 1, 50)], [77])])
def test_decode(paged, name, heads, group, P, groups, lengths):
    gen, table, cache = build(paged, len(lengths) + heads, groups, lengths, heads, P)
    q = torch.randn((len(lengths), heads * group, 128), generator=gen, device="cuda").to(TYPES[name][0])
    check(paged, q, cache, table, lengths, [1] * len(lengths), None, groups, name)


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("heads, group, P, groups, lengths, counts", [
    (2, 4, 64, [(0, 3, 300)], [320, 333, 900], [2, 3, 8]), (4, 1, 16, [(0, 4, 64)], [70, 80, 90, 100], [5, 0, 1, 9]), (1, 2, 32, [(0, 2, 100)], [230, 260], [100, 5]),
    (2, 4, 64, [(0, 4, 128)], [257, 256, 255, 129], [129, 128, 127, 1]), (2, 3, 48, [(0, 2, 555)], [1000, 600], [400, 33]), (8, 4, 64, [(0, 2, 130), (2, 4, 64)], [2000, 150, 700, 300], [1, 1, 636, 5]),
    (1, 1, 16, [(0, 2, 1500)], [3100, 1600], [1600, 100]), (1, 1, 16, [(0, 8, 48)], [49 + i for i in range(8)], [1] * 8), (2, 4, 16, [(0, 3, 1000)], [1030, 1010, 1300], [0, 0, 4]),
    (1, 8, 128, [(0, 2, 5000), (2, 3, 100)], [5017, 5100, 300], [17, 2, 40])])
def test_several_queries_per_request(paged, name, heads, group, P, groups, lengths, counts):
    gen, table, cache = build(paged, sum(counts), groups, lengths, heads, P)
    q = torch.randn((sum(counts), heads * group, 128), generator=gen, device="cuda").to(TYPES[name][0])
    check(paged, q, cache, table, lengths, counts, starts_of(counts), groups, name)


@pytest.mark.parametrize("lengths, counts", [
    ([100, 0, 700, 650], [1, 1, 1, 1]),         # shorter than the common tokens, the first among them; an idle place
    ([0, 0, 0, 650], [1, 1, 1, 1]), ([0, 0, 0, 0], [1, 1, 1, 1]), ([640, 640, 641, 640], [1, 1, 1, 1]),  # no tokens of their own
    ([640, 642, 641, 700], [2, 3, 1, 1]),       # the first query does not see all of them; sees just all of them
    ([0, 640, 900, 3], [0, 1, 200, 3]), ([30, 640, 900, 3], [40, 300, 261, 7]), ([700, 100, 800, 900], [100, 90, 5, 1])])
@pytest.mark.parametrize("heads, group", [(2, 4), (1, 1), (1, 16)])
def test_requests_that_do_not_see_all_common_tokens(paged, lengths, counts, heads, group):
    """they are attended by themselves; more queries than tokens; none"""
    groups = [(0, 4, 650)]
    gen, table, cache = build(paged, 3, groups, lengths, heads, 64)
    q = torch.randn((sum(counts), heads * group, 128), generator=gen, device="cuda").to(torch.bfloat16)
    check(paged, q, cache, table, lengths, counts, starts_of(counts), groups, "bf16")
    if max(counts) == min(counts) == 1:
        check(paged, q, cache, table, lengths, counts, None, groups, "bf16")


@pytest.mark.parametrize("common", [-5, 0, 63, 1 << 30, (1 << 31) - 1])
@pytest.mark.parametrize("counts", [[1, 1, 1], [30, 2, 90]])
def test_numbers_of_common_tokens_that_no_request_has(paged, common, counts):
    lengths, heads, group = [512, 512, 500], 2, 4
    gen, table, cache = build(paged, 4, [(0, 3, 0)], lengths, heads, 64, width=8)
    q = torch.randn((sum(counts), heads * group, 128), generator=gen, device="cuda").to(torch.bfloat16)
    out, lse = paged.attend_shared(q, cache, table, ints(lengths), starts_of(counts), None, ints([common]), return_lse=True)
    agree(out, lse, pu.attend(q, cache.units, cache.k_scale, cache.v_scale, table, lengths, counts), "bf16")


@pytest.mark.parametrize("cuts", [[2, 4, 6], [0, 0, 3, 6, 6], [3, 3], [-4, 2, 9], [6, 6, 6], [0, 6, 100]])
def test_groups_without_requests_and_requests_without_a_group(paged, cuts):
    lengths, heads, group, P = [400 + 11 * i for i in range(6)], 2, 4, 32
    gen, table, cache = build(paged, 5, [(0, 6, 384)], lengths, heads, P)
    q = torch.randn((6, heads * group, 128), generator=gen, device="cuda").to(torch.bfloat16)
    common = ints([320 + 32 * i for i in range(len(cuts) - 1)])
    for starts in (None, starts_of([1] * 6)):
        out, lse = paged.attend_shared(q, cache, table, ints(lengths), starts, ints(cuts), common.clamp(max=384), return_lse=True)
        agree(out, lse, pu.attend(q, cache.units, cache.k_scale, cache.v_scale, table, lengths, [1] * 6), "bf16")


@pytest.mark.parametrize("counts", [[1, 1, 1], [6, 2, 1], [200, 30, 3]])
@pytest.mark.parametrize("order", ["rising", "falling", "one", "other", "flat"])
def test_scores_of_every_order(paged, order, counts):
    """scores that grow or fall along the sequence by hundreds, one far above the others in the common or in the own tokens"""
    lengths, heads, group, P, groups = [1777, 1500, 1400], 2, 4, 64, [(0, 3, 1100)]
    gen, table, cache = build(paged, 6, groups, lengths, heads, P)
    for b, length in enumerate(lengths):
        position = torch.arange(length, device="cuda")
        height = {"rising": position / 100.0, "falling": (1777 - position) / 100.0, "one": torch.where(position == 900, 25.0, 0.02), "other": torch.where(position == 1200, 25.0, 0.02),
                  "flat": torch.full((length,), 0.5, device="cuda")}[order]
        k = (height[:, None, None] * torch.ones((1, heads, 128), device="cuda")).to(torch.bfloat16)
        v = torch.randn((length, heads, 128), generator=gen, device="cuda").to(torch.bfloat16)
        paged.append(cache, k, v, (table[b, position // P].long() * P + position % P).to(torch.int32))
    q = (torch.rand((sum(counts), heads * group, 128), generator=gen, device="cuda") + 0.5).to(torch.bfloat16)
    check(paged, q, cache, table, lengths, counts, starts_of(counts), groups, "bf16", scale=0.05)


@pytest.mark.parametrize("group, counts", [(4, [1, 1, 1, 1]), (4, [2, 1, 3, 1]), (2, [30, 2, 100, 1]), (16, [1, 1, 1, 1])])
def test_not_a_number_in_common_and_own_tokens(paged, group, counts):
    """a NaN block of V or a NaN in K reaches the rows that see it: a common one those of the whole group, but not of a request that ends before it"""
    lengths, heads, P, groups = [400, 300, 500, 100], 2, 64, [(0, 4, 256)]
    gen, table, cache = build(paged, 7, groups, lengths, heads, P)
    q = torch.randn((sum(counts), heads * group, 128), generator=gen, device="cuda").to(torch.bfloat16)
    zeroed = with_bad_values(cache, table, 0, [(200, 1, 4, 0x7F)])
    again = with_bad_values(cache, table, 2, [(500 - counts[2], 0, 2, 0xFF)])
    pu.fields(again)[3][int(table[0, 200 // P]), 1, 200 % P // 16, 200 % 16, 4] = 0
    nan = torch.zeros(q.shape, dtype=torch.bool, device="cuda")
    nan[: sum(counts[:3]), group:, 64:80] = True
    nan[sum(counts[:2]) : sum(counts[:3]), :group, 32:48] = True
    cuts, common = group_args(groups)
    out, lse = paged.attend_shared(q, cache, table, ints(lengths), starts_of(counts), cuts, common, return_lse=True)
    assert torch.equal(out.isnan(), nan) and zeroed.shape == again.shape
    value, weight, log = pu.attend(q, again, cache.k_scale, cache.v_scale, table, lengths, counts)
    agree(torch.where(nan, value.to(out.dtype), out), lse, (value, weight, log), "bf16")
    pu.fields(cache.units)[2][int(table[0, 3]), 0, 1, 3, 6] = 0x7F  # K of token 211
    out = paged.attend_shared(q, cache, table, ints(lengths), starts_of(counts), cuts, common)
    nan[: sum(counts[:3]), :group] = True
    assert torch.equal(out.isnan(), nan)


@pytest.mark.parametrize("counts", [[1, 1, 1], [3, 1, 2], [150, 90, 1]])
def test_pages_that_are_not_there(paged, counts):
    """common and own tokens of table entries outside the pool are not seen; a length beyond the table's width is cut"""
    lengths, P, groups = [500, 500, 8 * 64 + 100], 64, [(0, 3, 320)]
    gen, table, cache = build(paged, 8, groups, [500, 500, 512], 2, P, width=8)
    table[:, 2], table[0, 7], table[1, 5], table[:, 0] = -1, cache.pages, 1 << 30, -(1 << 31)
    q = torch.randn((sum(counts), 8, 128), generator=gen, device="cuda").to(torch.bfloat16)
    cuts, common = group_args(groups)
    out, lse = paged.attend_shared(q, cache, table, ints(lengths), starts_of(counts), cuts, common, return_lse=True)
    agree(out, lse, pu.attend(q, cache.units, cache.k_scale, cache.v_scale, torch.where((table >= 0) & (table < cache.pages), table, -1), lengths, counts), "bf16")


@pytest.mark.parametrize("counts", [[1, 1, 1], [4, 3, 2], [130, 77, 1]])
def test_strides_rows_of_no_request_slices_and_another_stream(paged, counts):
    lengths, heads, group, P, pad, groups = [700, 422, 400], 4, 4, 32, 5, [(0, 3, 260)]
    gen, table, cache = build(paged, 9, groups, lengths, heads, P)
    wide = torch.zeros((cache.pages, 3, heads + 1, P // 16, 2304), dtype=torch.uint8, device="cuda")
    wide[:, 1, :heads] = cache.units
    cache = paged.PagedCache(wide[:, 1, :heads], cache.k_scale, cache.v_scale)
    rows = torch.randn((sum(counts) + pad, heads * group + 7, 128), generator=gen, device="cuda").to(torch.bfloat16)
    q, (cuts, common) = rows[:, 3 : 3 + heads * group], group_args(groups)
    table = torch.cat((table, table), 1)[:, : table.shape[1]]
    want = pu.attend(q[: sum(counts)], cache.units, cache.k_scale, cache.v_scale, table, lengths, counts)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        out, lse = paged.attend_shared(q, cache, table, ints(lengths), starts_of(counts), cuts, common, return_lse=True)
        assert bool((out[sum(counts) :] == 0).all()) and bool(torch.isneginf(lse[sum(counts) :]).all())
        agree(out[: sum(counts)], lse[: sum(counts)], want, "bf16")
        # the last two requests as a slice of the step's; rows that q does not have
        out, lse = paged.attend_shared(q, cache, table[1:], ints(lengths)[1:], starts_of(counts)[1:], None, common, return_lse=True)
        assert bool((out[: counts[0]] == 0).all()) and bool(torch.isneginf(lse[: counts[0]]).all())
        agree(out[counts[0] : sum(counts)], lse[counts[0] : sum(counts)], [x[counts[0] :] for x in want], "bf16")
        n = counts[0] + 1
        out, lse = paged.attend_shared(q[:n], cache, table, ints(lengths), starts_of(counts), cuts, common, return_lse=True)
        agree(out, lse, [x[:n] for x in want], "bf16")


def test_calls_of_all_shapes_one_after_the_other(paged):
    """calls of the three attentions on one stream without a wait between them: each leaves the scratch as the next one needs it"""
    rng, shapes = random.Random(6), []
    for i in range(12):
        batch = rng.randint(2, 9)
        counts = [rng.choice([1, 1, 2, 7, 40, 300]) for _ in range(batch)] if i % 3 else [1] * batch
        common = rng.choice([100, 1000, 3000])
        shapes.append((common, [common + n + rng.randint(0, 900) for n in counts], counts, rng.choice([1, 2, 8]), rng.choice([1, 4, 6])))
    calls = []
    for seed, (common, lengths, counts, heads, group) in enumerate(shapes):
        gen, table, cache = build(paged, 50 + seed, [(0, len(counts), common)], lengths, heads, 64)
        q = torch.randn((sum(counts), heads * group, 128), generator=gen, device="cuda").to(torch.bfloat16)
        calls.append(((q, cache, table, ints(lengths), None if max(counts) == 1 else starts_of(counts)), ints([common])))
    torch.cuda.synchronize()
    results = []
    for _ in range(4):
        for call, common in calls:
            results.append(paged.attend_shared(*call, None, common, return_lse=True))
            paged.attend(*call)
            paged.cross_attend(*call)
    for i, (out, lse) in enumerate(results[12:]):
        assert torch.equal(out, results[i % 12][0]) and torch.equal(lse, results[i % 12][1])
    for (call, _), (_, lengths, counts, _, _), (out, lse) in zip(calls, shapes, results):
        agree(out, lse, pu.attend(call[0], call[1].units, call[1].k_scale, call[1].v_scale, call[2], lengths, counts), "bf16")


def test_captured_steps_follow_lengths_groups_and_common_tokens(paged):
    """two graphs of calls on two streams, replayed at once for other lengths, groups and numbers of common tokens"""
    lengths, heads, group, P = [500 + 20 * i for i in range(8)], 2, 4, 32
    gen, table, cache = build(paged, 10, [(0, 8, 480)], lengths, heads, P)
    q = torch.randn((8, heads * group, 128), generator=gen, device="cuda").to(torch.bfloat16)
    held, cuts, common = ints(lengths), ints([0, 4, 8]), ints([480, 480])
    streams, graphs, results = [torch.cuda.Stream() for _ in range(2)], [], []
    torch.cuda.synchronize()
    for stream in streams:
        with torch.cuda.stream(stream):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                results.append(paged.attend_shared(q, cache, table, held, None, cuts, common, return_lse=True))
            graphs.append(graph)
    for lengths, at, tokens in ((lengths, [0, 4, 8], [480, 480]), ([490 + i for i in range(8)], [0, 2, 7], [100, 450]), ([1, 2, 3, 4, 481, 482, 500, 600], [0, 8, 8], [480, 0]),
                                ([600] * 8, [1, 1, 1], [480, 480])):
        lengths = [min(n, 500 + 20 * i) for i, n in enumerate(lengths)]
        held.copy_(ints(lengths))
        cuts.copy_(ints(at))
        common.copy_(ints(tokens))
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        want = pu.attend(q, cache.units, cache.k_scale, cache.v_scale, table, lengths, [1] * 8)
        for out, lse in results:
            agree(out, lse, want, "bf16")


def test_a_step_from_the_projection_to_both_attentions(paged):
    """a decoder layer's step as an engine runs it: pages for the new tokens, rotation and append, attention over common and own tokens, cross attention to an encoder's states; against the
    same tokens kept densely and rotated in 64 bits"""
    from tests.test_gpu_paged_rotate import angles, rotate, round16
    heads, group, P, batch, prompt = 2, 4, 16, 4, 100
    gen = generator(15)
    cache, states = paged.empty(90, heads, P), paged.empty(40, heads, P, v_scale=torch.full((heads,), 0.5))
    table = torch.full((batch, 20), -1, dtype=torch.int32, device="cuda")
    ring, cursor = torch.randperm(90, generator=gen, device="cuda").to(torch.int32), torch.tensor([0, 90], dtype=torch.int64, device="cuda")
    cos_sin = angles(400, 128)

    def qkv(n):
        return torch.randn((n, heads * group + 2 * heads, 128), generator=gen, device="cuda").to(torch.bfloat16).split([heads * group, heads, heads], 1)

    # the encoders' states
    sources = [30, 200, 0, 77]
    source_table, _ = pu.tables(gen, sources, P, spare=0)
    rows = torch.randn((sum(sources), 2 * heads, 128), generator=gen, device="cuda").to(torch.bfloat16)
    at = torch.cat([source_table[b, torch.arange(n, device="cuda") // P] * P + torch.arange(n, device="cuda") % P for b, n in enumerate(sources)]).to(torch.int32)
    paged.append(states, rows[:, :heads], rows[:, heads:], at)
    # the common prompt is the first request's; the others take its whole pages
    one = table[:1]
    _, k, v = qkv(prompt)
    step = paged.assign(one, ints([0]), ints([prompt]), ring, cursor, P, prompt)
    cursor = step.cursor
    whole = prompt // P * P
    kept = [[], []]
    paged.append_rotated(cache, k[:, :0], k, v, step.slots, step.positions, cos_sin)
    kept[0].append(round16(rotate(k, cos_sin[:prompt], False)[0], "bf16"))
    kept[1].append(v)
    table[1:, : whole // P] = table[:1, : whole // P]
    lengths = ints([prompt] + [whole] * (batch - 1))
    mine = [[torch.cat([kept[j][0][: prompt if b == 0 else whole]]) for b in range(batch)] for j in (0, 1)]
    for added in ([1, 17, 3, 9], [1, 1, 1, 1], [5, 1, 0, 40], [1, 1, 1, 1]):
        n = sum(added)
        q, k, v = qkv(n)
        step = paged.assign(table, lengths, ints(added), ring, cursor, P, n)
        turned = paged.append_rotated(cache, q, k, v, step.slots, step.positions, cos_sin)
        starts = None if added == [1] * batch else step.starts
        out, lse = paged.attend_shared(turned, cache, table, step.lengths, starts, None, ints([prompt]), return_lse=True)
        cross = paged.cross_attend(turned, states, source_table, ints(sources), starts)
        same = paged.attend(turned, cache, table, step.lengths, starts)
        assert float((out.float() - same.float()).abs().max()) <= 0.02 * float(same.abs().max())
        lengths, cursor = step.lengths, step.cursor
        k = round16(rotate(k, cos_sin[step.positions.long()], False)[0], "bf16")
        first = 0
        for b, m in enumerate(added):
            mine[0][b], mine[1][b] = torch.cat((mine[0][b], k[first : first + m])), torch.cat((mine[1][b], v[first : first + m]))
            for queries, factor, count, causal, got in ((mine, (cache.k_scale, cache.v_scale), lengths[b], True, out),
                                                        ([rows[sum(sources[:b]) : sum(sources[: b + 1]), j * heads : (j + 1) * heads] for j in (0, 1)], (states.k_scale, states.v_scale), sources[b], False, cross)):
                keys, vals = (queries[0][b], queries[1][b]) if causal else queries
                if keys.shape[0] == 0:
                    assert bool((got[first : first + m] == 0).all())
                    continue
                assert keys.shape[0] == int(count)
                (kc, ks), (vc, vs) = pu.quantise(keys, factor[0]), pu.quantise(vals, factor[1])
                kd, vd = pu.values(kc, ks, factor[0].cpu().double()[:, None]).cuda(), pu.values(vc, vs, factor[1].cpu().double()[:, None]).cuda()
                for i in range(m):
                    seen = keys.shape[0] - m + i + 1 if causal else keys.shape[0]
                    for x in range(heads * group):
                        s = kd[:seen, x // group] @ turned[first + i, x].double() / math.sqrt(128)
                        p = (s - torch.logsumexp(s, 0)).exp()
                        value = p @ vd[:seen, x // group]
                        assert bool(((got[first + i, x].double() - value).abs() <= 2.0 ** -10 * (p @ vd[:seen, x // group].abs()) + 2.0 ** -8 * value.abs() + 1e-7).all())
            first += m
    assert int(cursor[2]) == 0


def through_c(paged, q, cache, table, lengths, starts, cuts, common, fill=0xFF):
    """the C call with a scratch whose first 8192 bytes are zeros and the others `fill`, into outputs that hold 77"""
    tokens, heads, _ = q.shape
    out, lse = torch.full_like(q, 77.0), torch.full((tokens, heads), 77.0, device="cuda")
    call = paged._ATTEND.pack(lengths.numel(), tokens, heads, paged._TYPES[q.dtype], q.data_ptr(), q.stride(0), q.stride(1), out.data_ptr(), out.stride(0), out.stride(1),
                              lse.data_ptr(), table.data_ptr(), table.stride(0), table.shape[1], lengths.data_ptr(), 0 if starts is None else starts.data_ptr(), 0.0)
    groups = paged._COMMON.pack(common.numel(), 0 if cuts is None else cuts.data_ptr(), common.data_ptr())
    scratch = torch.full((paged._lib.mlops_paged_attend_shared_scratch_bytes(call, groups, cache.units.shape[1]),), fill, dtype=torch.uint8, device="cuda")
    scratch[:8192] = 0
    pool = paged._pool(cache)[0]
    for _ in range(2):
        status = paged._lib.mlops_paged_attend_shared(call, groups, pool, scratch.data_ptr(), scratch.numel(), torch.cuda.current_stream().cuda_stream)
        assert status == 0, paged._lib.mlops_paged_last_error()
    return out, lse


@pytest.mark.parametrize("fill", [0xFF, 0x7F, 0x01])
@pytest.mark.parametrize("counts", [[1, 1, 1, 1], [3, 0, 2, 5], [90, 2, 0, 150]])
def test_a_scratch_that_held_anything(paged, counts, fill):
    """zeros in front are all that a call asks for; requests that see nothing, rows of no request"""
    lengths, groups = [700, 0, 650, 900], [(0, 4, 600)]
    gen, table, cache = build(paged, 20, groups, lengths, 2, 64)
    q = torch.randn((sum(counts) + 3, 8, 128), generator=gen, device="cuda").to(torch.bfloat16)
    cuts, common = group_args(groups)
    out, lse = through_c(paged, q, cache, table, ints(lengths), starts_of(counts), cuts, common, fill)
    assert bool((out[sum(counts) :] == 0).all()) and bool(torch.isneginf(lse[sum(counts) :]).all())
    want = pu.attend(q[: sum(counts)], cache.units, cache.k_scale, cache.v_scale, table, lengths, counts)
    agree(out[: sum(counts)], lse[: sum(counts)], want, "bf16")


@pytest.mark.parametrize("fill", [0xFF, 0x01])
@pytest.mark.parametrize("starts, cuts", [([8, 2, 12, 12, 20], [0, 4]), ([0, 5, 3, 9, 20], [2, 1, 4]), ([0, 1, 2, 3, 4], [3, 0, 9]), ([0, 1000, -5, 20, 20], [0, 3, 1, 4]), ([0, 5, 10, 15, 20], [-7, 1 << 30])])
def test_starts_and_groups_out_of_order(paged, starts, cuts, fill):
    """no row means anything then, but each is written at most, and nothing beside them; the requests' rows that are in order are as they would be"""
    lengths = [300, 310, 320, 330]
    gen, table, cache = build(paged, 21, [(0, 4, 256)], lengths, 2, 64)
    rows = torch.randn((26, 8, 128), generator=gen, device="cuda").to(torch.bfloat16)
    out, lse = through_c(paged, rows[:20], cache, table, ints(lengths), ints(starts), ints(cuts), ints([256] * (len(cuts) - 1)), fill)
    assert out.shape == (20, 8, 128)
    if starts == [0, 5, 10, 15, 20]:
        agree(out, lse, pu.attend(rows[:20], cache.units, cache.k_scale, cache.v_scale, table, lengths, [5] * 4), "bf16")


@pytest.mark.parametrize("batch, groups", [(1500, 500), (2047, 1), (1024, 1024)])
def test_as_many_requests_and_groups_as_a_call_takes(paged, batch, groups):
    size = -(-batch // groups)
    cuts = [min(g * size, batch) for g in range(groups + 1)]
    lengths = [33 + (7 * b) % 60 for b in range(batch)]
    gen, table, cache = build(paged, 22, [(a, b, 32) for a, b in zip(cuts, cuts[1:])], lengths, 1, 16)
    q = torch.randn((batch, 2, 128), generator=gen, device="cuda").to(torch.bfloat16)
    out, lse = paged.attend_shared(q, cache, table, ints(lengths), None, ints(cuts), ints([32] * groups), return_lse=True)
    agree(out, lse, pu.attend(q, cache.units, cache.k_scale, cache.v_scale, table, lengths, [1] * batch), "bf16")
    with pytest.raises(ValueError, match="2048"):
        paged.attend_shared(q, cache, table, ints(lengths), None, torch.zeros(2049 - batch + 1, dtype=torch.int32, device="cuda"), torch.zeros(2049 - batch, dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("counts", [[1, 1, 1], [6, 2, 1], [150, 90, 3]])
def test_a_pool_of_more_than_4_gib(paged, counts):
    """pages far beyond 2^32 bytes from the pool's start: rotation and append, attention over common and own tokens, cross attention"""
    from tests.test_gpu_paged_rotate import angles, rotate, round16
    heads, P, lengths, unit = 2, 64, [500, 470, 400], 4 * 2304
    gen, table, small = build(paged, 23, [(0, 3, 256)], lengths, heads, P)
    pages = small.pages
    stride = ((5 << 30) // pages + 4095) // 4096 * 4096
    units = torch.zeros(pages * stride, dtype=torch.uint8, device="cuda").as_strided((pages, heads, P // 16, 2304), (stride, unit, 2304, 1))
    units.copy_(small.units)
    cache = paged.PagedCache(units, small.k_scale, small.v_scale)
    q = torch.randn((sum(counts), heads * 4, 128), generator=gen, device="cuda").to(torch.bfloat16)
    check(paged, q, cache, table, lengths, counts, starts_of(counts), [(0, 3, 256)], "bf16")
    same = paged.cross_attend(q, small, table, ints(lengths), starts_of(counts))
    assert torch.equal(same, paged.cross_attend(q, cache, table, ints(lengths), starts_of(counts)))
    k = torch.randn((3, heads, 128), generator=gen, device="cuda").to(torch.bfloat16)
    slots, cos_sin, positions = ints([(pages - 1) * P + 1, (pages - 1) * P + 63, (pages - 2) * P]), angles(600, 128), ints([5, 500, 599])
    paged.append_rotated(cache, q[:3], k, k, slots, positions, cos_sin)
    turned = round16(rotate(k, cos_sin[positions.long()], False)[0], "bf16")
    for got, x in zip(pu.at_slots(units, slots), sum(zip(pu.quantise(turned, cache.k_scale), pu.quantise(k, cache.v_scale)), ())):
        assert torch.equal(got.cpu(), x)


def test_a_long_beginning(paged):
    """200 000 common tokens, as one item of the stream and of the tile kernel"""
    common = 200000
    for batch in (3, 12):
        lengths = [common + 1 + 50 * b for b in range(batch)]
        gen, table, cache = build(paged, 24, [(0, batch, common)], lengths, 1, 256)
        q = torch.randn((batch, 4, 128), generator=gen, device="cuda").to(torch.bfloat16)
        check(paged, q, cache, table, lengths, [1] * batch, None, [(0, batch, common)], "bf16")


@pytest.mark.parametrize("rows", [79, 80, 81, 82, 100])
def test_on_both_sides_of_requests_that_fill_rows_of_work(paged, rows):
    """80 queries of four heads each are 320 columns: up to there on average a group's tokens are taken together"""
    lengths, counts, groups = [700, 720, 800, 300], [rows, 80, 80, 5], [(0, 3, 500), (3, 4, 100)]
    gen, table, cache = build(paged, 25, groups, lengths, 2, 64)
    q = torch.randn((sum(counts), 8, 128), generator=gen, device="cuda").to(torch.float16)
    check(paged, q, cache, table, lengths, counts, starts_of(counts), groups, "fp16")


def guarded(shape, kind, value):
    """an array between two stretches of sentinels, and the whole"""
    n, around = math.prod(shape), 4096
    whole = torch.full((n + 2 * around,), value, dtype=kind, device="cuda")
    return whole[around : around + n].view(shape), whole, around


@pytest.mark.parametrize("fill", [0xFF, 0x01])
@pytest.mark.parametrize("starts", [[0, 5, 10, 15, 20], [8, 2, 12, 12, 20], [0, 5, 3, 9, 20], [0, 1, 2, 3, 4], [0, 1000, -5, 20, 20], [3, 9, 20, 31, 60], [6, 0, 90, 95, 200]])
@pytest.mark.parametrize("cuts", [[0, 4], [2, 1, 4], [3, 0, 9], [0, 3, 1, 4], [-7, 1 << 30], [2, 4, 0, 2]])
def test_rows_that_only_one_request_and_group_name(paged, starts, cuts, fill):
    """starts and groups in any order: a row that belongs to one request, and lies in the rows of one group at most, has what attention by itself gives; nothing is written around the arrays or into
    what a call reads"""
    lengths, heads, tokens, batch = [300, 310, 320, 330], 2, 20, 4
    gen, table, cache = build(paged, 26, [(0, 4, 256)], lengths, heads, 64)
    rows = torch.randn((tokens, 8, 128), generator=gen, device="cuda").to(torch.bfloat16)
    common = [256 - 64 * (g % 3) for g in range(len(cuts) - 1)]
    out, out_whole, around = guarded((tokens, 8, 128), torch.bfloat16, 77.0)
    lse, lse_whole, _ = guarded((tokens, 8), torch.float32, 77.0)
    held, begins, groups_at, common_at = ints(lengths), ints(starts), ints(cuts), ints(common)
    call = paged._ATTEND.pack(batch, tokens, 8, 0, rows.data_ptr(), 1024, 128, out.data_ptr(), 1024, 128, lse.data_ptr(), table.data_ptr(), table.stride(0), table.shape[1], held.data_ptr(),
                              begins.data_ptr(), 0.0)
    groups = paged._COMMON.pack(len(common), groups_at.data_ptr(), common_at.data_ptr())
    scratch, scratch_whole, _ = guarded((paged._lib.mlops_paged_attend_shared_scratch_bytes(call, groups, heads),), torch.uint8, fill)
    scratch[:8192] = 0
    inputs = [x.clone() for x in (rows, cache.units, table, held, begins, groups_at, common_at)]
    for _ in range(2):
        assert paged._lib.mlops_paged_attend_shared(call, groups, paged._pool(cache)[0], scratch.data_ptr(), scratch.numel(), torch.cuda.current_stream().cuda_stream) == 0
    for x, y in zip(inputs, (rows, cache.units, table, held, begins, groups_at, common_at)):
        assert torch.equal(x, y)
    for whole, value in ((out_whole, 77.0), (lse_whole, 77.0), (scratch_whole, fill)):
        assert bool((whole[:around] == value).all()) and bool((whole[-around:] == value).all())
    assert bool((scratch[:8192] == 0).all())

    clip = lambda x, lo, hi: min(max(x, lo), hi)
    mine = [(clip(starts[b], 0, tokens), min(starts[b + 1], tokens)) for b in range(batch)]
    firsts = [(clip(cuts[g], 0, batch), clip(cuts[g + 1], 0, batch)) for g in range(len(common))]
    theirs = [(clip(starts[a], 0, tokens), min(starts[b], tokens)) for a, b in firsts if b - a > 1]
    edges = clip(starts[0], 0, tokens), min(max(starts[-1], starts[0], 0), tokens)  # rows of no request are before and behind
    once = [edges[0] <= i < edges[1] and sum(a <= i < b for a, b in mine) == 1 and sum(a <= i < b for a, b in theirs) <= 1 for i in range(tokens)]
    checked = 0
    for b, (first, end) in enumerate(mine):
        n = max(end - first, 0)
        if n == 0:
            continue
        value, weight, log = pu.attend(rows[first:end], cache.units, cache.k_scale, cache.v_scale, table[b : b + 1], [max(lengths[b] - starts[b + 1] + end, 0)], [n])
        keep = torch.tensor(once[first:end], device="cuda")
        agree(out[first:end][keep], lse[first:end][keep], [x[keep] for x in (value, weight, log)], "bf16")
        checked += int(keep.sum())
    assert checked == sum(once)
    for free in (slice(0, edges[0]), slice(edges[1], tokens)):
        untouched = [i for i in range(tokens)[free] if not any(a <= i < b for a, b in mine)]
        assert bool((out[untouched] == 0).all()) and bool(torch.isneginf(lse[untouched]).all())


@pytest.mark.parametrize("tokens, heads, kv_heads, with_starts", [(1, 8, 8, False), (8, 32, 8, False), (9, 32, 8, False), (64, 32, 8, False), (8, 32, 8, True), (9, 32, 8, True), (3, 40, 1, False), (1, 40, 1, True)])
def test_the_scratch_that_a_call_asks_for(paged, tokens, heads, kv_heads, with_starts):
    """1056 bytes per row of q and query head beside attend's: that of a call with starts where there are more than 32 rows per KV head, that of one without where there are no more"""
    def attend(starts, heads=heads):
        return paged._lib.mlops_paged_attend_scratch_bytes(paged._ATTEND.pack(tokens, tokens, heads, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 4096 if starts else 0, 0.0), kv_heads)
    call = paged._ATTEND.pack(tokens, tokens, heads, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 4096 if with_starts else 0, 0.0)
    many = tokens * heads // kv_heads > 32
    beside = attend(True) if many else attend(False, kv_heads)
    assert paged._lib.mlops_paged_attend_shared_scratch_bytes(call, paged._COMMON.pack(1, 0, 4096), kv_heads) == beside + 1056 * tokens * heads
