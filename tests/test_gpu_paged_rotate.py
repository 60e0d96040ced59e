"""append_rotated against plain rotation in 64 bits: the cache's bytes are those of the exact rotation rounded once to 16 bits, q is off by its own rounding and that of FP32.

The bound of q: fl(x c - fl(y s)) in FP32 is off by at most 2^-24 |y s| + 2^-24 |x c - y s|, below 2^-23 (|x c| + |y s|); the type's rounding adds half a step of the value, at
least half its smallest number (2^-25 for FP16, 2^-134 for BF16)."""
import math
import random
import struct
from fractions import Fraction

import pytest
import torch

from tests import paged_util as pu
from tests.test_gpu_paged import TYPES, factors, generator, ints

pytestmark = pytest.mark.gpu
LEAST = {"bf16": 2.0 ** -134, "fp16": 2.0 ** -25}


@pytest.fixture(scope="module")
def paged():
    from mlops_b200.attention import paged
    return paged


def angles(reach, R, base=10000.0):
    a = torch.arange(reach, dtype=torch.float64, device="cuda")[:, None] * base ** (-torch.arange(0, R, 2, dtype=torch.float64, device="cuda") / R)
    return torch.cat((a.cos(), a.sin()), -1).float()


def rotate(x, rows, interleaved):
    """(the rotation of x [tokens, heads, 128] in 64 bits, |x c| + |y s| element by element)"""
    R = rows.shape[1]
    out, size = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    for i in range(R // 2):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
        c, s, y, z = rows[:, None, i].double(), rows[:, None, R // 2 + i].double(), x[..., a].double(), x[..., b].double()
        out[..., a], out[..., b] = y * c - z * s, z * c + y * s
        size[..., a], size[..., b] = (y * c).abs() + (z * s).abs(), (z * c).abs() + (y * s).abs()
    return out, size


def round16(x, name):
    """64-bit numbers rounded once to the type, halfway to even"""
    bits, least = (8, -133) if name == "bf16" else (11, -24)
    unit = torch.exp2((torch.frexp(x)[1].double() - bits).clamp(min=least))
    return torch.where(torch.isfinite(x), torch.round(x / unit) * unit, x).to(TYPES[name][0])


def check(paged, name, q, k, v, units, k_scale, v_scale, slots, positions, table, interleaved, **how):
    cache = paged.PagedCache(units, k_scale, v_scale)
    before, reach = units.clone(), table.shape[0]
    out = paged.append_rotated(cache, q, k, v, slots, positions, table, interleaved=interleaved, **how)
    known = (positions >= 0) & (positions < reach)
    rows = table[positions.clamp(0, max(reach - 1, 0)).long()] if reach else torch.zeros((len(positions), table.shape[1]), device="cuda")
    want, size = rotate(q, rows, interleaved)
    assert out.dtype == q.dtype and out.shape == q.shape and out.is_contiguous()
    off = (out.double() - want).abs()[known]
    assert bool((off <= TYPES[name][1] * want.abs()[known] + 2.0 ** -23 * size[known] + LEAST[name]).all())
    R = table.shape[1]
    assert torch.equal(out[known][..., R:], q[known][..., R:])
    assert bool((out[positions < 0] == 0).all()) and bool(out[positions >= reach].isnan().all())
    turned = round16(rotate(k, rows, interleaved)[0], name)
    turned[positions >= reach] = math.nan
    P = units.shape[2] * 16
    stored = (slots >= 0) & (slots < units.shape[0] * P) & (positions >= 0)
    at = torch.where(stored, slots, 0)
    there = stored.cpu()
    for got, x in zip(pu.at_slots(units, at), sum(zip(pu.quantise(turned, k_scale), pu.quantise(v, v_scale)), ())):
        assert torch.equal(got.cpu()[there], x[there])
    rest = torch.ones(units.shape[0] * P, dtype=torch.bool, device="cuda")
    rest[slots[stored].long()] = False
    rest = rest.nonzero().view(-1).to(torch.int32)
    for got, x in zip(pu.at_slots(units, rest), pu.at_slots(before, rest)):
        assert torch.equal(got, x)  # nothing else was written
    return out


def case(seed, tokens, heads, group, page_size, name, reach, R, wide=0):
    gen = generator(seed)
    pages = -(-tokens // page_size) + 2
    units = torch.full((pages, heads, page_size // 16, 2304), 0xA5, dtype=torch.uint8, device="cuda")
    slots = torch.randperm(pages * page_size, generator=gen, device="cuda")[:tokens].to(torch.int32)
    positions = torch.randint(0, reach, (tokens,), generator=gen, device="cuda").to(torch.int32)
    n = heads * group
    rows = torch.randn((tokens, n + 2 * heads + wide, 8, 16), generator=gen, device="cuda") * torch.exp2(torch.randint(-8, 9, (tokens, n + 2 * heads + wide, 8, 1), generator=gen, device="cuda").float())
    q, k, v = rows.flatten(-2).to(TYPES[name][0])[:, wide:].split([n, heads, heads], 1)
    return gen, q, k, v, units, *factors(gen, heads), slots, positions


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens, heads, group, page_size, R", [(1, 1, 1, 16, 128), (3, 8, 4, 64, 128), (257, 2, 5, 32, 64), (70, 5, 3, 48, 96), (40, 9, 1, 16, 32), (2500, 3, 3, 256, 128)])
def test_the_exact_rotation_is_stored(paged, name, interleaved, tokens, heads, group, page_size, R):
    _, q, k, v, units, ks, vs, slots, positions = case(tokens + R, tokens, heads, group, page_size, name, 5000, R)
    check(paged, name, q, k, v, units, ks, vs, slots, positions, angles(5000, R), interleaved)


@pytest.mark.parametrize("name", ["bf16", "fp16"])
def test_many_tokens(paged, name):
    """more tokens than the device holds warps for: a warp then has all heads of a token"""
    _, q, k, v, units, ks, vs, slots, positions = case(5, 9001, 2, 4, 64, name, 131072, 128)
    check(paged, name, q, k, v, units, ks, vs, slots, positions, angles(131072, 128), False)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("R", [32, 128])
def test_tokens_without_a_slot_or_a_position(paged, interleaved, R):
    _, q, k, v, units, ks, vs, slots, positions = case(7, 64, 2, 3, 32, "bf16", 100, R)
    slots[3], slots[9], slots[11] = -1, 1 << 30, -(1 << 31)
    positions[3], positions[20], positions[21], positions[30], positions[31], positions[9] = 5, -1, -(1 << 31), 100, (1 << 31) - 1, 100
    check(paged, "bf16", q, k, v, units, ks, vs, slots, positions, angles(100, R), interleaved)


@pytest.mark.parametrize("reach", [0, 1])
def test_tables_of_no_position_and_of_one(paged, reach):
    _, q, k, v, units, ks, vs, slots, positions = case(8, 5, 1, 2, 16, "fp16", 3, 128)
    positions[:3] = ints([0, -1, 1])
    check(paged, "fp16", q, k, v, units, ks, vs, slots, positions, angles(3, 128)[:reach].contiguous(), False)


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_values_that_are_not_finite(paged, name, interleaved):
    """infinity and NaN in q and k reach their pairs and no other channel; a block of k with one reads as NaN, V's are V's own"""
    _, q, k, v, units, ks, vs, slots, positions = case(9, 6, 1, 1, 16, name, 50, 128)
    q, k, v = q.clone(), k.clone(), v.clone()
    positions[0] = 0  # (cosine 1, sine 0: infinity times 0 is NaN)
    q[0, 0, 3], q[1, 0, 70], k[0, 0, 3], k[1, 0, 70], k[2, 0, 127], v[3, 0, 64] = math.inf, math.nan, math.inf, -math.inf, math.nan, math.nan
    table = angles(50, 128)
    out = paged.append_rotated(paged.PagedCache(units, ks, vs), q, k, v, slots, positions, table, interleaved=interleaved)
    want = rotate(q, table[positions.long()], interleaved)[0]
    assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out.isinf(), want.isinf())
    kc, vc, kscale, vscale = pu.at_slots(units, slots)
    bad = ~torch.isfinite(rotate(k, table[positions.long()], interleaved)[0]).unflatten(-1, (8, 16)).all(-1)
    assert torch.equal(kscale == 0x7F, bad) and torch.equal(vscale == 0x7F, ~torch.isfinite(v.float()).unflatten(-1, (8, 16)).all(-1))
    assert bool((kc.unflatten(-1, (8, 8))[bad] == 0).all())


def test_rotations_halfway_between_two_numbers(paged):
    """x c - y s that lie a little beside the middle of two BF16 numbers, by less than FP32 holds: the side decides"""
    heads, tokens = 1, 32
    q = torch.zeros((tokens, 1, 128), dtype=torch.bfloat16, device="cuda")
    k = torch.zeros((tokens, 1, 128), dtype=torch.bfloat16, device="cuda")
    # c = 0.75 - 2^-9 is halfway between 0.75 - 2^-8 and 0.75, and 0.75 between the codes of 0.5 and 1 where the block's largest element is 6: x = 1, and y s = +- 2^-26 .. 2^-41 beside
    # it (most too small for FP32), or 0
    k[:, 0, :64], k[:, 0, 64:], k[:, 0, :64:16] = 1.0, 2.0 ** -7, 6.0
    table = torch.zeros((tokens, 128), device="cuda")
    table[:, :64], table[:, :64:16] = 0.75 - 2.0 ** -9, 1.0
    for p in range(1, tokens):
        table[p, 64:] = (-1) ** p * 2.0 ** (-19 - p // 2)
    table[:, 64::16] = 0.0
    units = torch.zeros((2, 1, 1, 2304), dtype=torch.uint8, device="cuda")
    one, at = torch.ones(1, device="cuda"), torch.arange(tokens, dtype=torch.int32, device="cuda")
    check(paged, "bf16", q, k, k, units, one, one, at, at, table, False)
    codes = pu.at_slots(units, at)[0][:, 0, 1]
    assert codes.tolist() == [0x22 if p == 0 or p % 2 else 0x11 for p in range(tokens)]  # (x c - y s: odd p have a negative s)


@pytest.mark.parametrize("wide", [1, 3])
def test_slices_of_a_projection_at_any_place(paged, wide):
    """rows that begin 16 bytes off a 32-byte boundary, a table inside a wider one, q in rows of its own"""
    gen, q, k, v, units, ks, vs, slots, positions = case(11, 50, 2, 2, 32, "bf16", 40, 64, wide)
    flat = torch.randn((50, (4 + 4) * 128 + 8), generator=gen, device="cuda").to(torch.bfloat16)
    q, k, v = flat[:, 8 : 8 + 512].view(50, 4, 128), flat[:, 520 : 520 + 256].unflatten(1, (2, 128)), flat[:, 776 : 776 + 256].unflatten(1, (2, 128))
    wider = torch.cat((angles(40, 64), torch.full((40, 4), math.nan, device="cuda")), 1)
    check(paged, "bf16", q, k, v, units, ks, vs, slots, positions, wider[:, :64], True)


def test_no_query_heads_and_no_tokens(paged):
    _, q, k, v, units, ks, vs, slots, positions = case(12, 20, 3, 1, 16, "fp16", 40, 128)
    other = units.clone()
    out = paged.append_rotated(paged.PagedCache(units, ks, vs), q[:, :0], k, v, slots, positions, angles(40, 128))
    assert out.shape == (20, 0, 128)
    paged.append_rotated(paged.PagedCache(other, ks, vs), q, k, v, slots, positions, angles(40, 128))
    assert torch.equal(units, other)
    assert paged.append_rotated(paged.PagedCache(units, ks, vs), q[:0], k[:0], v[:0], slots[:0], positions[:0], angles(40, 128)).shape == (0, 3, 128) and torch.equal(units, other)


@pytest.mark.parametrize("tokens", [40, 6000])
def test_q_in_place_through_the_c_call(paged, tokens):
    _, q, k, v, units, ks, vs, slots, positions = case(13, tokens, 2, 4, 16, "bf16", 400, 128)
    table, other = angles(400, 128), units.clone()
    want = paged.append_rotated(paged.PagedCache(other, ks, vs), q, k, v, slots, positions, table)
    rows = torch.cat((q, k, v), 1)
    a = paged._ROTATE.pack(tokens, 8, 0, 128, 0, 400, table.data_ptr(), 128, rows.data_ptr(), rows[:, 8:].data_ptr(), rows[:, 10:].data_ptr(), 12 * 128, 128, 12 * 128, 128, 12 * 128, 128,
                           rows.data_ptr(), 12 * 128, 128, slots.data_ptr(), positions.data_ptr())
    assert paged._lib.mlops_paged_append_rotated(paged._pool(paged.PagedCache(units, ks, vs))[0], a, torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(rows[:, :8], want) and torch.equal(rows[:, 8:10], k) and torch.equal(units, other)


def test_a_captured_call_follows_positions_and_slots(paged):
    gen, q, k, v, units, ks, vs, slots, positions = case(14, 30, 2, 4, 32, "bf16", 300, 128)
    q, k, v, table, cache = q.contiguous(), k.contiguous(), v.contiguous(), angles(300, 128), paged.PagedCache(units, ks, vs)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = paged.append_rotated(cache, q, k, v, slots, positions, table)
        for step in range(3):
            positions.copy_(torch.randint(0, 300, (30,), generator=gen, device="cuda"))
            slots.copy_(slots.roll(1))
            k.copy_(torch.randn(k.shape, generator=gen, device="cuda"))
            graph.replay()
            other = paged.PagedCache(units.clone(), ks, vs)
            assert torch.equal(out, paged.append_rotated(other, q, k, v, slots, positions, table)) and torch.equal(other.units, units)


def nearest16(x, name):
    """the number of the type nearest to a fraction, halfway to even"""
    bits, least = (8, -133) if name == "bf16" else (11, -24)
    if x == 0:
        return 0.0
    size = abs(x).numerator.bit_length() - abs(x).denominator.bit_length()  # floor(log2 |x|), or one above it
    size -= abs(x) < Fraction(2) ** size
    unit = Fraction(2) ** max(size - bits + 1, least)
    return float(round(x / unit) * unit)


def fp32(x):
    return struct.unpack("f", struct.pack("f", x))[0]


def beside_a_middle(rng, name):
    """(x, c, y, s) whose x c - y s lies beside the middle of two numbers of the type, of which a code's border is one, by far less than FP32 tells apart: x c is off the middle, and rounds to it in
    FP32, by what y s takes away again but for its own rounding; or x c is the middle and y s below what FP32 holds of a product's error"""
    bits = 8 if name == "bf16" else 11
    border, up = rng.choice([(0.75, False), (1.75, False), (3.5, False), (0.25, True), (1.25, True), (2.5, True), (5.0, True)])  # a border belongs to the even code beside it
    middle = border + (1 if up else -1) * 2.0 ** (math.frexp(border)[1] - bits - 1)
    number = lambda: rng.choice([-1, 1]) * (1 + rng.randrange(1 << (bits - 1)) / (1 << (bits - 1)))
    if rng.random() < 0.2:
        return 1.0, middle, 2.0 ** -7, rng.choice([-1, 1]) * 2.0 ** -rng.choice([30, 60, 100, 120, 126, 133, 142, 149])
    while True:
        x, y = number() * rng.choice([1, 2, 4]), number()
        c = fp32(rng.choice([-1, 1]) * middle / x)
        off = x * c - math.copysign(middle, x * c)  # (x c is exact in FP64, and so is the difference of numbers so near to each other)
        s = fp32(off / y)
        if off and fp32(x * c) == math.copysign(middle, x * c) and off != y * s:
            return x, c, y, s


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotations_that_only_the_exact_sum_tells_from_a_middle(paged, name, interleaved):
    """against whole-number fractions; the side of the middle decides a code where a block's scale is 1, as its 6 makes it mostly"""
    tokens, rng = 96, random.Random(31 + interleaved)
    k, table = torch.zeros((tokens, 1, 128), dtype=torch.float64), torch.zeros((tokens, 128), dtype=torch.float64)
    want = torch.zeros((tokens, 1, 128), dtype=torch.float64)
    middles = 0
    for t in range(tokens):
        for i in range(64):
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + 64)
            if i % 8 == 0:
                x, c, y, s = 6.0, 1.0, 6.0, 0.0
            else:
                x, c, y, s = beside_a_middle(rng, name)
                if rng.random() < 0.5:  # y c + x s of the pair
                    x, y, s = y, x, -s
            k[t, 0, a], k[t, 0, b], table[t, i], table[t, 64 + i] = x, y, c, s
            x, c, y, s = (Fraction(z) for z in (x, c, y, s))
            want[t, 0, a], want[t, 0, b] = nearest16(x * c - y * s, name), nearest16(y * c + x * s, name)
            middles += i % 8 > 0
    kind, one, at = TYPES[name][0], torch.ones(1, device="cuda"), torch.arange(tokens, dtype=torch.int32, device="cuda")
    assert torch.equal(k.to(kind).double(), k) and torch.equal(table.float().double(), table) and torch.equal(want.to(kind).double(), want) and middles == tokens * 56
    units = torch.zeros((tokens // 16, 1, 1, 2304), dtype=torch.uint8, device="cuda")
    k, table = k.to(kind).cuda(), table.float().cuda()
    paged.append_rotated(paged.PagedCache(units, one, one), k[:, :0], k, k, at, at, table, interleaved=interleaved)
    codes, scales = pu.quantise(want.to(kind), one)
    assert float((scales == 0x38).double().mean()) > 0.9  # (some of the pairs' other sums are above 6)
    got = pu.at_slots(units, at)
    assert torch.equal(got[0].cpu(), codes) and torch.equal(got[2].cpu(), scales)


@pytest.mark.parametrize("name, x, c, y, s, right", [("bf16", 1.09375, "0x1.933334p-1", 1.0859375, "0x1.9c8bf8p-26", 0.86328125), ("bf16", 1.8359375, "0x1.c1e808p-2", 1.171875, "-0x1.1eb852p-26", 0.80859375),
                                                     ("fp16", 1.5322265625, "0x1.552b90p-2", 1.6044921875, "-0x1.84e878p-28", 0.51025390625)])
def test_rotations_whose_products_errors_cancel(paged, name, x, c, y, s, right):
    """what is left behind both products' errors decides. The head's factor puts the border of the codes 0 and 0.5 between the two numbers"""
    kind, bits = TYPES[name][0], 8 if name == "bf16" else 11
    c, s = float.fromhex(c), float.fromhex(s)
    exact = Fraction(x) * Fraction(c) - Fraction(y) * Fraction(s)
    assert nearest16(exact, name) == right
    unit = 2.0 ** (math.frexp(right)[1] - bits)
    other = right - unit if exact < right else right + unit
    low, high = min(right, other), max(right, other)
    k, table = torch.zeros((1, 1, 128)), torch.ones((1, 128))
    table[:, 64:] = 0
    k[0, 0, 0], k[0, 0, 64], table[0, 0], table[0, 64] = x, y, c, s
    factor = 2 * (low + high)
    k[0, 0, 1] = 6 * factor  # (rounded to the type: the block's scale is 1 all the same)
    one, at = torch.full((1,), factor, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    units, k = torch.zeros((1, 1, 1, 2304), dtype=torch.uint8, device="cuda"), k.to(kind).cuda()
    cache = paged.PagedCache(units, one, one)
    paged.append_rotated(cache, k[:, :0], k, k, at, at, table.cuda())
    got = [z.cpu() for z in pu.at_slots(units, at)]
    codes = []
    for z in (low, high):
        turned = k.cpu().clone()
        turned[0, 0, 0], turned[0, 0, 64] = z, nearest16(Fraction(y) * Fraction(c) + Fraction(x) * Fraction(s), name)
        codes.append(pu.quantise(turned, one))
    assert not torch.equal(codes[0][0], codes[1][0])  # (the border tells them apart)
    assert torch.equal(got[0], codes[right == high][0]) and torch.equal(got[2], codes[right == high][1])
