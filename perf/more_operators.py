"""Further operators of the paged 4-bit cache (`mlops_b200.attention.paged`) as cases that can be timed and compared.

`append_rotated` takes a step's queries, keys and values as the projection leaves them: it rotates q and k by their tokens' positions (a table of
cosines and sines) and writes k and v into the cache on the way. `cross_attend` is attention to states of another length (an encoder's) that the cache holds:
every query of a request sees all of its states. `attend_shared` is the attention of a batch whose requests begin with the same tokens, in the same pages
(a system's prompt, a document that is asked about many times): what `attend` gives, with the common pages read once for all.

The pool: uint8 [pages, KV heads, page_size / 16, 2304]; the 2304 bytes of a block hold 16 tokens of one KV head:
K codes [16][64], V codes [16][64], K scales [16][8], V scales [16][8]. A code is E2M1 (sign, two bits of exponent, one of
mantissa), channel 2 i in the low and 2 i + 1 in the high half of byte i; a scale is E4M3 and serves 16 channels; the value is
code * scale * k_scale[head] (v_scale for V). It is what `append` writes: y = x * (1 / factor), scale = E4M3(max |y| / 6), code = E2M1(y / scale), each in FP32 with one
rounding per operation.

Rotation of a pair (x, y) by (c, s) of its position: (x c - y s, y c + x s); pairs are (i, i + R / 2) of the first R channels of a head, or (2 i, 2 i + 1). A row of the
table holds R / 2 cosines, then R / 2 sines. Rotated K is rounded once to its 16-bit type before it is quantised, as a model that rotates by itself has it.

`own` False computes the same in elementary torch operations, in 32 bits, the rotation of K in 64 (a stored code asks on which side of a border a value lies). A case's lengths
follow from its `mix`, so that its work is known; its values follow from the seed.
"""
import math
import random

import torch

own = False

D, BLOCK, BLOCK_BYTES = 128, 16, 2304
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # an engine's decode step: one token for each of 64 requests, at positions of their own; launches and latency count
        dict(name="rotate_64", op="rotate", tokens=64, kv_heads=8, group=4, page_size=64, dtype="bf16", rotated=128, interleaved=False, reach=65536, mix=1),
        # a chunk of an odd length of a model that rotates half of the channels, in pairs of neighbours
        dict(name="rotate_999", op="rotate", tokens=999, kv_heads=2, group=7, page_size=32, dtype="fp16", rotated=64, interleaved=True, reach=20000, mix=2),
        # two prompts of 8192 tokens at once
        dict(name="rotate_16k", op="rotate", tokens=16384, kv_heads=8, group=4, page_size=64, dtype="bf16", rotated=128, interleaved=False, reach=16384, mix=3),
        # the smallest decode: one new token, one encoder's states, a KV head per query head
        dict(name="cross_b1_1500", op="cross", batch=1, held_lo=1500, held_hi=1500, new_lo=1, new_hi=1, idle=0, kv_heads=16, group=1, page_size=64, dtype="bf16", lse=False, mix=4),
        # a decode batch of 64 encoders of 100 to 4000 states, two of its places idle
        dict(name="cross_b64", op="cross", batch=64, held_lo=100, held_hi=4000, new_lo=1, new_hi=1, idle=2, kv_heads=16, group=1, page_size=64, dtype="bf16", lse=False, mix=5),
        # five beams per encoder, small pages, the log-sum-exp asked for
        dict(name="cross_beams", op="cross", batch=16, held_lo=300, held_hi=2000, new_lo=5, new_hi=5, idle=0, kv_heads=8, group=2, page_size=32, dtype="fp16", lse=True, mix=6),
        # whole target texts over long sources
        dict(name="cross_texts", op="cross", batch=4, held_lo=2000, held_hi=4096, new_lo=200, new_hi=2048, idle=0, kv_heads=8, group=4, page_size=64, dtype="bf16", lse=False, mix=7),
        # a small batch behind a prompt of 2048 tokens that all have in common
        dict(name="shared_b8_2k", op="shared", batch=8, groups=1, prefix=2048, held_lo=1, held_hi=200, new_lo=1, new_hi=1, idle=0, kv_heads=8, group=4, page_size=64, dtype="bf16", lse=False, mix=8),
        # serving: 64 requests behind a document of 16K tokens, one place idle
        dict(name="shared_b64_16k", op="shared", batch=64, groups=1, prefix=16384, held_lo=100, held_hi=4000, new_lo=1, new_hi=1, idle=1, kv_heads=8, group=4, page_size=64, dtype="bf16", lse=False, mix=9),
        # drafted tokens of requests behind two prompts, the first one's end inside a page
        dict(name="shared_verify", op="shared", batch=24, groups=2, prefix=5000, held_lo=20, held_hi=1500, new_lo=3, new_hi=6, idle=0, kv_heads=8, group=4, page_size=32, dtype="fp16", lse=True, mix=10),
        # many samples of one long context
        dict(name="shared_b256_32k", op="shared", batch=256, groups=1, prefix=32768, held_lo=64, held_hi=2000, new_lo=1, new_hi=1, idle=0, kv_heads=8, group=4, page_size=64, dtype="bf16", lse=False, mix=11),
        # a step that mixes decode and chunks of the requests' own prompts behind the common one
        dict(name="shared_chunks", op="shared", batch=6, groups=1, prefix=6000, held_lo=1, held_hi=500, new_lo=1, new_hi=900, idle=0, kv_heads=8, group=4, page_size=64, dtype="bf16", lse=False, mix=12),
    ]


def _log(rng, lo, hi):
    """a whole number between lo and hi, spread over its logarithm"""
    return min(hi, max(lo, round(max(lo, 1) * (hi / max(lo, 1)) ** rng.random()))) if hi > lo else lo


def draw(rng):
    op = rng.choice(["rotate", "cross", "cross", "shared", "shared", "shared"])
    mix, page_size, dtype, kv_heads = rng.randrange(1, 1 << 30), rng.choice([16, 32, 64, 64, 128, 256]), rng.choice(["bf16", "bf16", "fp16"]), rng.choice([1, 2, 4, 8, 8])
    if op == "rotate":
        tokens = _log(rng, 1, 16384)
        return dict(op=op, tokens=tokens, kv_heads=kv_heads, group=rng.choice([1, 2, 4, 5]), page_size=page_size, dtype=dtype, rotated=rng.choice([128, 128, 96, 64, 32]),
                    interleaved=rng.random() < 0.3, reach=tokens + _log(rng, 100, 100000), mix=mix)
    group = rng.choice([1, 2, 3, 4, 4, 5, 8, 16 if kv_heads <= 4 else 4])
    kind = rng.choice(["decode", "decode", "verify", "chunk"])
    if op == "cross":
        held_hi = _log(rng, 1, 8000)
        if kind == "decode":
            batch, new_lo, new_hi = _log(rng, 1, 200), 1, 1
        elif kind == "verify":
            batch, new_lo, new_hi = _log(rng, 1, 40), rng.randint(1, 4), rng.randint(4, 12)
        else:
            batch, new_lo, new_hi = _log(rng, 1, 8), 1, _log(rng, 20, 2048)
        # at most the largest listed work: padded scores of 4 x 32 heads x 2048 x 4096, padded K of 64 x 16 heads x 4000
        while batch * kv_heads * group * new_hi * held_hi > 4 * 32 * 2048 * 4096 or batch * kv_heads * held_hi > 64 * 16 * 4000:
            if batch > 1:
                batch -= -(-batch // 8)
            else:
                held_hi = held_hi * 7 // 8
        return dict(op=op, batch=batch, held_lo=rng.choice([1, max(held_hi // 10, 1), held_hi]), held_hi=held_hi, new_lo=min(new_lo, new_hi), new_hi=new_hi, idle=rng.choice([0, 0, 1]) if batch > 3 else 0,
                    kv_heads=kv_heads, group=group, page_size=page_size, dtype=dtype, lse=rng.random() < 0.3, mix=mix)
    prefix, held_hi = _log(rng, 20, 50000), _log(rng, 1, 2000)
    if kind == "decode":
        batch, new_lo, new_hi = _log(rng, 2, 256), 1, 1
    elif kind == "verify":
        batch, new_lo, new_hi = _log(rng, 2, 40), rng.randint(1, 4), rng.randint(4, 12)
    else:
        batch, new_lo, new_hi = _log(rng, 2, 8), 1, _log(rng, 20, 900)
    # at most the largest listed work: scores of 256 x 32 heads x 34768, padded K of the requests' own of 256 x 8 heads x 2000
    while batch * kv_heads * group * new_hi * (prefix + held_hi + new_hi) > 256 * 32 * 34768 or batch * kv_heads * (held_hi + new_hi) > 256 * 8 * 2000:
        if batch > 2:
            batch -= -(-batch // 8)
        elif prefix > new_hi:
            prefix = prefix * 7 // 8
        else:
            new_hi = new_hi * 7 // 8
    return dict(op=op, batch=batch, groups=min(rng.choice([1, 1, 2, 5]), batch), prefix=prefix, held_lo=rng.choice([0, held_hi // 10, held_hi]), held_hi=held_hi, new_lo=min(new_lo, new_hi), new_hi=new_hi,
                idle=rng.choice([0, 0, 1]) if batch > 3 else 0, kv_heads=kv_heads, group=group, page_size=page_size, dtype=dtype, lse=rng.random() < 0.3, mix=mix)


def _requests(case):
    """(tokens held beside the common ones, new tokens) of every request; the first has the largest of both, the last `idle` have none"""
    rng, n, idle = random.Random(case["mix"]), case["batch"], case["idle"]
    held = [case["held_hi"]] + [_log(rng, case["held_lo"], case["held_hi"]) for _ in range(n - 1)]
    new = [case["new_hi"]] + [_log(rng, case["new_lo"], case["new_hi"]) for _ in range(n - 1)]
    for b in range(n - idle, n):
        held[b], new[b] = None, 1 if case["new_hi"] == case["new_lo"] == 1 else 0  # (an idle place of a decode batch has a query and no tokens)
    return held, new


def _shared(case):
    """where the groups of requests begin, and end; the tokens that each one's requests have in common"""
    rng, n = random.Random(case["mix"] + 1), case["batch"]
    cuts = sorted(rng.sample(range(1, n), case["groups"] - 1))
    common = [case["prefix"]] + [_log(rng, case["prefix"] // 8 + 1, case["prefix"]) for _ in cuts]
    return [0] + cuts + [n], common


def _lengths(case):
    """tokens that each request sees: a cross attention's states; common, held and new tokens"""
    held, new = _requests(case)
    if case["op"] == "cross":
        return [h or 0 for h in held]
    cuts, common = _shared(case)
    return [0 if held[b] is None else common[g] + held[b] + new[b] for g in range(len(common)) for b in range(cuts[g], cuts[g + 1])]


def work(case):
    per_token = 2 * case["kv_heads"] * (D // 2 + D // 16)
    if case["op"] == "rotate":  # q, k, v, the tables' rows; q rotated, the codes; and the codes and values of the read that returns them
        n, heads = case["tokens"], case["kv_heads"] * case["group"]
        rows = 4 * case["rotated"] * n
        return {"bytes": n * (2 * 2 * heads * D + 2 * 2 * 2 * case["kv_heads"] * D + 2 * per_token + 12) + rows, "flops": 0}
    heads, P = case["kv_heads"] * case["group"], case["page_size"]
    _, new = _requests(case)
    lengths = _lengths(case)
    queries, tokens = sum(new), sum(lengths)
    if case["op"] == "cross":
        pairs = sum(a * n for a, n in zip(lengths, new))
    else:
        cuts, common = _shared(case)
        pairs = sum(n * (a - n) + n * (n + 1) // 2 for a, n in zip(lengths, new) if a > 0)
        for g, c in enumerate(common):  # the common pages are read once
            tokens -= (sum(a > 0 for a in lengths[cuts[g] : cuts[g + 1]]) - 1) * (c // P * P)
    entries = sum(-(-a // P) for a in lengths)
    return {"bytes": tokens * per_token + 2 * 2 * queries * heads * D + (4 * queries * heads if case["lse"] else 0) + 4 * entries + 8 * len(lengths), "flops": 4 * D * heads * pairs}


# ---- the format, plainly ------------------------------------------------------------------------------------------------------
def _quantise(x, factor):
    """x [..., heads, 128] -> codes uint8 [..., heads, 64], scales uint8 [..., heads, 8]"""
    y = (x.float() * (1.0 / factor)[:, None]).unflatten(-1, (D // 16, 16))
    scale = (y.abs().amax(-1, keepdim=True) * 0.1666666716337204).clamp_(max=448.0).to(torch.float8_e4m3fn)
    s = scale.float()
    m = torch.where(s > 0, y.abs() / s, 0.0)
    code = (m > 0.25).to(torch.uint8)  # halfway cases go to the even code
    for above, edge in ((False, 0.75), (True, 1.25), (False, 1.75), (True, 2.5), (False, 3.5), (True, 5.0)):
        code += (m > edge) if above else (m >= edge)
    code += torch.signbit(y).to(torch.uint8) * 8
    code = code.flatten(-2)
    return code[..., 0::2] + code[..., 1::2] * 16, scale.view(torch.uint8).squeeze(-1)


def _values(codes, scales, factor):
    """codes uint8 [..., 64], scales uint8 [..., 8] and a factor that broadcasts to [..., 1] -> float [..., 128]"""
    code = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    c = (code & 7).float()
    x = c * 0.5  # 0, 0.5, 1, 1.5, 2, 3, 4, 6
    x.add_((c - 4).clamp_(min=0), alpha=0.5).add_((c - 6).clamp_(min=0))
    del c
    x.mul_((code >> 3).float().mul_(-2).add_(1))
    x.unflatten(-1, (D // 16, 16)).mul_(scales.view(torch.float8_e4m3fn).float()[..., None])
    return x.mul_(factor)


def _fields(units):
    """a pool's bytes as K codes, V codes, K scales, V scales: views [pages, heads, blocks, 16, 64 or 8]"""
    return (units[..., :1024].unflatten(-1, (16, 64)), units[..., 1024:2048].unflatten(-1, (16, 64)),
            units[..., 2048:2176].unflatten(-1, (16, 8)), units[..., 2176:].unflatten(-1, (16, 8)))


def _token_fields(units, slots):
    """the fields of single tokens, [tokens, heads, 64 or 8]"""
    P = units.shape[2] * BLOCK
    page, block, row = slots // P, slots % P // BLOCK, slots % BLOCK
    return [f[page, :, block, row] for f in _fields(units)]


def _write(units, slots, codes_k, codes_v, scales_k, scales_v):
    P = units.shape[2] * BLOCK
    page, block, row = slots // P, slots % P // BLOCK, slots % BLOCK
    for f, x in zip(_fields(units), (codes_k, codes_v, scales_k, scales_v)):
        f[page, :, block, row] = x


def _rounded(x, dtype):
    """64-bit values rounded once to 16 bits: through 32 bits with the last bit set where they are not exact, so that no second rounding meets a halfway case"""
    y = x.float()
    bits, off = y.view(torch.int32), x - y.double()
    move = (off != 0) & (bits & 1 == 0) & torch.isfinite(y)
    away = (off > 0) == (y > 0)  # from zero
    return torch.where(move, torch.where(away, bits + 1, bits - 1), bits).view(torch.float32).to(dtype)


def _rotate(x, rows, interleaved):
    """x [tokens, heads, 128], rows [tokens, R] (cosines, sines), in the bits of `rows`"""
    R = rows.shape[1]
    x = x.to(rows.dtype)
    c, s = (y[:, None] for y in (rows[:, : R // 2], rows[:, R // 2 :]))
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if interleaved else (x[..., : R // 2], x[..., R // 2 : R])
    turned = (a * c - b * s, b * c + a * s)
    turned = torch.stack(turned, -1).flatten(-2) if interleaved else torch.cat(turned, -1)
    return torch.cat((turned, x[..., R:]), -1)


# ---- inputs -------------------------------------------------------------------------------------------------------------------
def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, dtype=torch.bfloat16, device="cuda")


def _pool(gen, pages, kv_heads, page_size, filled=True):
    """units of `pages` pages; K and V are N(0, 1), 4 of the 128 channels of every head times 8 in K, V at a sixteenth"""
    units = torch.empty((pages, kv_heads, page_size // BLOCK, BLOCK_BYTES), dtype=torch.uint8, device="cuda")
    k_scale = torch.exp2(torch.randint(-1, 2, (kv_heads,), generator=gen, device="cuda").float())
    v_scale = 0.05 + 0.1 * torch.rand((kv_heads,), generator=gen, device="cuda")
    order = torch.rand((kv_heads, D), generator=gen, device="cuda").argsort(-1)
    loud = torch.where(order < 4, 8.0, 1.0).to(torch.bfloat16)
    if not filled:
        units.fill_(255)
        return units, k_scale, v_scale, loud
    step = max(1, (1 << 28) // (kv_heads * page_size * D))
    for p in range(0, pages, step):
        n = min(step, pages - p)
        kc, vc, ks, vs = (f[p : p + n] for f in _fields(units))
        for codes, scales, factor, gain in ((kc, ks, k_scale, loud), (vc, vs, v_scale, 0.0625)):
            x = _normal(gen, n, page_size, kv_heads, D) * gain
            c, s = _quantise(x, factor)
            codes.copy_(c.unflatten(1, (-1, 16)).permute(0, 3, 1, 2, 4))
            scales.copy_(s.unflatten(1, (-1, 16)).permute(0, 3, 1, 2, 4))
    return units, k_scale, v_scale, loud


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _tables(gen, lengths, page_size, width, spare=3):
    """a block table of pages in no order; places that hold nothing carry -1; also the number of pages"""
    counts = [-(-max(n, 0) // page_size) for n in lengths]
    total = sum(counts)
    order = torch.randperm(total + spare, generator=gen, device="cuda").to(torch.int32)
    column = torch.arange(width, device="cuda")[None]
    count = _int(counts)[:, None]
    first = count.cumsum(0) - count
    table = torch.where(column < count, order[(first + column).clamp_(max=total + spare - 1)], -1).to(torch.int32)
    return table, total + spare


def _angles(reach, rotated):
    """cosines and sines of positions 0 .. reach - 1, float32 [reach, rotated]: frequencies 10000^(-2 i / rotated)"""
    angle = torch.arange(reach, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (-torch.arange(0, rotated, 2, dtype=torch.float64, device="cuda") / rotated)
    return torch.cat((angle.cos(), angle.sin()), -1).float()


def _prepare_rotate(case, gen):
    rng, n, P, H, R = random.Random(case["mix"]), case["tokens"], case["page_size"], case["kv_heads"], case["rotated"]
    if n <= 64:  # one token of each of n requests, anywhere
        lengths, first = [1] * n, [rng.randrange(case["reach"]) for _ in range(n)]
    else:  # chunks of a few requests
        cuts = sorted(rng.randrange(n + 1) for _ in range(3))
        lengths = [b - a for a, b in zip([0] + cuts, cuts + [n])]
        first = [rng.randrange(case["reach"] - m + 1) for m in lengths]
    table, pages = _tables(gen, [m + P for m in lengths], P, -(-(max(lengths) + P) // P))  # (a chunk begins inside a page)
    row = torch.repeat_interleave(torch.arange(len(lengths), device="cuda"), _int(lengths), output_size=n)
    i = torch.arange(n, device="cuda") - (_int(lengths).cumsum(0) - _int(lengths))[row]
    at = i + _int([f % P for f in first])[row]
    slots = (table[row, at // P].long() * P + at % P).to(torch.int32)
    positions = (i + _int(first)[row]).to(torch.int32)
    units, k_scale, v_scale, loud = _pool(gen, pages, H, P, filled=False)
    heads, dtype = H * case["group"], _DTYPES[case["dtype"]]
    rows = _normal(gen, n, heads + 2 * H, D)  # of a fused projection: queries, keys, values
    rows[:, heads : heads + H] *= loud
    rows[:, heads + H :] *= 0.0625
    q, k, v = rows.to(dtype).split([heads, H, H], 1)
    return dict(units=units, k_scale=k_scale, v_scale=v_scale, slots=slots, positions=positions, cos_sin=_angles(case["reach"], R), q=q, k=k, v=v, dtype=dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "rotate":
        return {"case": case, **_prepare_rotate(case, gen)}
    P, H = case["page_size"], case["kv_heads"]
    _, new = _requests(case)
    lengths = _lengths(case)
    width = max(-(-max(lengths) // P), 1)
    state = {"case": case}
    if case["op"] == "cross":
        table, pages = _tables(gen, lengths, P, width)
    else:
        cuts, common = _shared(case)
        whole = [c // P for c in common]  # (the page in which a common beginning ends is a request's own)
        member = [g for g in range(len(common)) for _ in range(cuts[g], cuts[g + 1])]
        mine, pages = _tables(gen, [a - whole[g] * P for a, g in zip(lengths, member)], P, width, spare=3 + sum(whole))
        # (the pages that the requests' own do not take serve as the common ones)
        taken = torch.zeros(pages, dtype=torch.bool, device="cuda")
        taken[mine[mine >= 0].long()] = True
        rest = (~taken).nonzero().view(-1).to(torch.int32)
        table, first = torch.full_like(mine, -1), 0
        for g, n in enumerate(whole):
            rows = table[cuts[g] : cuts[g + 1]]
            rows[:, :n] = rest[first : first + n]
            rows[:, n:] = mine[cuts[g] : cuts[g + 1], : width - n]
            first += n
        table[_int(lengths) == 0] = -1
        state.update(groups=None if len(common) == 1 else _int(cuts), shared=_int(common), cuts=cuts, whole=whole)
    units, k_scale, v_scale, _ = _pool(gen, pages, H, P)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    q = _normal(gen, starts[-1], H * case["group"], D).to(_DTYPES[case["dtype"]])
    state.update(units=units, k_scale=k_scale, v_scale=v_scale, q=q, table=table, lengths=_int(lengths), starts=None if case["new_hi"] == case["new_lo"] == 1 else _int(starts), longest=max(new))
    return state


# ---- the operators, plainly -----------------------------------------------------------------------------------------------------
def _attend(s, lo, hi, first, causal):
    """requests lo .. hi - 1, whose first `first` pages are the same: (rows of q, outputs, log-sum-exps)"""
    case, q, units, P = s["case"], s["q"].float(), s["units"], s["case"]["page_size"]
    H, G, B, n = case["kv_heads"], case["group"], hi - lo, s["longest"]
    table, lengths = s["table"][lo:hi].long(), s["lengths"][lo:hi].long()
    starts = torch.arange(case["batch"] + 1, device=q.device) if s["starts"] is None else s["starts"].long()
    starts = starts[lo : hi + 1]
    count = starts[1:] - starts[:-1]
    i = torch.arange(n, device=q.device)
    at = (starts[:-1, None] + i).clamp_(max=max(q.shape[0] - 1, 0))
    last = (lengths - count)[:, None] + i if causal else (lengths - 1)[:, None].expand(B, n)  # the last token that a query sees
    rows = q[at].view(B, n, H, G, D).permute(0, 2, 3, 1, 4)  # [B, H, G, n, 128]

    def scores_of(rows, table, token0):
        """rows [B or 1, H, rows, 128] -> their scores, and the pages' values"""
        kc, vc, ks, vs = (f[table.clamp(min=0)].transpose(1, 2).flatten(2, 4) for f in _fields(units))  # [., H, tokens, 64 or 8]
        scores = torch.matmul(rows, _values(kc, ks, s["k_scale"][:, None, None]).transpose(2, 3)).mul_(1 / math.sqrt(D))
        values = _values(vc, vs, s["v_scale"][:, None, None])
        token = token0 + torch.arange(scores.shape[-1], device=q.device)
        return scores, values, token

    parts = []
    if first:
        scores, values, token = scores_of(rows.permute(1, 0, 2, 3, 4).reshape(1, H, B * G * n, D), table[:1, :first], 0)
        parts.append((scores.view(H, B, G, n, -1).transpose(0, 1), values, token))  # [B, H, G, n, tokens]
    if table.shape[1] > first:
        scores, values, token = scores_of(rows.reshape(B, H, G * n, D), table[:, first:], first * P)
        values = torch.where(token[:, None] < lengths[:, None, None, None], values, 0.0)  # (pages end behind the last token)
        parts.append((scores.view(B, H, G, n, -1), values, token))
    for scores, _, token in parts:
        scores.masked_fill_(~(token <= last[:, :, None])[:, None, None], -math.inf)
    top = parts[0][0].amax(-1, keepdim=True)
    for scores, _, _ in parts[1:]:
        top = torch.maximum(top, scores.amax(-1, keepdim=True))
    top = torch.where(torch.isinf(top), 0.0, top)
    mass, out = torch.zeros_like(top), torch.zeros((B, H, G, n, D), device=q.device)
    for scores, values, _ in parts:
        scores.sub_(top).exp_()
        mass += scores.sum(-1, keepdim=True)
        if values.shape[0] == B:
            out += torch.matmul(scores.reshape(B, H, G * n, -1), values).view(B, H, G, n, D)
        else:
            out += torch.matmul(scores.transpose(0, 1).reshape(1, H, B * G * n, -1), values).view(H, B, G, n, D).transpose(0, 1)
    out = torch.where(mass > 0, out / mass, 0.0)
    here = (i < count[:, None]).view(-1).nonzero().view(-1)
    return out.permute(0, 3, 1, 2, 4).reshape(B * n, H * G, D)[here].to(s["q"].dtype), (top + mass.log()).squeeze(-1).permute(0, 3, 1, 2).reshape(B * n, H * G)[here]


def run(state):
    case = state["case"]
    if case["op"] == "rotate":
        slots, dtype = state["slots"], state["dtype"]
        if own:
            from mlops_b200.attention import paged
            cache = paged.PagedCache(state["units"], state["k_scale"], state["v_scale"])
            q = paged.append_rotated(cache, state["q"], state["k"], state["v"], slots, state["positions"], state["cos_sin"], interleaved=case["interleaved"])
            k, v = paged.read(cache, slots, dtype)  # (what the cache now holds for the tokens)
            return {"q": q, "k": k, "v": v}
        rows = state["cos_sin"][state["positions"].long()]
        q = _rotate(state["q"], rows, case["interleaved"]).to(dtype)
        k = _rounded(_rotate(state["k"], rows.double(), case["interleaved"]), dtype)
        kc, ks = _quantise(k, state["k_scale"])
        vc, vs = _quantise(state["v"], state["v_scale"])
        _write(state["units"], slots.long(), kc, vc, ks, vs)
        kc, vc, ks, vs = _token_fields(state["units"], slots.long())
        return {"q": q, "k": _values(kc, ks, state["k_scale"][:, None]).to(dtype), "v": _values(vc, vs, state["v_scale"][:, None]).to(dtype)}
    if own:
        from mlops_b200.attention import paged
        cache = paged.PagedCache(state["units"], state["k_scale"], state["v_scale"])
        if case["op"] == "cross":
            result = paged.cross_attend(state["q"], cache, state["table"], state["lengths"], state["starts"], return_lse=case["lse"])
        else:
            result = paged.attend_shared(state["q"], cache, state["table"], state["lengths"], state["starts"], state["groups"], state["shared"], return_lse=case["lse"])
        return {"out": result[0], "lse": result[1]} if case["lse"] else {"out": result}
    if case["op"] == "cross":
        parts = [_attend(state, 0, case["batch"], 0, False)]
    else:
        cuts = state["cuts"]
        parts = [_attend(state, lo, hi, first, True) for lo, hi, first in zip(cuts, cuts[1:], state["whole"])]
    out, lse = (torch.cat(x) for x in zip(*parts))
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}


# ---- in 64 bits -------------------------------------------------------------------------------------------------------------------
def _stored(codes, scales, factor):
    """values in 64 bits by tables: [..., 64] and [..., 8] bytes, the head's factor"""
    level = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    level = torch.tensor(level + [-x for x in level], dtype=torch.float64, device=codes.device)
    step = [(-1 if b >> 7 else 1) * (math.ldexp(8 + (b & 7), (b >> 3 & 15) - 10) if b >> 3 & 15 else math.ldexp(b & 7, -9)) for b in range(256)]
    step[127] = step[255] = math.nan
    step = torch.tensor(step, dtype=torch.float64, device=codes.device)
    byte = codes.int()
    x = torch.empty((*codes.shape[:-1], D), dtype=torch.float64, device=codes.device)
    x[..., 0::2], x[..., 1::2] = level[byte % 16], level[byte // 16]
    return x * step[scales.int()].repeat_interleave(16, -1) * factor


def _nearest(x, levels):
    """the member of the ascending `levels` nearest to x; halfway, the one with the even index"""
    hi = torch.searchsorted(levels, x).clamp_(1, levels.numel() - 1)
    below, above = x - levels[hi - 1], levels[hi] - x
    up = (above < below) | ((above == below) & (hi % 2 == 0))
    return torch.where(up, levels[hi], levels[hi - 1])


def _held(x, factor):
    """what the cache holds of 16-bit x [tokens, heads, 128]: each 32-bit operation of the format in 64 bits and rounded"""
    e2m1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=x.device)
    e4m3 = torch.tensor([math.ldexp(8 + (b & 7), (b >> 3) - 10) if b >> 3 else math.ldexp(b, -9) for b in range(127)], dtype=torch.float64, device=x.device)
    g = factor.double()[:, None, None]
    y = (x.double().unflatten(-1, (8, 16)) * (1 / g).float().double()).float().double()
    sixth = torch.tensor(1 / 6, dtype=torch.float32).double().item()
    s = _nearest((y.abs().amax(-1, keepdim=True) * sixth).float().double().clamp_(max=448.0), e4m3)
    c = _nearest((y.abs() / torch.where(s > 0, s, 1.0)).float().double().clamp_(max=6.0), e2m1)
    return (torch.where(s > 0, c * torch.sign(y) * s, 0.0) * g).flatten(-2)


def _nearest16(x, dtype):
    """64-bit x rounded once to 16 bits: its significand as a whole number of the type's bits, halfway to even"""
    _, e = torch.frexp(x)
    bits, least = (8, -133) if dtype == torch.bfloat16 else (11, -24)
    unit = torch.exp2((e.double() - bits).clamp(min=least))
    return torch.round(x / unit) * unit


def exact(case, seed):
    s = prepare(case, seed)
    H, P = case["kv_heads"], case["page_size"]
    if case["op"] == "rotate":
        R, turned = case["rotated"], []
        angle = s["cos_sin"].double()[s["positions"].long()][:, None]
        for x in (s["q"], s["k"]):
            y = x.double().clone()
            for i in range(R // 2):
                a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + R // 2)
                c, d = angle[..., i], angle[..., R // 2 + i]
                y[..., a], y[..., b] = x[..., a].double() * c - x[..., b].double() * d, x[..., b].double() * c + x[..., a].double() * d
            turned.append(y)
        return {"q": turned[0], "k": _held(_nearest16(turned[1], s["dtype"]), s["k_scale"]), "v": _held(s["v"], s["v_scale"])}
    kc, vc, ks, vs = _fields(s["units"])
    gk, gv = s["k_scale"].double(), s["v_scale"].double()
    _, new = _requests(case)
    heads, lengths = H * case["group"], _lengths(case)
    out = torch.zeros((sum(new), heads, D), dtype=torch.float64, device="cuda")
    lse = torch.full((sum(new), heads), -math.inf, dtype=torch.float64, device="cuda")
    first = 0
    for b, (length, n) in enumerate(zip(lengths, new)):
        if length > 0 and n > 0:
            pages = s["table"][b, : -(-length // P)].long()
            limit = torch.arange(length - n, length, device="cuda")[:, None] if case["op"] == "shared" else torch.full((n, 1), length, device="cuda")
            for x in range(H):
                k, v = (_stored(c[pages, x].reshape(-1, 64)[:length], t[pages, x].reshape(-1, 8)[:length], g[x]) for c, t, g in ((kc, ks, gk), (vc, vs, gv)))
                mine = slice(x * case["group"], (x + 1) * case["group"])
                score = torch.einsum("nhd,td->nht", s["q"][first : first + n, mine].double(), k) / math.sqrt(D)
                score = score.masked_fill_(torch.arange(length, device="cuda") > limit[:, :, None], -math.inf)
                lse[first : first + n, mine] = torch.logsumexp(score, -1)
                out[first : first + n, mine] = (score - lse[first : first + n, mine, None]).exp_() @ v
        first += n
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}
