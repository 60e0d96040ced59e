"""The operators of the paged 4-bit cache (`mlops_b200.attention.paged`) as cases that can be timed and compared.

An engine that serves requests of many lengths keeps their K / V in pages of a common pool. In every step it gives the
requests pages for their new tokens (`assign`), writes the new K / V into them in 4 bits (`append`) and attends over what
the pages hold (`attend`); now and then it takes stored tokens out again (`read`: a prefix that moves to another pool, or to
an attention that wants 16 bits). The cases go through these four calls; `own` False computes the same in elementary
torch operations, in 32 bits.

The pool: uint8 [pages, KV heads, page_size / 16, 2304]; the 2304 bytes of a block hold 16 tokens of one KV head:
K codes [16][64], V codes [16][64], K scales [16][8], V scales [16][8]. A code is E2M1 (sign, two bits of exponent, one of
mantissa), channel 2 i in the low and 2 i + 1 in the high half of byte i; a scale is E4M3 and serves 16 channels; the value is
code * scale * k_scale[head] (v_scale for V).

A case's lengths follow from its `mix`, so that its work is known; its values follow from the seed.
"""
import math
import random

import torch

own = False

D, BLOCK, BLOCK_BYTES = 128, 16, 2304
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # an engine's decode step: one new token for each of 64 requests of 1K to 64K tokens; launches and latency count
        dict(name="assign_b64", op="assign", batch=64, held_lo=1024, held_hi=65536, new_lo=1, new_hi=1, page_size=64, mix=1),
        # a busy step: 500 requests, most in decode, some with a chunk of a prompt, small pages
        dict(name="assign_b500_mixed", op="assign", batch=500, held_lo=1, held_hi=16384, new_lo=1, new_hi=512, page_size=16, mix=2),
        # the decode step's K / V of 64 requests, slices of the fused projection's rows
        dict(name="append_64", op="append", tokens=64, kv_heads=8, group=4, page_size=64, dtype="bf16", mix=3),
        # four prompts of 8192 tokens written at once
        dict(name="append_32k", op="append", tokens=32768, kv_heads=8, group=4, page_size=64, dtype="bf16", mix=4),
        # a short prefix taken out, an odd length
        dict(name="read_999", op="read", tokens=999, kv_heads=4, page_size=32, dtype="fp16", mix=5),
        # a context of 64K tokens taken out
        dict(name="read_64k", op="read", tokens=65536, kv_heads=8, page_size=128, dtype="bf16", mix=6),
        # the smallest decode: one request, a short context
        dict(name="decode_b1_4k", op="attend", batch=1, held_lo=4095, held_hi=4095, new_lo=1, new_hi=1, idle=0, kv_heads=8, group=2, page_size=64, dtype="bf16", lse=False, mix=7),
        # one request with a long context; its log-sum-exp is asked for, to be joined with another part of the sequence
        dict(name="decode_b1_128k", op="attend", batch=1, held_lo=131071, held_hi=131071, new_lo=1, new_hi=1, idle=0, kv_heads=8, group=4, page_size=64, dtype="bf16", lse=True, mix=8),
        # mixed serving: contexts of 1K to 64K tokens in one batch, two of its places idle
        dict(name="serving_b64", op="attend", batch=64, held_lo=1023, held_hi=65535, new_lo=1, new_hi=1, idle=2, kv_heads=8, group=4, page_size=64, dtype="bf16", lse=False, mix=9),
        # drafted tokens checked against long contexts, small pages
        dict(name="verify_b16", op="attend", batch=16, held_lo=5000, held_hi=16000, new_lo=3, new_hi=6, idle=0, kv_heads=8, group=4, page_size=16, dtype="fp16", lse=False, mix=10),
        # a step that mixes decode, drafted tokens and chunks of prompts
        dict(name="mixed_b8", op="attend", batch=8, held_lo=500, held_hi=6000, new_lo=1, new_hi=1500, idle=0, kv_heads=8, group=4, page_size=64, dtype="bf16", lse=False, mix=11),
        # two whole prompts of 8192 tokens
        dict(name="prompts_2x8k", op="attend", batch=2, held_lo=0, held_hi=0, new_lo=8192, new_hi=8192, idle=0, kv_heads=8, group=4, page_size=64, dtype="bf16", lse=False, mix=12),
    ]


def _log(rng, lo, hi):
    """a whole number between lo and hi, spread over its logarithm"""
    return min(hi, max(lo, round(max(lo, 1) * (hi / max(lo, 1)) ** rng.random()))) if hi > lo else lo


def draw(rng):
    op = rng.choice(["assign", "append", "read", "attend", "attend", "attend", "attend"])
    mix, page_size = rng.randrange(1, 1 << 30), rng.choice([16, 32, 64, 64, 128, 256])
    if op == "assign":
        batch = _log(rng, 1, 2048)
        new_hi = rng.choice([1, 1, 8, _log(rng, 16, 4096)])
        held_hi = _log(rng, 16, 65536)
        return dict(op=op, batch=batch, held_lo=rng.choice([0, 1, held_hi // 16]), held_hi=held_hi, new_lo=rng.choice([0, 1]), new_hi=new_hi, page_size=page_size, mix=mix)
    kv_heads, dtype = rng.choice([1, 2, 4, 8, 8]), rng.choice(["bf16", "bf16", "fp16"])
    if op == "append":
        return dict(op=op, tokens=_log(rng, 1, 32768), kv_heads=kv_heads, group=rng.choice([1, 2, 4, 5]), page_size=page_size, dtype=dtype, mix=mix)
    if op == "read":
        return dict(op=op, tokens=_log(rng, 1, 65536), kv_heads=kv_heads, page_size=page_size, dtype=dtype, mix=mix)
    group = rng.choice([1, 2, 3, 4, 4, 5, 8, 16 if kv_heads <= 4 else 4])
    kind = rng.choice(["decode", "decode", "verify", "chunk"])
    if kind == "decode":
        batch, held_hi, new_lo, new_hi = _log(rng, 1, 200), _log(rng, 30, 131000), 1, 1
    elif kind == "verify":
        batch, held_hi, new_lo, new_hi = _log(rng, 1, 40), _log(rng, 100, 30000), rng.randint(1, 4), rng.randint(4, 12)
    else:
        batch, held_hi, new_lo, new_hi = _log(rng, 1, 12), _log(rng, 1, 16000), 1, _log(rng, 20, 8192)
    # at most the largest listed work: padded scores of 2 x 32 heads x 8192 x 8192, padded K / V of 64 x 8 heads x 65536
    while batch * kv_heads * group * new_hi * (held_hi + new_hi) > 64 * 8192 * 8192 or batch * kv_heads * (held_hi + new_hi) > 24 * 8 * 65536:
        if batch > 1:
            batch -= -(-batch // 8)
        elif held_hi > new_hi:
            held_hi = held_hi * 7 // 8
        else:
            new_hi = new_hi * 7 // 8
    held_lo = rng.choice([0, held_hi // 10, held_hi // 2, held_hi])
    return dict(op="attend", batch=batch, held_lo=held_lo, held_hi=held_hi, new_lo=min(new_lo, new_hi), new_hi=new_hi, idle=rng.choice([0, 0, 1]) if batch > 3 else 0,
                kv_heads=kv_heads, group=group, page_size=page_size, dtype=dtype, lse=rng.random() < 0.3, mix=mix)


def _requests(case):
    """(tokens held, new tokens) of every request; the first has the largest of both, the last `idle` have none"""
    rng, n, idle = random.Random(case["mix"]), case["batch"], case.get("idle", 0)
    held = [case["held_hi"]] + [_log(rng, case["held_lo"], case["held_hi"]) for _ in range(n - 1)]
    new = [case["new_hi"]] + [_log(rng, case["new_lo"], case["new_hi"]) for _ in range(n - 1)]
    decode = case["new_hi"] == case["new_lo"] == 1
    for b in range(n - idle, n):
        held[b], new[b] = (-1, 1) if decode else (0, 0)  # (an idle place of a decode batch has a query and no tokens)
    return held, new


def work(case):
    if case["op"] == "assign":
        held, new = _requests(case)
        total, P = sum(new), case["page_size"]
        pages = sum(-(-(h + n) // P) - -(-h // P) for h, n in zip(held, new))
        return {"bytes": 16 * len(held) + 8 * total + 8 * pages + 48, "flops": 0}
    per_token = 2 * case["kv_heads"] * (D // 2 + D // 16)
    if case["op"] == "append":  # the new K / V, their codes; and the codes and values of the read that returns them
        n = case["tokens"]
        return {"bytes": n * (2 * 2 * case["kv_heads"] * D * 2 + 2 * per_token + 8), "flops": 0}
    if case["op"] == "read":
        n = case["tokens"]
        return {"bytes": n * (2 * case["kv_heads"] * D * 2 + per_token + 4), "flops": 0}
    held, new = _requests(case)
    heads = case["kv_heads"] * case["group"]
    tokens, queries = sum(h + n for h, n in zip(held, new)), sum(new)
    pairs = sum(n * h + n * (n + 1) // 2 for h, n in zip(held, new) if h >= 0)
    pages = sum(-(-(h + n) // case["page_size"]) for h, n in zip(held, new))
    return {"bytes": tokens * per_token + 2 * 2 * queries * heads * D + (4 * queries * heads if case["lse"] else 0) + 4 * pages + 8 * len(held), "flops": 4 * D * heads * pairs}


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


def _slots(gen, case):
    """slots of `tokens` tokens of a few requests, pages in no order, and the number of pages"""
    rng, n, P = random.Random(case["mix"]), case["tokens"], case["page_size"]
    cuts = sorted(rng.randrange(n + 1) for _ in range(min(3, n - 1))) if n > 64 else list(range(1, n))
    lengths = [b - a for a, b in zip([0] + cuts, cuts + [n])]
    table, pages = _tables(gen, lengths, P, -(-n // P))
    first = _int([rng.randrange(P) if n <= 64 else 0 for _ in lengths])  # (single tokens lie anywhere in their page)
    row = torch.repeat_interleave(torch.arange(len(lengths), device="cuda"), _int(lengths), output_size=n)
    pos = torch.arange(n, device="cuda") - (_int(lengths).cumsum(0) - _int(lengths))[row] + first[row]
    return (table[row, pos // P].long() * P + pos % P).to(torch.int32), pages


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    if case["op"] == "assign":
        held, new = _requests(case)
        P, batch = case["page_size"], len(held)
        width = -(-(case["held_hi"] + case["new_hi"]) // P) + 1
        table, taken = _tables(gen, held, P, width, spare=0)
        free = sum(-(-(h + n) // P) - -(-h // P) for h, n in zip(held, new)) + 37
        ring = (torch.randperm(free, generator=gen, device="cuda") + taken).to(torch.int32)
        ring = torch.cat((torch.full((taken,), -1, dtype=torch.int32, device="cuda"), ring)).roll(free // 2)  # (the free pages wrap around its end)
        head = taken + free // 2
        cursor = torch.tensor([head, head + free, 0], dtype=torch.int64, device="cuda")
        state.update(table=table, held=_int(held), new=_int(new), ring=ring, cursor=cursor, tokens=sum(new))
        return state
    dtype, H = _DTYPES[case["dtype"]], case["kv_heads"]
    if case["op"] in ("append", "read"):
        slots, pages = _slots(gen, case)
        units, k_scale, v_scale, loud = _pool(gen, pages, H, case["page_size"], filled=case["op"] == "read")
        state.update(units=units, k_scale=k_scale, v_scale=v_scale, slots=slots, dtype=dtype)
        if case["op"] == "append":  # rows of a fused projection: queries, keys, values
            q = H * case["group"]
            rows = _normal(gen, case["tokens"], q + 2 * H, D)
            rows[:, q : q + H] *= loud
            rows[:, q + H :] *= 0.0625
            rows = rows.to(dtype)
            state.update(k=rows[:, q : q + H], v=rows[:, q + H :])
    else:
        held, new = _requests(case)
        lengths = [h + n for h, n in zip(held, new)]
        table, pages = _tables(gen, lengths, case["page_size"], -(-max(lengths) // case["page_size"]))
        units, k_scale, v_scale, _ = _pool(gen, pages, H, case["page_size"])
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        q = _normal(gen, starts[-1], H * case["group"], D).to(dtype)
        state.update(units=units, k_scale=k_scale, v_scale=v_scale, q=q, table=table, lengths=_int(lengths),
                     starts=None if case["new_hi"] == case["new_lo"] == 1 else _int(starts), longest=max(new))
    return state


# ---- the operators, plainly -----------------------------------------------------------------------------------------------------
def _assign(table, held, added, ring, cursor, P, tokens):
    starts = torch.nn.functional.pad(added.cumsum(0), (1, 0))
    lengths = held + added
    first = (held + P - 1) // P
    need = (lengths + P - 1) // P - first
    before = need.cumsum(0) - need
    i = torch.arange(tokens, device=held.device)
    row = torch.searchsorted(starts[1:].contiguous(), i, right=True).clamp_(max=held.numel() - 1)
    pos = held[row] + i - starts[row]
    column = pos // P
    nth = before[row] + column - first[row]
    left = cursor[1] - cursor[0]
    fresh = torch.where(nth < left, ring[(cursor[0] + nth) % ring.numel()], -1)
    page = torch.where(column < first[row], table[row, column], fresh)
    slots = torch.where((i < starts[-1]) & (page >= 0), page * P + pos % P, -1)
    opens = (i < starts[-1]) & (pos % P == 0)
    at = (row * table.shape[1] + column)[opens]
    table.view(-1)[at] = page[opens].to(torch.int32)
    total = need.sum()
    taken = torch.minimum(total, left)
    moved = torch.stack((cursor[0] + taken, cursor[1], total - taken))
    return {"table": table, "slots": slots.to(torch.int32), "positions": pos.to(torch.int32), "starts": starts.to(torch.int32), "lengths": lengths, "cursor": moved}


def _attend(s):
    case, q, table, lengths, units = s["case"], s["q"].float(), s["table"].long(), s["lengths"].long(), s["units"]
    H, G, B, n = case["kv_heads"], case["group"], case["batch"], s["longest"]
    starts = torch.arange(B + 1, device=q.device) if s["starts"] is None else s["starts"].long()
    count = starts[1:] - starts[:-1]
    i = torch.arange(n, device=q.device)
    at = (starts[:-1, None] + i).clamp_(max=max(q.shape[0] - 1, 0))
    # rows of one KV head: its group's heads, then the request's queries
    rows = q[at].view(B, n, H, G, D).permute(0, 2, 3, 1, 4).reshape(B, H, G * n, D)
    kc, vc, ks, vs = (f[table.clamp(min=0)].transpose(1, 2).flatten(2, 4) for f in _fields(units))  # [B, H, tokens, 64 or 8]
    keys = _values(kc, ks, s["k_scale"][:, None, None])
    scores = torch.matmul(rows, keys.transpose(2, 3)).mul_(1 / math.sqrt(D)).view(B, H, G, n, -1)
    del keys, kc, ks
    token = torch.arange(scores.shape[-1], device=q.device)
    seen = token <= (lengths - count)[:, None, None] + i[:, None]  # [B, n, tokens]
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), 0.0, top)
    scores.sub_(top).exp_()
    mass = scores.sum(-1, keepdim=True)
    values = _values(vc, vs, s["v_scale"][:, None, None])
    values = torch.where(token[:, None] < lengths[:, None, None, None], values, 0.0)  # (pages end behind the last token)
    out = torch.matmul(scores.view(B, H, G * n, -1), values).view(B, H, G, n, D)
    out = torch.where(mass > 0, out / mass, 0.0)
    here = (i < count[:, None]).view(-1).nonzero().view(-1)
    result = {"out": out.permute(0, 3, 1, 2, 4).reshape(B * n, H * G, D)[here].to(s["q"].dtype)}
    if case["lse"]:
        result["lse"] = (top + mass.log()).squeeze(-1).permute(0, 3, 1, 2).reshape(B * n, H * G)[here]
    return result


def run(state):
    case = state["case"]
    if case["op"] == "assign":
        if own:
            from mlops_b200.attention import paged
            step = paged.assign(state["table"], state["held"], state["new"], state["ring"], state["cursor"], case["page_size"], state["tokens"])
            return {"table": state["table"], "slots": step.slots, "positions": step.positions, "starts": step.starts, "lengths": step.lengths, "cursor": step.cursor}
        return _assign(state["table"], state["held"], state["new"], state["ring"], state["cursor"], case["page_size"], state["tokens"])
    if own:
        from mlops_b200.attention import paged
        cache = paged.PagedCache(state["units"], state["k_scale"], state["v_scale"])
        if case["op"] == "attend":
            if case["lse"]:
                out, lse = paged.attend(state["q"], cache, state["table"], state["lengths"], state["starts"], return_lse=True)
                return {"out": out, "lse": lse}
            return {"out": paged.attend(state["q"], cache, state["table"], state["lengths"], state["starts"])}
        if case["op"] == "append":
            paged.append(cache, state["k"], state["v"], state["slots"])
        k, v = paged.read(cache, state["slots"], state["dtype"])  # (after an append: what the cache now holds for the tokens)
        return {"k": k, "v": v}
    if case["op"] == "attend":
        return _attend(state)
    slots = state["slots"].long()
    if case["op"] == "append":
        kc, ks = _quantise(state["k"], state["k_scale"])
        vc, vs = _quantise(state["v"], state["v_scale"])
        _write(state["units"], slots, kc, vc, ks, vs)
    kc, vc, ks, vs = _token_fields(state["units"], slots)
    return {"k": _values(kc, ks, state["k_scale"][:, None]).to(state["dtype"]), "v": _values(vc, vs, state["v_scale"][:, None]).to(state["dtype"])}


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


def _through_cache(x, factor):
    """what the cache holds of x [tokens, heads, 128], in 64 bits"""
    e2m1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=x.device)
    e4m3 = torch.tensor([math.ldexp(8 + (b & 7), (b >> 3) - 10) if b >> 3 else math.ldexp(b, -9) for b in range(127)], dtype=torch.float64, device=x.device)
    g = factor.double()[:, None, None]
    y = x.double().unflatten(-1, (8, 16)) / g
    s = _nearest((y.abs().amax(-1, keepdim=True) / 6).clamp_(max=448.0), e4m3)
    c = _nearest((y.abs() / torch.where(s > 0, s, 1.0)).clamp_(max=6.0), e2m1)
    return (torch.where(s > 0, c * torch.sign(y) * s, 0.0) * g).flatten(-2)


def exact(case, seed):
    if case["op"] == "assign":
        return None
    s = prepare(case, seed)
    H, P = case["kv_heads"], case["page_size"]
    if case["op"] == "append":
        return {"k": _through_cache(s["k"], s["k_scale"]), "v": _through_cache(s["v"], s["v_scale"])}
    kc, vc, ks, vs = _fields(s["units"])
    gk, gv = s["k_scale"].double(), s["v_scale"].double()
    if case["op"] == "read":
        slot = s["slots"].long()
        at = (slot // P, slice(None), slot % P // 16, slot % 16)
        return {"k": _stored(kc[at], ks[at], gk[:, None]), "v": _stored(vc[at], vs[at], gv[:, None])}
    held, new = _requests(case)
    heads = H * case["group"]
    out = torch.zeros((sum(new), heads, D), dtype=torch.float64, device="cuda")
    lse = torch.full((sum(new), heads), -math.inf, dtype=torch.float64, device="cuda")
    first = 0
    for b, (h, n) in enumerate(zip(held, new)):
        length = h + n
        if length > 0 and n > 0:
            pages = s["table"][b, : -(-length // P)].long()
            limit = torch.arange(h, length, device="cuda")[:, None]
            for x in range(H):
                k, v = (_stored(c[pages, x].reshape(-1, 64)[:length], t[pages, x].reshape(-1, 8)[:length], g[x]) for c, t, g in ((kc, ks, gk), (vc, vs, gv)))
                for y in range(x * case["group"], (x + 1) * case["group"]):
                    score = s["q"][first : first + n, y].double() @ k.T / math.sqrt(D)
                    score = score.masked_fill_(torch.arange(length, device="cuda") > limit, -math.inf)
                    lse[first : first + n, y] = torch.logsumexp(score, -1)
                    out[first : first + n, y] = (score - lse[first : first + n, y, None]).exp_() @ v
        first += n
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}
