"""The paged 4-bit cache in plain torch (test infrastructure): the format of include/mlops_paged.h, page assignment by loops, and attention in 64 bits."""
import math

import torch

D, BLOCK, BLOCK_BYTES = 128, 16, 2304
LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
E4M3 = [math.ldexp(8 + (b & 7), (b >> 3) - 10) if b >> 3 else math.ldexp(b, -9) for b in range(127)]  # the finite ones, ascending


def nearest_even(x, levels):
    """indexes of the members of the ascending `levels` nearest to x >= 0, halfway cases to the even index, the last one above its range"""
    levels = torch.tensor(levels, dtype=torch.float64)
    hi = torch.searchsorted(levels, x.double().clamp(max=float(levels[-1]))).clamp(1, len(levels) - 1)
    below, above = x.double().clamp(max=float(levels[-1])) - levels[hi - 1], levels[hi] - x.double().clamp(max=float(levels[-1]))
    return torch.where((above < below) | ((above == below) & (hi % 2 == 0)), hi, hi - 1)


def quantise(x, factor):
    """x [tokens, heads, 128] (16 bits), factor [heads] -> (codes uint8 [tokens, heads, 64], scales uint8 [tokens, heads, 8]), on the CPU"""
    x, factor = x.cpu().float(), factor.cpu().float()
    y = (x * (1.0 / factor)[:, None]).unflatten(-1, (8, 16))
    fine = torch.isfinite(y).all(-1, keepdim=True)
    top = torch.where(fine, y.abs(), 0.0).amax(-1, keepdim=True) * torch.tensor(0.1666666716337204)
    scale = nearest_even(top, E4M3)
    s = torch.tensor(E4M3, dtype=torch.float32)[scale]
    m = torch.where(fine & (s > 0), y.abs() / s, 0.0)  # (an FP32 quotient, rounded once)
    code = nearest_even(m, LEVELS) + 8 * torch.signbit(y)
    code = torch.where(fine & (s > 0), code, 0).flatten(-2)
    return (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8), torch.where(fine, scale, 127).squeeze(-1).to(torch.uint8)


def values(codes, scales, factor):
    """64-bit values of codes [..., 64] and scales [..., 8]; factor broadcasts to [..., 1]"""
    level = torch.tensor(LEVELS + [-x for x in LEVELS], dtype=torch.float64, device=codes.device)
    step = torch.tensor(E4M3 + [math.nan] + [-x for x in E4M3] + [math.nan], dtype=torch.float64, device=codes.device)
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).int()
    return level[c] * step[scales.int()].repeat_interleave(16, -1) * factor


def fields(units):
    """views of a pool: K codes, V codes [pages, heads, blocks, 16, 64], K scales, V scales [pages, heads, blocks, 16, 8]"""
    return (units[..., :1024].unflatten(-1, (16, 64)), units[..., 1024:2048].unflatten(-1, (16, 64)),
            units[..., 2048:2176].unflatten(-1, (16, 8)), units[..., 2176:].unflatten(-1, (16, 8)))


def at_slots(units, slots):
    """K codes, V codes, K scales, V scales of slots, [tokens, heads, 64 or 8]"""
    P, s = units.shape[2] * BLOCK, slots.long()
    return [f[s // P, :, s % P // BLOCK, s % BLOCK] for f in fields(units)]


def random_units(gen, pages, heads, page_size, device="cuda"):
    """a pool of random codes; scales between 1/16 and 2"""
    units = torch.randint(0, 256, (pages, heads, page_size // BLOCK, BLOCK_BYTES), generator=gen, dtype=torch.uint8, device=device)
    units[..., 2048:] = torch.randint(24, 65, units[..., 2048:].shape, generator=gen, dtype=torch.uint8, device=device)
    return units


def tables(gen, lengths, page_size, spare=3, width=None, device="cuda"):
    """a block table int32 [batch, width] of pages in no order, -1 behind a request's last, and the number of pages"""
    counts = [-(-max(n, 0) // page_size) for n in lengths]
    order = torch.randperm(sum(counts) + spare, generator=gen, device=device).to(torch.int32)
    table = torch.full((len(lengths), max(counts + [1]) if width is None else width), -1, dtype=torch.int32, device=device)
    first = 0
    for b, n in enumerate(counts):
        table[b, :n] = order[first : first + n]
        first += n
    return table, sum(counts) + spare


def spoil_behind(units, table, lengths):
    """0xff (NaN scales among it) in every slot that no request uses"""
    P = units.shape[2] * BLOCK
    used = torch.zeros(units.shape[0] * P, dtype=torch.bool, device=units.device)
    for b, n in enumerate(lengths):
        p = torch.arange(max(n, 0), device=units.device)
        page = table[b, p // P].long()
        used[(page * P + p % P)[page >= 0]] = True
    free = (~used).nonzero().view(-1)
    for f in fields(units):
        f[free // P, :, free % P // BLOCK, free % BLOCK] = 255


def attend(q, units, k_scale, v_scale, table, lengths, counts, scale=None):
    """(out, weight, lse) in 64 bits; weight = sum p |v| / sum p, what the roundings of p and v scale with. counts: queries per request"""
    tokens, heads, _ = q.shape
    H, P = units.shape[1], units.shape[2] * BLOCK
    group = heads // H
    out, weight = (torch.zeros((tokens, heads, D), dtype=torch.float64, device=q.device) for _ in range(2))
    lse = torch.full((tokens, heads), -math.inf, dtype=torch.float64, device=q.device)
    kc, vc, ks, vs = fields(units)
    first = 0
    for b, n in enumerate(counts):
        length = min(lengths[b], table.shape[1] * P)
        if n > 0 and length > 0:
            page = table[b, : -(-length // P)].long()
            there = (page >= 0).repeat_interleave(P)[:length]
            page = page.clamp(min=0)
            seen = (torch.arange(length, device=q.device)[None] <= torch.arange(lengths[b] - n, lengths[b], device=q.device)[:, None]) & there
            for h in range(H):
                k, v = (values(c[page, h].reshape(-1, 64)[:length], s[page, h].reshape(-1, 8)[:length], g[h].double()) for c, s, g in ((kc, ks, k_scale), (vc, vs, v_scale)))
                k, v = (torch.where(there[:, None], x, 0.0) for x in (k, v))
                for x in range(h * group, (h + 1) * group):
                    s = q[first : first + n, x].double() @ k.T * (1 / math.sqrt(D) if scale is None else scale)
                    s = s.masked_fill(~seen, -math.inf)
                    mass = torch.logsumexp(s, -1)
                    p = torch.where(seen, (s - mass[:, None]).exp(), 0.0)
                    out[first : first + n, x], weight[first : first + n, x], lse[first : first + n, x] = p @ v, p @ v.abs(), mass
        first += n
    return out, weight, lse
