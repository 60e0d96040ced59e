"""What the paged cache refuses, through the C interface, and its plain model's facts. Needs no GPU: every refusal comes before the first CUDA call."""
import ctypes
import math
import os

import pytest
import torch

from tests import paged_util as pu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def paged():
    if not os.path.exists(os.path.join(ROOT, "mlops_b200", "lib", "libmlops_attention.so")):
        import __graft_entry__
        __graft_entry__.build()
    from mlops_b200.attention import paged
    return paged


def refused(paged, status, words):
    assert status == 1 and words in paged._lib.mlops_paged_last_error().decode()


UNIT = 4 * 2304


def pool(paged, **changes):
    c = paged._Cache(4096, 4096, 4096, 8 * UNIT, UNIT, 10, 64, 8)
    for name, value in changes.items():
        setattr(c, name, value)
    return ctypes.byref(c)


@pytest.mark.parametrize("changes, words", [
    ({"units": None}, "null"), ({"k_scale": None}, "null"), ({"v_scale": None}, "null"), ({"pages": 0}, "pages"), ({"kv_heads": 0}, "kv_heads"), ({"page_size": 0}, "multiple of 16"),
    ({"page_size": 24}, "multiple of 16"), ({"pages": 1 << 26}, "2^31"), ({"page_stride": 8 * UNIT + 8}, "16 bytes"), ({"head_stride": UNIT - 16}, "unit"), ({"page_stride": 16}, "unit"),
    ({"units": 4104}, "16-byte")])
def test_a_pool_that_cannot_be_used(paged, changes, words):
    c = pool(paged, **changes)
    refused(paged, paged._lib.mlops_paged_append(c, 1, 0, 4096, 1024, 128, 4096, 1024, 128, 4096, None), words)
    refused(paged, paged._lib.mlops_paged_read(c, 1, 0, 4096, 4096, 4096, None), words)
    refused(paged, paged._lib.mlops_paged_attend(ctypes.byref(paged._Attend()), c, 4096, 1 << 30, None), words)


def test_append_and_read_refusals(paged):
    lib, c = paged._lib, pool(paged)
    good = [1, 0, 4096, 1024, 128, 4096, 1024, 128, 4096]
    for at, value, words in ((0, -1, "tokens"), (0, 1 << 28, "split the tokens"), (1, 2, "type"), (1, -1, "type"), (2, None, "null"), (5, None, "null"), (8, None, "null"), (2, 4104, "16-byte"), (3, 1028, "multiples of 8"),
                             (4, 129, "multiples of 8"), (5, 4098, "16-byte"), (6, 4, "multiples of 8"), (7, 4, "multiples of 8")):
        call = list(good)
        call[at] = value
        refused(paged, lib.mlops_paged_append(c, *call, None), words)
    for at, value, words in ((0, -1, "tokens"), (0, 1 << 28, "split the tokens"), (1, 7, "type"), (2, None, "null"), (3, None, "null"), (4, None, "null"), (3, 4104, "16-byte"), (4, 4100, "16-byte")):
        call = [1, 0, 4096, 4096, 4096]
        call[at] = value
        refused(paged, lib.mlops_paged_read(c, *call, None), words)
    assert lib.mlops_paged_append(c, 0, 0, None, 0, 0, None, 0, 0, None, None) == 0 and lib.mlops_paged_last_error() == b""
    assert lib.mlops_paged_read(c, 0, 1, None, None, None, None) == 0


def test_assign_refusals(paged):
    def call(**changes):
        a = paged._Assign(4, 4, 64, 10, 10, 4096, 4096, 4096, 4096, 50, 4096, 4096, 4096, 4096, 4096, 4096)
        for name, value in changes.items():
            setattr(a, name, value)
        return paged._lib.mlops_paged_assign(ctypes.byref(a), None)
    refused(paged, paged._lib.mlops_paged_assign(None, None), "null")
    for changes, words in (({"starts": None}, "null"), ({"moved": None}, "null"), ({"cursor": None}, "null"), ({"batch": -1}, "batch"), ({"batch": 16385}, "batch"), ({"tokens": -1}, "tokens"),
                           ({"width": -1}, "width"), ({"ring_size": -1}, "ring_size"), ({"page_size": 40}, "multiple of 16"), ({"page_size": 0}, "multiple of 16"), ({"held": None}, "held"),
                           ({"added": None}, "added"), ({"lengths": None}, "lengths"), ({"table": None}, "table"), ({"table_stride": 9}, "stride"), ({"slots": None}, "slots"),
                           ({"positions": None}, "positions"), ({"ring": None}, "ring"), ({"held": 4098}, "4-byte"), ({"cursor": 4100}, "8-byte"), ({"moved": 4100}, "8-byte")):
        refused(paged, call(**changes), words)


def test_attend_refusals(paged):
    lib, c = paged._lib, pool(paged)

    def args(**changes):
        a = paged._Attend(2, 2, 32, 0, 4096, 4096, 128, 4096, 4096, 128, None, 4096, 10, 10, 4096, None, 0.0)
        for name, value in changes.items():
            setattr(a, name, value)
        return a
    for changes, words in (({"batch": -1}, "batch"), ({"batch": 16385, "tokens": 16385}, "batch"), ({"tokens": -1}, "tokens"), ({"q_heads": 0}, "q_heads"), ({"q_heads": 33}, "divides"),
                           ({"type": 2}, "type"), ({"scale": -1.0}, "scale"), ({"scale": math.nan}, "scale"), ({"scale": math.inf}, "scale"), ({"tokens": 3}, "one query per request"),
                           ({"width": -1}, "width"), ({"table_stride": 9}, "stride"), ({"width": 1 << 27, "table_stride": 1 << 27}, "split the batch"), ({"q": None}, "null"), ({"out": None}, "null"), ({"lengths": None}, "null"), ({"table": None}, "null"),
                           ({"q": 4104}, "16-byte"), ({"out": 4100}, "16-byte"), ({"q_token_stride": 4100}, "multiples of 8"), ({"q_head_stride": 4}, "multiples of 8"),
                           ({"out_head_stride": 130}, "multiples of 8"), ({"lengths": 4098}, "4-byte"), ({"starts": 4097}, "4-byte"), ({"lse": 4098}, "4-byte")):
        refused(paged, lib.mlops_paged_attend(ctypes.byref(args(**changes)), c, 4096, 1 << 40, None), words)
    refused(paged, lib.mlops_paged_attend(ctypes.byref(args()), c, None, 1 << 40, None), "null")
    refused(paged, lib.mlops_paged_attend(ctypes.byref(args()), c, 4100, 1 << 40, None), "16-byte")
    refused(paged, lib.mlops_paged_attend(ctypes.byref(args()), c, 4096, 0, None), "scratch")
    assert lib.mlops_paged_attend(ctypes.byref(args(batch=0, tokens=0)), c, 4096, 1 << 40, None) == 0
    for bad in (args(q_heads=33), args(batch=-1), args(tokens=-1), args(q_heads=0)):
        assert lib.mlops_paged_attend_scratch_bytes(ctypes.byref(bad), 8) == 0
    assert lib.mlops_paged_attend_scratch_bytes(ctypes.byref(args()), 0) == 0 and lib.mlops_paged_attend_scratch_bytes(None, 8) == 0


def test_python_refusals(paged):
    with pytest.raises(ValueError, match="multiple of 16"):
        paged.empty(3, 2, 40, device="cpu")
    with pytest.raises(ValueError, match="2\\^31"):
        paged.empty(1 << 25, 2, 64, device="cpu")
    cache = paged.empty(3, 2, 32, device="cpu", k_scale=torch.tensor([1.0, 2.0]))
    assert cache.pages == 3 and cache.page_size == 32 and cache.units.shape == (3, 2, 2, 2304) and cache.k_scale.tolist() == [1.0, 2.0] and cache.v_scale.tolist() == [1.0, 1.0]
    x, one = torch.zeros((1, 2, 128), dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32)
    for call in (lambda: paged.append(cache, x, x, one), lambda: paged.read(cache, one), lambda: paged.attend(x, cache, one.view(1, 1), one),
                 lambda: paged.assign(one.view(1, 1), one, one, one, torch.zeros(2, dtype=torch.int64), 16, 1)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_the_plain_quantiser_is_the_nearest_stored_value(paged):
    """no code of the block's scale is nearer to the element than the one that is stored (64 bits, every element up to the largest code)"""
    gen = torch.Generator().manual_seed(1)
    x = (torch.randn((50, 3, 128), generator=gen) * torch.exp2(torch.randint(-6, 8, (50, 3, 1), generator=gen).float())).to(torch.bfloat16)
    factor = torch.tensor([1.0, 0.5, 4.0])
    codes, scales = pu.quantise(x, factor)
    held = pu.values(codes, scales, factor.double()[:, None])
    step = pu.values(torch.full_like(codes, 0x22), scales, factor.double()[:, None])  # the value of code 2, which is 1: the scale times the factor
    level = torch.tensor(pu.LEVELS + [-y for y in pu.LEVELS], dtype=torch.float64)
    best = (x.double()[..., None] - step[..., None] * level).abs().amin(-1)
    assert torch.equal((x.double() - held).abs(), best)
    assert float((held - x.double()).norm() / x.double().norm()) < 0.12
