"""What append_rotated, cross_attend and attend_shared refuse, through the C interface and Python. Needs no GPU: every refusal comes before the first CUDA call."""
import ctypes
import math

import pytest
import torch

from tests.test_paged_cpu import paged, pool, refused  # noqa: F401  (paged: the fixture)
from tests.test_paged_cpu import test_a_pool_that_cannot_be_used as pools


def changed(a, changes):
    for name, value in changes.items():
        setattr(a, name, value)
    return a


def rotate_args(paged, **changes):
    return changed(paged._Rotate(2, 32, 0, 128, 0, 100, 4096, 128, 4096, 4096, 4096, 6144, 128, 6144, 128, 6144, 128, 4096, 4096, 128, 4096, 4096), changes)


def attend_args(paged, **changes):
    return changed(paged._Attend(2, 2, 32, 0, 4096, 4096, 128, 4096, 4096, 128, None, 4096, 10, 10, 4096, None, 0.0), changes)


@pytest.mark.parametrize("changes, words", [m for m in pools.pytestmark[0].args[1]])
def test_a_pool_that_cannot_be_used(paged, changes, words):  # noqa: F811
    c, common = pool(paged, **changes), paged._Common(1, None, 4096)
    refused(paged, paged._lib.mlops_paged_append_rotated(c, ctypes.byref(rotate_args(paged)), None), words)
    refused(paged, paged._lib.mlops_paged_cross_attend(ctypes.byref(attend_args(paged)), c, 4096, 1 << 30, None), words)
    refused(paged, paged._lib.mlops_paged_attend_shared(ctypes.byref(attend_args(paged)), ctypes.byref(common), c, 4096, 1 << 30, None), words)


def test_append_rotated_refusals(paged):  # noqa: F811
    lib, c = paged._lib, pool(paged)
    refused(paged, lib.mlops_paged_append_rotated(c, None, None), "needs")
    for changes, words in (({"tokens": -1}, "tokens"), ({"q_heads": -1}, "q_heads"), ({"reach": -1}, "reach"), ({"type": 2}, "type"), ({"rotated": 0}, "rotated"), ({"rotated": 16}, "rotated"),
                           ({"rotated": 48}, "rotated"), ({"rotated": 160}, "rotated"), ({"rotated": -32}, "rotated"), ({"interleaved": 2}, "neighbours"), ({"interleaved": -1}, "neighbours"),
                           ({"tokens": 1 << 26}, "split the tokens"), ({"q": None}, "null"), ({"k": None}, "null"), ({"v": None}, "null"), ({"q_out": None}, "null"), ({"slots": None}, "null"),
                           ({"positions": None}, "null"), ({"angles": None}, "null"), ({"q": 4104}, "16-byte"), ({"k": 4104}, "16-byte"), ({"v": 4098}, "16-byte"), ({"q_out": 4100}, "16-byte"),
                           ({"q_token_stride": 6148}, "multiples of 8"), ({"k_head_stride": 132}, "multiples of 8"), ({"v_token_stride": 1}, "multiples of 8"), ({"out_head_stride": 4}, "multiples of 8"),
                           ({"angles": 4104}, "angles"), ({"angle_stride": 130}, "angles"), ({"angle_stride": 64}, "angles"), ({"slots": 4098}, "4-byte"), ({"positions": 4097}, "4-byte")):
        refused(paged, lib.mlops_paged_append_rotated(c, ctypes.byref(rotate_args(paged, **changes)), None), words)
    assert lib.mlops_paged_append_rotated(c, ctypes.byref(rotate_args(paged, tokens=0, q=None, k=None, v=None, slots=None, positions=None)), None) == 0


def test_attention_refusals(paged):  # noqa: F811
    lib, c, common = paged._lib, pool(paged), paged._Common(1, None, 4096)
    calls = (lambda a, s=4096, n=1 << 40: lib.mlops_paged_cross_attend(ctypes.byref(a), c, s, n, None), lambda a, s=4096, n=1 << 40: lib.mlops_paged_attend_shared(ctypes.byref(a), ctypes.byref(common), c, s, n, None))
    for call, function in zip(calls, (b"mlops_paged_cross_attend", b"mlops_paged_attend_shared")):
        for changes, words in (({"batch": -1}, "batch"), ({"batch": 2049, "tokens": 2049}, "batch"), ({"tokens": -1}, "tokens"), ({"q_heads": 0}, "q_heads"), ({"q_heads": 33}, "divides"),
                               ({"type": 2}, "type"), ({"scale": -1.0}, "scale"), ({"scale": math.nan}, "scale"), ({"scale": math.inf}, "scale"), ({"tokens": 3}, "one query per request"),
                               ({"width": -1}, "width"), ({"table_stride": 9}, "stride"), ({"width": 1 << 27, "table_stride": 1 << 27}, "split the batch"), ({"q": None}, "null"), ({"out": None}, "null"),
                               ({"lengths": None}, "null"), ({"table": None}, "null"), ({"q": 4104}, "16-byte"), ({"out": 4100}, "16-byte"), ({"q_token_stride": 4100}, "multiples of 8"),
                               ({"out_head_stride": 130}, "multiples of 8"), ({"lengths": 4098}, "4-byte"), ({"starts": 4097}, "4-byte"), ({"lse": 4098}, "4-byte")):
            refused(paged, call(attend_args(paged, **changes)), words)
            assert lib.mlops_paged_last_error().startswith(function)
        refused(paged, call(attend_args(paged), None), "null")
        refused(paged, call(attend_args(paged), 4100), "16-byte")
        refused(paged, call(attend_args(paged), 4096, 0), "scratch")
        assert call(attend_args(paged, batch=0, tokens=0)) == 0


def test_group_refusals(paged):  # noqa: F811
    lib, c = paged._lib, pool(paged)
    refused(paged, lib.mlops_paged_attend_shared(ctypes.byref(attend_args(paged)), None, c, 4096, 1 << 40, None), "null")
    for common, words in (((0, None, 4096), "groups"), ((-1, 4096, 4096), "groups"), ((2, None, 4096), "groups"), ((2047, 4096, 4096), "2048"), ((1, None, None), "null"), ((1, 4098, 4096), "4-byte"),
                          ((2, 4096, 4097), "4-byte")):
        g = paged._Common(*common)
        refused(paged, lib.mlops_paged_attend_shared(ctypes.byref(attend_args(paged)), ctypes.byref(g), c, 4096, 1 << 40, None), words)
    for g in (None, paged._Common(0, None, 4096), paged._Common(2, None, 4096), paged._Common(2047, 4096, 4096)):
        assert lib.mlops_paged_attend_shared_scratch_bytes(ctypes.byref(attend_args(paged)), g if g is None else ctypes.byref(g), 8) == 0


def test_python_refusals(paged):  # noqa: F811
    cache = paged.empty(3, 2, 32, device="cpu")
    x, one = torch.zeros((1, 2, 128), dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32)
    for call in (lambda: paged.append_rotated(cache, x, x, x, one, one, torch.zeros((4, 128))), lambda: paged.cross_attend(x, cache, one.view(1, 1), one),
                 lambda: paged.attend_shared(x, cache, one.view(1, 1), one, None, None, one)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_groups_without_their_common_tokens(paged):  # noqa: F811
    cache = paged.empty(3, 2, 32, device="cpu")
    x, one = torch.zeros((1, 2, 128), dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32)
    for groups in (None, torch.zeros(2, dtype=torch.int32)):
        with pytest.raises(ValueError, match="shared"):
            paged.attend_shared(x, cache, one.view(1, 1), one, None, groups, None)
