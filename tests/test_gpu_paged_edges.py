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
