"""What the paged cache's documents say where its kernels decide nothing. Needs no GPU."""
import inspect
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def paged():
    if not os.path.exists(os.path.join(ROOT, "mlops_b200", "lib", "libmlops_attention.so")):
        import __graft_entry__
        __graft_entry__.build()
    from mlops_b200.attention import paged
    return paged


def test_append_promises_nothing_for_a_repeated_slot(paged):
    """eight threads store a (token, head) with nothing that orders them against another token's: no document names a winner, all ask for distinct slots"""
    with open(os.path.join(ROOT, "include", "mlops_paged.h")) as f:
        header = f.read()
    with open(os.path.join(ROOT, "INTEGRATION.md")) as f:
        notes = f.read()
    assert "one of them stays" not in header
    assert all("distinct" in text for text in (header, notes, inspect.getdoc(paged.append)))
