"""Sizes that leave 31 or 63 bits at the C entries in front of and around a paged cache: refused on the host, before a launch."""
import pytest

from test_paged_pages_cpu import descriptors
from VAR_Q import _cabi

LAST = 2 ** 31 - 1


@pytest.mark.parametrize("B,L,q_heads,k_heads", [(LAST, LAST, 2, 2), (LAST, LAST, 0, 1), (1 << 16, 1 << 16, LAST, LAST), (1 << 16, 1 << 16, 1 << 30, 1 << 30), (1, LAST, LAST, LAST),
                                                 (LAST, 1, 1, 0), (1 << 16, 1 << 15, 1, 0)])
def test_rows_of_a_rotation_are_counted_without_wrapping(B, L, q_heads, k_heads):
    """strides of zero make such sizes a call that somebody can write down: the product of them is no small number"""
    lib = _cabi.lib()
    _, rot, _ = descriptors()
    shared = _cabi.Tensor(256, _cabi.F16, 0, 0, 0, 0)
    assert lib.varq_rotate(rot, shared, shared, B, L, q_heads, k_heads, 64, shared, shared, None) == -2 and b"2^31" in lib.varq_last_error()


@pytest.mark.parametrize("q_heads,k_heads", [(LAST - 1, 0), (0, LAST - 1), (LAST - 3, 2), (LAST - 2 ** 19, 1)])
def test_rows_of_a_token_end_before_their_number_does(q_heads, k_heads):
    """the steps from row to row go behind the last one: none of them leaves an int"""
    lib = _cabi.lib()
    cache, rot, _ = descriptors()
    shared = _cabi.Tensor(256, _cabi.F16, 0, 0, 0, 0)
    assert lib.varq_rotate(rot, shared, shared, 1, 1, q_heads, k_heads, 64, shared, shared, None) == -2 and b"2^31" in lib.varq_last_error()
    if q_heads:
        assert lib.varq_paged_append_rotated(cache, rot, shared, shared, shared, 256, 1, q_heads - 4, 1e-12, shared, None) == -2 and b"2^31" in lib.varq_last_error()


@pytest.mark.parametrize("tokens", [LAST, LAST - 1, LAST - 127, 2 ** 31 - 512])
def test_drafted_tokens_end_before_their_number_does(tokens):
    """the threads of a block go through a sequence's tokens in steps of an int"""
    lib = _cabi.lib()
    assert lib.varq_paged_tree(256, 256, 256, 1, tokens, 32, 1, 256, 256, None) == -2 and b"2^31" in lib.varq_last_error()
