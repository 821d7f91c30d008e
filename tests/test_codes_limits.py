"""Operands held in few bits, without a GPU: sizes that the library's 32-bit extents cannot hold."""
import pytest

from wmma_extension_b200 import tcec


@pytest.mark.parametrize("size", [-1, 2**31, 2**32 + 128])
def test_sizes_that_are_no_extents_are_refused(size):
    """2^32 + 128 would arrive as 128."""
    for call in (lambda: tcec.q4_bytes(size, 128), lambda: tcec.q4_bytes(128, size), lambda: tcec.q8_bytes(size, 128), lambda: tcec.q8_bytes(128, size)):
        with pytest.raises(ValueError, match="2147483647"):
            call()
    assert tcec.q4_bytes(2**31 - 1, 1) == 2**24 * 8704 and tcec.q8_bytes(1, 2**31 - 1) == 2**24 * 16896
