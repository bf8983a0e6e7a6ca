"""Sizes that the 4-bit cache's kernels cannot address are refused before any device work (fake addresses)."""
import pytest

from tests.test_kv_q4_cpu import INVALID, UNSUPPORTED, _append, _decode, _prefill


@pytest.mark.parametrize("call", [_append, _decode, _prefill])
@pytest.mark.parametrize("page,status", [((1 << 24) + 16, UNSUPPORTED), (1 << 25, UNSUPPORTED), (1 << 26, UNSUPPORTED),
                                         (1 << 29, UNSUPPORTED), (1 << 30, INVALID)])
def test_pages_past_32_bits_of_bytes(call, page, status):
    """A (page, head) block has 72 bytes a position, and offsets inside it are 32 bits."""
    assert call(page=page, max_pages=1) == status
