"""Sizes near the ends of 64 bits choose the kernel that sizes near them choose, or are refused."""
import pytest

pytest.importorskip("torch")

from saccade_core import _lib
from test_paged_cpu import Call


@pytest.mark.parametrize("dtype", [_lib.SC_F16, _lib.SC_F32])
@pytest.mark.parametrize("heads", [(4, 2), (64, 1), (14, 2), (3, 3)])
def test_a_bound_of_any_size_on_the_new_tokens(dtype, heads):
    """The bound times the query heads of a KV head passes 64 bits: many new tokens, not few."""
    size = lambda q: _lib.LIB.sc_qwen2_paged_attention_scratch(3, *heads, 64, q, 100, dtype)  # noqa: E731
    assert size(1000) > 0
    for q in (1 << 31, 1 << 40, 1 << 58, 1 << 60, 1 << 61, 1 << 62, (1 << 63) - 1):
        assert size(q) == size(1000)


def test_more_pages_than_31_bits_of_positions():
    c = Call()
    for pages in ((1 << 31) // 16, 1 << 59, 1 << 60, 1 << 62, (1 << 63) - 1):
        for call in (c.append, c.attention):
            assert call(max_pages=pages) == _lib.SC_EINVAL and "max_pages" in _lib.last_error()
    assert c.attention(max_pages=(1 << 31) // 16 - 1, nbytes=0) == _lib.SC_ENOMEM  # that many pass
