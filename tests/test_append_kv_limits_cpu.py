"""Sizes of append_kv at which its byte counts would pass 64 bits (no GPU)."""
import pytest

from test_paged_attention_cpu import INVALID, append, at


@pytest.mark.parametrize("pos", [(1 << 48) + 1, 1 << 54, 1 << 62, (1 << 63) - 1])
def test_append_refuses_rotary_tables_beyond_counting(pos):
    assert append(pos=pos) == INVALID


def test_append_rotary_table_over_the_cache_at_every_size():
    """It begins 2^40 bytes before q_out and reaches over it."""
    for bits in (32, 40, 48):
        assert append(ptrs={5: at(7)}, pos=1 << bits) == INVALID
