"""CPU tests of the limits of the mixture operators: refused before anything is launched."""
import ctypes

import pytest

from tilelang_ascend_b200 import _lib

SOME = ctypes.c_void_p(4096)  # a pointer that no refused call follows
MAX_BLOCKS = (2 ** 31 - 1) // 3  # three 32-bit numbers an entry, addressed by 32-bit indexes


def _words(rc):
    assert rc != 0
    return _lib.last_error()


@pytest.mark.parametrize("entries,experts,block_M", [(MAX_BLOCKS + 1, 4, 1), (1 << 30, 1024, 1)])
def test_block_tables_beyond_32_bit_indexes_are_refused(entries, experts, block_M):
    lib = _lib.load()
    assert lib.qgemm_moe_block_count(entries, experts, block_M) > MAX_BLOCKS
    assert "no more than" in _words(lib.qgemm_moe_blocks(SOME, SOME, SOME, SOME, entries, experts, block_M, None))


@pytest.mark.parametrize("entries,experts,block_M", [(MAX_BLOCKS, 4, 1), (1 << 30, 1024, 2)])
def test_tables_up_to_the_limit_are_not(entries, experts, block_M):
    lib = _lib.load()
    assert "null" in _words(lib.qgemm_moe_blocks(None, SOME, SOME, SOME, entries, experts, block_M, None))
