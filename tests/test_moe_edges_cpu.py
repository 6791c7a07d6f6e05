"""CPU tests of the limits of the mixture operators: refused before anything is launched."""
import ctypes
import os
import re

import pytest

from tilelang_ascend_b200 import _lib, moe

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


def test_limits_of_the_python_layer_are_the_header_s():
    header = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "qgemm.h")).read()
    stated = {name: int(value) for name, value in re.findall(r"#define QGEMM_MOE_MAX_(\w+) (\d+)", header)}
    assert stated == dict(EXPERTS=moe._MOST["num_experts"], TOP_K=moe._MOST["top_k"], GROUPS=moe._MOST["num_groups"], BLOCK_M=moe._MOST["block_M"], BLOCKS=moe._MAX_BLOCKS)
    assert moe._MOST["top_groups"] == stated["GROUPS"] and stated["BLOCKS"] == MAX_BLOCKS


@pytest.mark.parametrize("name,most", [("top_k", 32), ("num_experts", 1024), ("block_M", 128), ("num_groups", 32), ("top_groups", 32), ("group_top", 2)])
def test_counts_above_their_limit(name, most):
    moe._check_counts(**{name: most})
    for v in (most + 1, 2 ** 63, 2 ** 64 + 1):
        with pytest.raises(_lib.QGemmError, match=name):
            moe._check_counts(**{name: v})
    for v in (0, -1, 1.0, None):
        with pytest.raises(ValueError, match=name):
            moe._check_counts(**{name: v})
