"""The least that attention over chunks asks for: a call of long tables is cut into parts, one a block, and every part has
room for two sums of a tile (of 32 rows at least) and a note."""

import pytest

from svdmlp import _lib

CUS, LEAST = 256, 512  # blocks that a class has at least on a full card; keys that one takes at most before another is there


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("D", [8, 64, 128, 200, 256])
@pytest.mark.parametrize("Hq,Hk", [(1, 1), (32, 8), (64, 8), (7, 7), (128, 1)])
def test_workspace_holds_the_parts(dtype, D, Hq, Hk):
    lib = _lib.load()
    for T in (1, 3, 64, 700, 9000, 1 << 20):
        for B in (1, 2, 64, 65, 1000):
            for page, width in ((16, 300), (64, 4000), (5, 65536), (1, 65536), (32768, 65532)):
                n = lib.svdmlp_chunk_attention_workspace_bytes(T, B, page, width, Hq, Hk, D, dtype)
                parts = min(CUS, page * width // LEAST)
                assert n >= parts * (32 + 8 * 32 * (D + 2)), (T, B, page, width, n)
            assert lib.svdmlp_chunk_attention_workspace_bytes(T, B, 5, 65537, Hq, Hk, D, dtype) == 0  # wider than a table may be


def test_workspace_of_one_part_is_none():
    lib = _lib.load()
    assert lib.svdmlp_chunk_attention_workspace_bytes(1, 1, 1, 1, 1, 1, 64, 1) == 0
