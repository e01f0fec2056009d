"""The scratch of the 4-bit cache's calls: one made for a size serves every smaller one."""

import pytest

from mla_kv_quant_b200 import _lib, build


@pytest.fixture(scope="module")
def size():
    if not _lib.LIB_PATH.exists():
        build.build()
    return _lib.load().rolaq_int4_workspace_bytes


@pytest.mark.parametrize("d", [256, 512])
def test_sizes_never_shrink_as_calls_grow(size, d):
    grid = [[size(8, t, h, d, 16) for h in range(1, 129)] for t in range(1, 65)]
    for t in range(64):
        for h in range(128):
            assert grid[t][h] > 0
            assert t == 0 or grid[t][h] >= grid[t - 1][h], (t + 1, h + 1)
            assert h == 0 or grid[t][h] >= grid[t][h - 1], (t + 1, h + 1)
    for t, h in ((1, 16), (1, 40), (3, 16), (64, 128)):
        by_batch = [size(b, t, h, d, 100) for b in (0, 1, 2, 7, 64, 1000, 65535)]
        by_pages = [size(8, t, h, d, p) for p in (0, 1, 3, 256, 2048, 1 << 20)]
        assert by_batch == sorted(by_batch) and by_pages == sorted(by_pages)
