"""The 8-bit products' built kernels, from the code objects' metadata (no GPU): nothing is built
that no call reaches, and registers spill where the source says."""
from __future__ import annotations

import pytest

from dflash_mlx import _build
from tests.test_code_objects import _gfx950_objects, _kernels

WIDE, NARROW = "ShapeILi4ELi2ELi8E", "ShapeILi2ELi2ELi4E"


@pytest.fixture(scope="module")
def tiles():
    if not _build.LIB_PATH.exists():
        pytest.skip("library not built")
    return {k[".name"]: k for o in _gfx950_objects(_build.LIB_PATH.read_bytes()) for k in _kernels(o)
            if "prompt_i8_kernel" in k[".name"]}


def test_only_small_tiles_split_k(tiles):
    """Three output types, plain and gated, of either tile; the splits' sums of the small one."""
    assert sum(WIDE in n for n in tiles) == 6 and sum(NARROW in n for n in tiles) == 7 and len(tiles) == 13
    assert [n for n in tiles if "Lb0ELb1E" in n and NARROW in n] and not [n for n in tiles if "Lb0ELb1E" in n and WIDE in n]


def test_scratch(tiles):
    for name, k in tiles.items():
        assert k[".private_segment_fixed_size"] <= (28 if WIDE in name else 0), name
