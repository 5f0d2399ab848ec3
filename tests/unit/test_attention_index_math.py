"""Bounds, bijectivity and bank spread of the attention tiles' LDS map (csrc/common/index_math.h)."""

import ctypes

import numpy as np
import pytest

from nanofed_amd import native_build


@pytest.fixture(scope="module")
def ix():
    native_build.build_host()
    return ctypes.CDLL(str(native_build.HOST_LIB))


@pytest.mark.parametrize("width", [64, 128])
def test_attention_tile_map(ix, width):
    pieces = width // 8
    offs = np.array([[ix.nf_ix_attn_off(width, r, p) for p in range(pieces)] for r in range(64)])
    assert offs.min() == 0 and offs.max() == 64 * width * 2 - 16 and (offs % 16 == 0).all()
    assert len(np.unique(offs)) == 64 * pieces
    assert ((offs // (width * 2)) == np.arange(64)[:, None]).all()  # a piece never leaves its row
    slot = (offs // 16) % 16
    # row reads: the 16 lanes of a read group take one piece of 16 rows
    groups = [[l for l in range(32) if ix.nf_ix_lds_b128_group(l) == g] for g in (0, 1)]
    for r0 in (0, 32):
        for g in groups:
            for p in range(pieces):
                assert len({int(slot[r0 + l, p]) for l in g}) == 16
    # transposing reads: 32 lanes take four consecutive rows at 32 consecutive columns
    for r in range(0, 64, 4):
        for p in range(0, pieces, 4):
            assert len({int(slot[r + i, p + j]) for i in range(4) for j in range(4)}) == 16
