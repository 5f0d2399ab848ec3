"""The generator of the dropout masks gives the words that its authors published for Philox4x32 with seven
rounds (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", known-answer tests)."""

import pytest
import torch

from nanofed_amd.ops.dropout import philox_words
from tests import transformer_oracles as oracle

VECTORS = [  # counter, key, words
    ((0, 0, 0, 0), (0, 0), (0x5F6FB709, 0x0D893F64, 0x4F121F81, 0x4F730A48)),
    ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x5207DDC2, 0x45165E59, 0x4D8EE751, 0x8C52F662)),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
     (0x4DFCCABA, 0x190A87F0, 0xC47362BA, 0xB6B5242A)),
]


@pytest.mark.parametrize("counter,key,words", VECTORS)
def test_published_words(counter, key, words):
    seed = key[0] | key[1] << 32
    c = [torch.tensor(x) for x in counter]
    assert tuple(philox_words(seed, counter[3], *c[:3]).tolist()) == words
    assert tuple(int(x) for x in oracle.philox(counter, seed)) == words
