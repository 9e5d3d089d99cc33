"""Buffers of the decode-step entry points that overlap: refused before any CUDA call (no GPU needed)."""
import pytest

from test_decode_refusals import INVALID, P, evict


@pytest.mark.parametrize("shift", [-4, 4])
def test_lengths_that_overlap(shift):
    assert evict(lens=P + 64, out=P + 64 + shift) == INVALID
