"""Buffers of the decode-step entry points that overlap: refused before any CUDA call (no GPU needed)."""
import pytest

from test_decode_refusals import INVALID, P, append, attention, evict


@pytest.mark.parametrize("shift", [-4, 4])
def test_lengths_that_overlap(shift):
    assert evict(lens=P + 64, out=P + 64 + shift) == INVALID


@pytest.mark.parametrize("kw", [
    dict(ko=P + 16), dict(vo=P + 16), dict(k=P + 1024, ko=P + 1024 - 16), dict(ko=P + 2048, vo=P + 2048),
    dict(ko=P + 2048, vo=P + 2048 + 256), dict(v=P + 1024, ko=P + 1024), dict(v=P + 1024, vo=P), dict(ks=256, vs=256, ko=P),
    dict(ko=P), dict(vo=P),  # k and v are both P here
])
def test_values_that_overlap(kw):
    assert append(**kw) == INVALID


@pytest.mark.parametrize("kw", [dict(out=P + 16), dict(q=P + 1024, out=P + 1008), dict(qs=512, out=P),
                                dict(q=P + 256, qs=512, out=P)])
def test_outputs_that_overlap(kw):
    assert attention(**{**dict(q=P, out=P), **kw}) == INVALID
