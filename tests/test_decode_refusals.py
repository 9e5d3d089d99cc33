"""What the decode-step entry points refuse, before any CUDA call (no GPU needed)."""
import ctypes as C

import pytest
import torch

from optimized_rocwmma_samples_b200 import _lib, api

OK, INVALID, UNSUPPORTED = _lib.B2SQ_OK, _lib.B2SQ_ERR_INVALID_ARG, _lib.B2SQ_ERR_UNSUPPORTED
BUF = (C.c_uint8 * 4096)()
P = (C.addressof(BUF) + 255) // 256 * 256


def moe(**kw):
    a = dict(x=P, t=_lib.F16, ldx=64, w=P, ids=P, sm1=P, w13=P, s13=P, sm2=P, w2=P, s2=P, out=P, tokens=2, hidden=64,
             inter=32, experts=4, topk=2, qmax=127.0, ws=P, n=1 << 20)
    a.update(kw)
    return _lib.load().b2sq_moe_layer(*a.values(), None)


@pytest.mark.parametrize("want,kw", [
    (INVALID, dict(t=_lib.I32)), (INVALID, dict(t=9)), (INVALID, dict(qmax=0.0)), (INVALID, dict(qmax=128.0)),
    (INVALID, dict(qmax=float("nan"))), (INVALID, dict(experts=0)), (INVALID, dict(experts=1025)), (INVALID, dict(topk=0)),
    (INVALID, dict(hidden=0)), (INVALID, dict(inter=0)), (UNSUPPORTED, dict(hidden=72)), (UNSUPPORTED, dict(inter=40)),
    (UNSUPPORTED, dict(hidden=131088, ldx=131088)), (UNSUPPORTED, dict(hidden=16400, ldx=16400)),
    (UNSUPPORTED, dict(inter=131088)), (UNSUPPORTED, dict(tokens=4096)), (OK, dict(tokens=0)),
    (INVALID, dict(x=None)), (INVALID, dict(w13=None)), (INVALID, dict(out=None)), (INVALID, dict(s2=None)),
    (INVALID, dict(ldx=48)), (UNSUPPORTED, dict(ldx=68)), (UNSUPPORTED, dict(x=P + 2)), (UNSUPPORTED, dict(w2=P + 8)),
    (INVALID, dict(sm1=P + 2)),
])
def test_moe_layer(want, kw):
    assert moe(**kw) == want
    if want != OK:
        assert b"moe_layer" in _lib.load().b2sq_last_error_message()


def test_moe_layer_workspace():
    lib, n = _lib.load(), C.c_size_t(7)
    assert lib.b2sq_moe_layer_workspace_size(0, 64, 32, 4, 2, C.byref(n)) == OK and n.value == 0
    assert lib.b2sq_moe_layer_workspace_size(1, 64, 32, 4, 2, None) == INVALID
    assert lib.b2sq_moe_layer_workspace_size(1, 60, 32, 4, 2, C.byref(n)) == UNSUPPORTED


def cache(**kw):
    a = dict(k=P, v=P, k_scale=P, v_scale=P, weight=P, pages=4, kv_heads=2, page_size=16, head_dim=64)
    a.update(kw)
    return _lib.Kv4CacheStruct(*a.values())


BAD_CACHE = [
    (INVALID, dict(k=None)), (INVALID, dict(v_scale=None)), (UNSUPPORTED, dict(head_dim=96)), (UNSUPPORTED, dict(head_dim=0)),
    (UNSUPPORTED, dict(page_size=24)), (UNSUPPORTED, dict(page_size=0)), (INVALID, dict(kv_heads=0)),
    (INVALID, dict(kv_heads=70000)), (UNSUPPORTED, dict(k=P + 4)), (UNSUPPORTED, dict(weight=P + 4)),
]


def append(c=None, **kw):
    c = cache() if c is None else c
    a = dict(k=P, v=P, t=_lib.BF16, tokens=3, ks=128, vs=128, c=C.addressof(c), table=P, batch=2, pages=2, lens=P, start=P,
             ko=None, vo=None)
    a.update(kw)
    return _lib.load().b2sq_kv4_append(*a.values(), None)


def attention(c=None, **kw):
    c = cache() if c is None else c
    a = dict(q=P, t=_lib.BF16, tokens=3, heads=4, qs=256, c=C.addressof(c), table=P, batch=2, pages=2, lens=P, start=P, most=1,
             scale=0.1, out=P, acc=0, ws=P, n=1 << 30)
    a.update(kw)
    return _lib.load().b2sq_kv4_attention(*a.values(), None)


def evict(c=None, **kw):
    c = cache() if c is None else c
    a = dict(c=C.addressof(c), table=P, batch=2, pages=2, lens=P, new=P + 64, new_pages=2, budget=8, recent=2, out=P)
    a.update(kw)
    return _lib.load().b2sq_kv4_evict(*a.values(), None)


@pytest.mark.parametrize("want,kw", BAD_CACHE)
def test_bad_caches(want, kw):
    for call in (append, attention, evict):
        assert call(cache(**kw)) == want


def test_no_cache():
    lib = _lib.load()
    assert lib.b2sq_kv4_append(P, P, 1, 3, 128, 128, None, P, 2, 2, P, P, None, None, None) == INVALID
    assert lib.b2sq_kv4_attention(P, 1, 3, 4, 256, None, P, 2, 2, P, P, 1, 0.1, P, 0, P, 64, None) == INVALID
    assert lib.b2sq_kv4_evict(None, P, 2, 2, P, P, 2, 8, 2, P, None) == INVALID


@pytest.mark.parametrize("want,kw", [
    (INVALID, dict(t=_lib.I32)), (OK, dict(tokens=0)), (OK, dict(batch=0)), (INVALID, dict(batch=70000)),
    (INVALID, dict(table=None)), (INVALID, dict(lens=None)), (INVALID, dict(start=P + 2)), (INVALID, dict(k=None)),
    (INVALID, dict(ks=127)), (UNSUPPORTED, dict(ks=132)), (UNSUPPORTED, dict(vs=129)), (UNSUPPORTED, dict(k=P + 8)),
    (UNSUPPORTED, dict(vo=P + 2)), (INVALID, dict(pages=0x10000000)), (INVALID, dict(tokens=0x80000000)),
])
def test_append(want, kw):
    assert append(**kw) == want


@pytest.mark.parametrize("want,kw", [
    (INVALID, dict(t=7)), (OK, dict(tokens=0)), (OK, dict(batch=0)), (OK, dict(most=0)), (INVALID, dict(heads=0)),
    (INVALID, dict(heads=3)), (INVALID, dict(scale=float("inf"))), (INVALID, dict(scale=float("nan"))),
    (INVALID, dict(q=None)), (INVALID, dict(out=None)), (INVALID, dict(qs=255)), (UNSUPPORTED, dict(qs=260)),
    (UNSUPPORTED, dict(q=P + 2)), (UNSUPPORTED, dict(out=P + 8)), (INVALID, dict(batch=70000)),
    (INVALID, dict(most=0x40000000)), (INVALID, dict(tokens=0x80000000)),
])
def test_attention(want, kw):
    assert attention(**kw) == want


def test_weights_are_needed():
    assert attention(cache(weight=None), acc=1) == INVALID
    assert evict(cache(weight=None)) == INVALID


@pytest.mark.parametrize("want,kw", [
    (INVALID, dict(recent=9)), (OK, dict(batch=0)), (INVALID, dict(table=None)), (INVALID, dict(new=None)),
    (INVALID, dict(out=None)), (INVALID, dict(new=P)), (INVALID, dict(new_pages=0x10000000)), (INVALID, dict(batch=70000)),
])
def test_evict(want, kw):
    assert evict(**kw) == want


def test_python_refuses_host_tensors():
    t = torch.zeros((2, 2, 16, 32), dtype=torch.uint8)
    s = torch.zeros((2, 2, 16, 1, 2), dtype=torch.float16)
    with pytest.raises(ValueError):
        api.KV4Cache(t, t, s, s)
    x = torch.zeros((2, 64), dtype=torch.float16)
    with pytest.raises(ValueError):
        api.moe_layer(x, *([x] * 8))
    with pytest.raises(ValueError):
        api.moe_layer(x.float(), *([x] * 8))


def test_pitches_past_32_bits():
    """The library takes pitches in 32 bits; longer ones are refused, not cut off."""
    class Rows:  # a view that no test could hold in memory
        shape = (2, 8, 64)

        def __init__(self, pitch):
            self.pitch = pitch

        def stride(self):
            return (self.pitch, 64, 1)

        def get_device(self):
            return 0

    dev = torch.device("cuda", 0)
    assert api._kv4_rows(Rows(2 ** 32 - 8), "q", dev) == (2, 8, 2 ** 32 - 8)
    with pytest.raises(ValueError, match="2\\^32"):
        api._kv4_rows(Rows(2 ** 32 + 512), "q", dev)
