"""The workspace size of the 4-bit cache's attention refuses what the call refuses (no GPU needed)."""
import ctypes as C

import pytest

from optimized_rocwmma_samples_b200 import _lib
from test_decode_refusals import INVALID, UNSUPPORTED, attention, cache


def size(**kw):
    a = dict(batch=2, heads=4, kv_heads=2, head_dim=64, page_size=16, pages=2, most=1, acc=0)
    a.update(kw)
    n = C.c_size_t(7)
    return _lib.load().b2sq_kv4_attention_workspace_size(*a.values(), C.byref(n)), n.value


@pytest.mark.parametrize("want,kw", [
    (INVALID, dict(batch=4097)), (INVALID, dict(batch=2 ** 32 - 1)), (UNSUPPORTED, dict(head_dim=96)),
    (UNSUPPORTED, dict(head_dim=0)), (UNSUPPORTED, dict(page_size=24)), (UNSUPPORTED, dict(page_size=0)),
    (INVALID, dict(kv_heads=0)), (INVALID, dict(kv_heads=70000, heads=70000)), (INVALID, dict(heads=0)), (INVALID, dict(heads=3)),
    (INVALID, dict(pages=0x10000000)), (INVALID, dict(most=0x40000000)),
    (INVALID, dict(batch=4096, kv_heads=2048, heads=2048, pages=1 << 20)),
])
def test_sizes(want, kw):
    assert size(**kw) == (want, 0)
    c = {k: kw[k] for k in ("head_dim", "page_size", "kv_heads") if k in kw}
    call = {k: kw[k] for k in ("batch", "heads", "pages", "most") if k in kw}
    assert attention(cache(**c), **call, **(dict(qs=8 << 20) if "heads" in kw else {})) == want
    assert b"kv4_attention" in _lib.load().b2sq_last_error_message()


def test_no_place_for_the_size():
    assert _lib.load().b2sq_kv4_attention_workspace_size(2, 4, 2, 64, 16, 2, 1, 0, None) == INVALID
