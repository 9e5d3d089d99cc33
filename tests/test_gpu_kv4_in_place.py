"""Calls that write over their inputs: eviction its lengths, append its keys and values, attention its queries."""
import pytest
import torch

import kv4_ref as R
from optimized_rocwmma_samples_b200 import api
from test_gpu_kv4 import DEV, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,kv,size,lens,budget,recent", [
    (64, 16, 16, [300 - i for i in range(40)], 100, 10),  # more blocks than the GPU holds: the last ones start late
    (128, 1, 64, [5000], 3000, 100),                      # several blocks a head
    (256, 8, 32, [700, 20, 0, 1000], 256, 256),
    (64, 2, 16, [50, -3], 0, 0),
])
def test_evict_in_place(cuda_device, D, kv, size, lens, budget, recent):
    table, pages = R.tables(lens, size, 20, DEV, spare=1)
    kept = [min(max(n, 0), budget) for n in lens]
    fresh, end = R.tables(kept, size, 21, DEV, first=pages)
    cache = R.random_cache(api, end + 1, kv, size, D, True, 22, DEV)
    names = ("k", "v", "k_scale", "v_scale", "weight")
    before = {n: getattr(cache, n).clone() for n in names}
    apart = api.kv4_evict(cache, table, ints(*lens), fresh, budget, recent)
    torch.cuda.synchronize()
    want = {n: getattr(cache, n).clone() for n in names}
    for n in names:
        getattr(cache, n).copy_(before[n])
    ln = ints(*lens)
    assert api.kv4_evict(cache, table, ln, fresh, budget, recent, new_lens=ln) is ln
    torch.cuda.synchronize()
    assert ln.tolist() == kept and torch.equal(ln, apart)
    for n in names:
        assert torch.equal(getattr(cache, n), want[n]), n


def test_evict_in_place_captured(cuda_device):
    """Captured with an attention behind it that reads the lengths, and replayed with others."""
    lens, size, kv, D, budget = [400, 90], 16, 4, 64, 64
    table, pages = R.tables(lens, size, 20, DEV)
    fresh, end = R.tables([budget + 16] * 2, size, 21, DEV, first=pages)
    cache = R.random_cache(api, end, kv, size, D, True, 22, DEV)
    q = torch.randn((2, 8, D), device=DEV).half()
    ln, st = ints(*lens), ints(0, 1, 2)
    out = torch.zeros_like(q)

    def step():
        api.kv4_evict(cache, table, ln, fresh, budget, 8, new_lens=ln)
        api.kv4_attention(q, cache, fresh, ln, st, out=out)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    ln.copy_(ints(333, 50))
    graph.replay()
    torch.cuda.synchronize()
    assert ln.tolist() == [64, 50]
    want, _, tol, _ = R.attention(q, cache, fresh, ln, st, D ** -0.5)
    assert torch.all((out.double() - want).abs() <= tol)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("counts", [[1, 1, 1], [700, 30, 2900]])
def test_append_in_place(cuda_device, counts, dtype):
    kv, D, size = 4, 128, 32
    table, pages = R.tables(counts, size, 2, DEV)
    st, ln = R.starts(counts, DEV), ints(*counts)
    k, v = (torch.randn((sum(counts), kv, D), device=DEV).to(dtype) for _ in range(2))
    k[0, 0, :64] = torch.linspace(-7.5, 7.5, 64, device=DEV).to(dtype)
    k[0, 0, 3] = 2.0 ** -24
    one, two = (api.KV4Cache.empty(pages, kv, size, D, device=DEV) for _ in range(2))
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    api.kv4_append(k, v, one, table, ln, st, k_out=ko, v_out=vo)
    api.kv4_append(k, v, two, table, ln, st, k_out=k, v_out=v)
    torch.cuda.synchronize()
    assert torch.equal(k, ko) and torch.equal(v, vo)
    for n in ("k", "v", "k_scale", "v_scale"):
        assert torch.equal(getattr(one, n), getattr(two, n)), n


@pytest.mark.parametrize("D,heads,kv,lens,counts", [(64, 8, 8, [9, 700], [1, 1]), (128, 32, 8, [3000, 20, 41], [1, 1, 1]),
                                                    (128, 16, 2, [600, 90], [40, 7]), (256, 8, 2, [500], [30])])
def test_attention_in_place(cuda_device, D, heads, kv, lens, counts):
    table, pages = R.tables(lens, 32, 2, DEV)
    cache = R.random_cache(api, pages, kv, 32, D, False, 3, DEV)
    q = torch.randn((sum(counts), heads, D), device=DEV).half()
    st, ln = R.starts(counts, DEV), ints(*lens)
    apart = api.kv4_attention(q, cache, table, ln, st, max_queries=max(counts))
    assert api.kv4_attention(q, cache, table, ln, st, max_queries=max(counts), out=q) is q
    torch.cuda.synchronize()
    assert torch.equal(q, apart)
