"""Prompts through the 4-bit cache's attention: more queries than one launch takes."""
import ctypes as C

import pytest
import torch

import kv4_ref as R
from optimized_rocwmma_samples_b200 import _lib, api
from test_gpu_kv4 import DEV, run_attention

pytestmark = pytest.mark.gpu


def size(*args):
    n = C.c_size_t(0)
    assert _lib.load().b2sq_kv4_attention_workspace_size(*args, C.byref(n)) == 0
    return n.value


def test_workspace_is_bounded(cuda_device):
    """Scores take 256 MiB, or one query's; the rest does not grow with the queries."""
    rest = size(1, 32, 8, 128, 64, 64, 4, 0)
    for batch, pages, queries in ((1, 2048, 8192), (7, 64, 4001), (1, 2048, 131072), (4, 1, 1 << 20)):
        assert size(batch, 32, 8, 128, 64, pages, queries, 1) <= (256 << 20) + 4 * rest
    one = size(48, 32, 8, 128, 64, 2048, 1, 1)
    assert one >= 48 * 8 * 131072 * 4 * 4 and size(48, 32, 8, 128, 64, 2048, 100, 1) <= one + 4 * rest


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,heads,kv,page,lens,counts", [
    (64, 4, 2, 16, [75, 40], [40, 13]),        # 8 queries a time
    (128, 6, 2, 32, [90, 30, 64], [33, 30, 1]),  # 3 query heads a key head
    (64, 16, 1, 16, [50, 9], [21, 9]),
    (256, 2, 2, 16, [60, 60], [60, 20]),
])
def test_weights_in_slices(cuda_device, D, heads, kv, page, lens, counts, dtype):
    """A table of 2^20 positions leaves room for a few queries' scores at a time."""
    table, pages = R.tables(lens, page, 5, DEV)
    table = torch.nn.functional.pad(table, (0, (1 << 20) // page - table.shape[1]), value=-1).contiguous()
    cache = R.random_cache(api, pages, kv, page, D, True, 11, DEV)
    assert size(len(lens), heads, kv, D, page, table.shape[1], max(counts), 1) < 300 << 20
    run_attention(cache, table, lens, counts, heads, D, dtype, True)


def test_more_chunks_than_32_bits(cuda_device):
    """A table of 2^30 positions, 640 rows: counted for the whole table, the chunks pass 32 bits."""
    lens, counts, page = [100, 30], [40, 7], 1 << 20
    cache = R.random_cache(api, 2, 1, page, 64, False, 11, DEV)
    table = torch.full((2, 1024), -1, dtype=torch.int32, device=DEV)
    table[0, 0], table[1, 0] = 1, 0
    run_attention(cache, table, lens, counts, 16, 64, torch.float16, False)


def test_prompt_then_decode(cuda_device):
    """A prompt of 700 tokens with its weights, as evictions go by, and the tokens after it."""
    kv, heads, D, page, n = 2, 8, 128, 64, 700
    table, pages = R.tables([n + 2], page, 5, DEV)
    table = torch.nn.functional.pad(table, (0, 3000), value=-1).contiguous()
    cache = api.KV4Cache.empty(pages, kv, page, D, weights=True, device=DEV)
    g = torch.Generator(device=DEV)
    g.manual_seed(2)
    for count, length in ((n, n), (1, n + 1), (1, n + 2)):
        k, v, q = (torch.randn((count, h, D), generator=g, device=DEV).half() for h in (kv, kv, heads))
        ln, st = torch.tensor([length], dtype=torch.int32, device=DEV), R.starts([count], DEV)
        api.kv4_append(k, v, cache, table, ln, st)
        run_attention(cache, table, [length], [count], heads, D, torch.float16, True, extra=0, q=q)


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("lens,counts", [([40], [33]), ([9, 50, 20], [1, 30, 7]), ([20, 30], [1, 1])])
def test_all_rows_by_default(cuda_device, lens, counts, accumulate):
    """Without max_queries no row of a prompt is left out."""
    heads, kv, D, page = 8, 2, 64, 16
    table, pages = R.tables(lens, page, 5, DEV)
    q = torch.randn((sum(counts), heads, D), device=DEV).half()
    ln, st = torch.tensor(lens, dtype=torch.int32, device=DEV), R.starts(counts, DEV)
    got, weights = [], []
    for kw in ({}, dict(max_queries=max(counts))):
        cache = R.random_cache(api, pages, kv, page, D, accumulate, 7, DEV)
        got.append(api.kv4_attention(q, cache, table, ln, st, accumulate_weight=accumulate, **kw))
        weights.append(cache.weight)
    torch.cuda.synchronize()
    want, _, tol, _ = R.attention(q, cache, table, ln, st, D ** -0.5)
    for out in got:
        assert torch.all((out.double() - want).abs() <= tol)
    if accumulate:  # sums of at most 50 scores' exponentials in another order: 50 * 2^-24 of them
        assert torch.all((weights[0] - weights[1]).abs() <= 2.0 ** -18 * weights[1])
