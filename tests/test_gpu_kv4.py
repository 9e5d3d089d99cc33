"""The 4-bit key/value cache on the GPU: append, attention and eviction against
plain 64-bit restatements (kv4_ref.py), at the lengths, masks and contents
where they can go wrong, and a run of them together."""
import pytest
import torch

import kv4_ref as R
from optimized_rocwmma_samples_b200 import _lib, api

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------ append
def check_append(x, data, scale, out, page, slot, ok, rows):
    """x [rows, heads, D] against the slots it went to."""
    q, step, base = R.quantise(x[rows])
    got = torch.stack([data & 15, data >> 4], -1).flatten(-2)[page, :, slot].double()
    gs, gz = scale[page, :, slot, :, 0], scale[page, :, slot, :, 1]
    assert torch.equal(torch.nan_to_num(gs, 7.0), torch.nan_to_num(step, 7.0))
    assert torch.equal(torch.nan_to_num(gz, 7.0), torch.nan_to_num(base, 7.0))
    # v - z is rounded to fp32 (2^-24 of it, in steps of s: 2^-20 at most), so a nibble may differ on a border only
    y = x[rows].double().clamp(-65504, 65504).unflatten(-1, (-1, 64))
    s, z = step.double()[..., None], base.double()[..., None]
    exact = torch.where(s > 0, (y - z) / s, torch.zeros_like(y)).flatten(-2)
    border = ((exact - exact.floor() - 0.5).abs() < 2.0 ** -20).nan_to_num(0)
    finite = torch.isfinite(step).repeat_interleave(64, -1)
    assert torch.equal(torch.where(finite & ~border, got, 0.0), torch.where(finite & ~border, q, 0.0))
    assert torch.all((got - q).abs()[finite & border] <= 1)
    if out is not None:
        want = (got.unflatten(-1, (-1, 64)) * s + z).flatten(-2)
        half = torch.finfo(x.dtype).eps / 2
        o = out[rows].double()
        assert torch.equal(o.isnan(), ~finite)
        tol = half * want.abs() * (1 + 2.0 ** -11) + 2.0 ** -25
        assert torch.all(((o - want).abs() <= tol) | ~finite)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,heads,size", [(64, 3, 16), (128, 8, 64), (256, 1, 48)])
def test_append(cuda_device, dtype, D, heads, size):
    counts = [1, 0, 17, 64, 5]
    lens = [1, 9, 17, 130, 100]
    T = sum(counts)
    g = torch.Generator(device=DEV)
    g.manual_seed(D + heads)
    qkv = torch.randn((T + 3, 3 * heads * D), generator=g, device=DEV).to(dtype)  # keys and values as slices
    k = qkv[:, heads * D:2 * heads * D].unflatten(-1, (heads, D))
    v = qkv[:, 2 * heads * D:].unflatten(-1, (heads, D))
    k[3, 0, 5] = float("nan")
    k[4, heads - 1, :] = 0.625  # a constant group
    v[6, 0, 1] = float("inf") if dtype == torch.float16 else 1e30
    v[7, 0, 2] = float("-inf")
    v[8, 0, :64] = torch.arange(64, device=DEV).to(dtype) * 0.5  # steps and halves of them: ties
    v[9, 0, :64] = torch.arange(64, device=DEV).to(dtype) * 2.0 ** -24  # subnormal fp16
    table, pages = R.tables(lens, size, 1, DEV, spare=1)
    cache = api.KV4Cache.empty(pages, heads, size, D, weights=True, device=DEV)
    cache.weight.fill_(3.0)
    ko, vo = torch.full((T + 3, heads, D), 9.0, dtype=dtype, device=DEV), torch.full((T + 3, heads, D), 9.0, dtype=dtype, device=DEV)
    st = R.starts(counts, DEV)
    api.kv4_append(k, v, cache, table, ints(*lens), st, k_out=ko, v_out=vo)
    torch.cuda.synchronize()
    touched = torch.zeros(cache.k.shape[:3], dtype=torch.bool, device=DEV)
    for b, n in enumerate(counts):
        page, slot, ok = R.slots(cache, table, b, lens[b])
        page, slot, ok = (x[lens[b] - n:] for x in (page, slot, ok))
        rows = torch.arange(st[b].item(), st[b].item() + n, device=DEV)
        check_append(k, cache.k, cache.k_scale, ko, page, slot, ok, rows)
        check_append(v, cache.v, cache.v_scale, vo, page, slot, ok, rows)
        touched[page, :, slot] = True
    assert torch.all(cache.weight[touched] == 0) and torch.all(cache.weight[~touched] == 3)
    assert torch.all(cache.k[~touched] == 0) and torch.all(cache.v_scale[~touched] == 0)
    assert torch.all(ko[T:] == 9) and torch.all(vo[T:] == 9)  # rows behind the last sequence


def test_append_without_a_place(cuda_device):
    """Bad pages, positions before the start and past the table, offsets that run backwards: nothing is written there."""
    D, heads, size = 64, 2, 16
    k = torch.randn((40, heads, D), device=DEV).half()
    cache = api.KV4Cache.empty(4, heads, size, D, device=DEV)
    table = ints(0, -1, 7, 1, 2, 3).view(3, 2)
    # sequence 0: tokens 0..19, the last 4 on page -1; 1: page 7 does not exist, then page 1; 2: 40 tokens for 32 places
    out = torch.full_like(k, 5.0)
    api.kv4_append(k, k, cache, table, ints(20, 18, 40), ints(0, 20, 25, 35), k_out=out)
    torch.cuda.synchronize()
    q, _, _ = R.quantise(k)
    got = torch.stack([cache.k & 15, cache.k >> 4], -1).flatten(-2).double()
    assert torch.equal(got[0], q[:16].transpose(0, 1))
    assert torch.equal(got[1, :, :2], q[23:25].transpose(0, 1)) and not got[1, :, 2:].any()
    assert not got[2].any() and torch.equal(got[3, :, 14:], q[25:27].transpose(0, 1)) and not got[3, :, :14].any()
    assert torch.all(out[16:23] == 5) and torch.all(out[27:] == 5)
    cache2 = api.KV4Cache.empty(4, heads, size, D, device=DEV)
    api.kv4_append(k, k, cache2, ints(0, 1, 2, 3).view(4, 1), ints(5, 5, 2, 0), ints(0, 3, 1, 9, 99))
    torch.cuda.synchronize()
    # offsets that run backwards break the contract: rows may be left out, but none goes where no sequence has it (0:
    # rows 0..2 at 2..4; 2: rows 1..8, length 2, the last two at 0 and 1; 1 and 3, past the tokens: nothing)
    got = torch.stack([cache2.k & 15, cache2.k >> 4], -1).flatten(-2).double()
    want = torch.zeros_like(got)
    want[0, :, 2:5], want[2, :, :2] = q[:3].transpose(0, 1), q[7:9].transpose(0, 1)
    written = got.any(-1, keepdim=True)
    assert torch.equal(got, torch.where(written, want, 0.0)) and written[2, :, :2].all() and written[0, :, 2].all()


# --------------------------------------------------------------- attention
def run_attention(cache, table, lens, counts, heads, D, dtype, accumulate, scale=None, seed=3, extra=2, q=None):
    T = sum(counts)
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    if q is None:
        joint = torch.randn((T + extra, (heads + 2) * D), generator=g, device=DEV).to(dtype)
        q = joint[:, :heads * D].unflatten(-1, (heads, D))  # a slice of a joint projection
    st, ln = R.starts(counts, DEV), ints(*lens)
    out = torch.full((T + extra, heads, D), 7.0, dtype=dtype, device=DEV)
    before = cache.weight.clone() if accumulate else None
    api.kv4_attention(q, cache, table, ln, st, max_queries=max(counts + [1]), scale=scale, out=out,
                      accumulate_weight=accumulate)
    torch.cuda.synchronize()
    sc = D ** -0.5 if scale is None else scale
    want, add, tol, add_tol = R.attention(q, cache, table, ln, st, sc)
    assert torch.all(out[T:] == 7)  # rows behind the last sequence
    err = (out[:T].double() - want[:T]).abs()
    assert torch.isfinite(out[:T]).all()
    assert torch.all(err <= tol[:T]), f"worst {((err - tol[:T]).max()).item()} over, err {err.max().item()}"
    if accumulate:
        total = before.double() + add
        werr = (cache.weight.double() - total).abs()
        assert torch.all(werr <= add_tol + total.abs() * 2.0 ** -21), f"weights off by {werr.max().item()}"
    return q, out


SHAPES = [  # D, heads, kv_heads, page, lengths, query counts
    (64, 4, 4, 16, [1, 15, 16, 17, 33], [1, 1, 1, 1, 1]),
    (128, 32, 8, 64, [300, 0, 64, 65, 1], [1, 1, 1, 1, 1]),
    (128, 8, 8, 32, [700], [1]),
    (128, 20, 4, 48, [95, 96, 97, 500], [3, 0, 2, 7]),
    (256, 6, 2, 16, [250, 31, 3], [2, 1, 5]),
    (128, 16, 1, 128, [1000, 129], [1, 4]),
    (64, 40, 8, 16, [2049, 5, 777], [8, 5, 1]),
    (64, 3, 1, 32, [40], [33]),
    (256, 32, 2, 64, [130], [3]),
    (128, 64, 8, 64, [5003], [1]),
    (128, 4, 2, 16, [70, 0, 20], [0, 0, 0]),
    (128, 5, 1, 16, [4], [9]),  # more queries than tokens: the first ones see nothing
    (64, 8, 2, 16, [(7 * i) % 61 for i in range(150)], [i % 4 for i in range(150)]),  # items shorter than a block's share
    (128, 16, 2, 32, [5, 40, 33, 0, 7], [5, 3, 8, 1, 2]),
    (128, 24, 8, 64, [(29 * i) % 200 + 1 for i in range(97)], [1] * 97),  # more items than blocks
]


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,heads,kv,size,lens,counts", SHAPES)
def test_attention(cuda_device, D, heads, kv, size, lens, counts, dtype, accumulate):
    table, pages = R.tables(lens, size, 5, DEV, spare=2)
    cache = R.random_cache(api, max(pages, 1), kv, size, D, accumulate, 11, DEV)
    run_attention(cache, table, lens, counts, heads, D, dtype, accumulate)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_attention_garbage_behind_the_end(cuda_device, D):
    """Slots behind a sequence's end hold NaN, infinite and huge steps; so do pages that no table names."""
    lens, size, kv = [19, 64, 33], 32, 2
    table, pages = R.tables(lens, size, 2, DEV)
    cache = R.random_cache(api, pages + 2, kv, size, D, True, 4, DEV)
    mask = torch.ones(cache.k.shape[:3], dtype=torch.bool, device=DEV)
    for b, n in enumerate(lens):
        page, slot, _ = R.slots(cache, table, b, n)
        mask[page, :, slot] = False
    where = mask[..., None, None].expand_as(cache.k_scale)
    bad = torch.tensor([float("nan"), float("inf"), 65504.0, -65504.0], device=DEV).half()
    for s in (cache.k_scale, cache.v_scale):
        s[where] = bad.repeat(int(where.sum()) // 4 + 1)[: int(where.sum())]
    run_attention(cache, table, lens, [1, 2, 1], 8, D, torch.bfloat16, True)


def test_attention_bad_pages(cuda_device):
    """Tokens on pages that do not exist are not seen; a sequence of nothing else gives zeros."""
    lens, size, kv, D = [200, 40, 64], 16, 2, 128
    table, pages = R.tables(lens, size, 8, DEV)
    cache = R.random_cache(api, pages, kv, size, D, True, 6, DEV)
    table[0, 3], table[0, 4], table[0, 0] = -1, pages, 2 ** 31 - 1
    table[1, :] = -5
    _, out = run_attention(cache, table, lens, [1, 1, 1], 4, D, torch.float16, True)
    assert torch.all(out[1] == 0)


def test_attention_length_past_the_table(cuda_device):
    lens, size, kv, D = [32, 48], 16, 1, 64
    table, pages = R.tables(lens, size, 8, DEV)
    cache = R.random_cache(api, pages, kv, size, D, False, 6, DEV)
    run_attention(cache, table[:, :2].contiguous(), [1000, 2 ** 31 - 1], [1, 1], 2, D, torch.float16, False)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attention_wide_range(cuda_device, dtype):
    """Sharp softmaxes, steps over five orders of magnitude between tokens, zero and tiny queries."""
    lens, size, kv, D = [515, 130], 64, 2, 128
    table, pages = R.tables(lens, size, 9, DEV)
    cache = R.random_cache(api, pages, kv, size, D, True, 12, DEV, spread=0.05)
    g = torch.Generator(device=DEV)
    g.manual_seed(1)
    f = torch.exp(torch.empty(cache.v_scale.shape[:-1], device=DEV).uniform_(-11.0, 3.0, generator=g))
    cache.v_scale.copy_(cache.v_scale.float() * f[..., None])
    q = torch.randn((4, 8, D), generator=g, device=DEV) * 20
    q[0, 1] = 0
    q[0, 2] *= 1e-6
    q[1, 3, 1:] = 0
    q[1, 4, 0] = 200
    run_attention(cache, table, lens, [1, 1], 8, D, dtype, True, q=q.to(dtype))


def test_attention_large_bf16_queries(cuda_device):
    """bf16 queries past fp16's range."""
    lens, size, kv, D = [100], 16, 1, 64
    table, pages = R.tables(lens, size, 9, DEV)
    cache = R.random_cache(api, pages, kv, size, D, False, 13, DEV)
    q = (torch.randn((3, 4, D), device=DEV) * 3e6).bfloat16()
    run_attention(cache, table, lens, [1], 4, D, torch.bfloat16, False, scale=1e-7, q=q)


def test_attention_nan_stays(cuda_device):
    """A NaN that a sequence does see reaches its outputs, and only those."""
    lens, size, kv, D = [50, 60], 16, 2, 64
    table, pages = R.tables(lens, size, 3, DEV)
    cache = R.random_cache(api, pages, kv, size, D, False, 14, DEV)
    page, slot, _ = R.slots(cache, table, 0, 50)
    cache.k_scale[page[20], 1, slot[20], 0, 0] = float("nan")
    q = torch.randn((2, 4, D), device=DEV).half()
    out = api.kv4_attention(q, cache, table, ints(*lens), ints(0, 1, 2))
    torch.cuda.synchronize()
    assert out[0, 2:].isnan().all() and not out[0, :2].isnan().any() and not out[1].isnan().any()
    q[1, 0, 3] = float("nan")
    out = api.kv4_attention(q, cache, table, ints(*lens), ints(0, 1, 2))
    torch.cuda.synchronize()
    assert out[1, 0].isnan().all() and not out[1, 1:].isnan().any()


def test_attention_many_short_sequences(cuda_device):
    lens = [(i * 37) % 90 for i in range(300)]
    table, pages = R.tables(lens, 16, 3, DEV)
    cache = R.random_cache(api, pages, 2, 16, 64, True, 15, DEV)
    run_attention(cache, table, lens, [1] * 300, 4, 64, torch.float16, True)


def test_attention_shared_prefix_and_repeat(cuda_device):
    """Two sequences that share pages; the same call again gives the same bits."""
    lens, size, kv, D = [150, 150, 64], 32, 2, 128
    table, pages = R.tables(lens, size, 3, DEV)
    table[1, :3] = table[0, :3]
    table[2, :2] = table[0, :2]
    cache = R.random_cache(api, pages, kv, size, D, False, 16, DEV)
    q, out = run_attention(cache, table, lens, [2, 1, 1], 8, D, torch.bfloat16, False)
    again = api.kv4_attention(q, cache, table, ints(*lens), ints(0, 2, 3, 4), max_queries=2)
    torch.cuda.synchronize()
    assert torch.equal(out[:4], again[:4]) and torch.all(again[4:] == 0)


def test_attention_far_pages(cuda_device):
    """A cache whose last pages lie past 4 GB (offsets past 32 bits), read and written there."""
    heads, size, D = 8, 64, 256
    pages = 70000  # 70000 * 8 * 64 * 128 bytes = 4.6 GB of keys
    cache = api.KV4Cache.empty(pages, heads, size, D, device=DEV)
    k = torch.randn((65, heads, D), device=DEV).half()
    v = torch.randn((65, heads, D), device=DEV).half()
    table = ints(pages - 1, 69000).view(1, 2)
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    api.kv4_append(k, v, cache, table, ints(65), ints(0, 65), k_out=ko, v_out=vo)
    q = torch.randn((1, heads, D), device=DEV).half()
    out = api.kv4_attention(q, cache, table, ints(65), ints(0, 1))
    torch.cuda.synchronize()
    p = torch.softmax(torch.einsum("hd,nhd->hn", q[0].double(), ko.double()) / 16, -1)
    want = torch.einsum("hn,nhd->hd", p, vo.double())
    # the values were rounded to fp16 once more here: 2^-11 of each key (scores: 2^-11 sum |q k| / 16) and value
    d = torch.einsum("hd,nhd->hn", q[0].double().abs(), ko.double().abs()).amax() / 16
    tol = (2 * d * 2.0 ** -11 + 4 * 2.0 ** -11) * torch.einsum("hn,nhd->hd", p, vo.double().abs() + 4)
    assert torch.all((out[0].double() - want).abs() <= tol)


def test_attention_graph_and_streams(cuda_device):
    """Captured and replayed with new contents, beside another call on a second stream."""
    lens, size, kv, D = [1200, 300], 64, 2, 128
    table, pages = R.tables(lens, size, 3, DEV)
    cache = R.random_cache(api, pages, kv, size, D, True, 17, DEV)
    q = torch.randn((2, 8, D), device=DEV).half()
    ln, st = ints(*lens), ints(0, 1, 2)
    out = torch.zeros_like(q)
    api.kv4_attention(q, cache, table, ln, st, out=out, accumulate_weight=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        api.kv4_attention(q, cache, table, ln, st, out=out, accumulate_weight=True)
    q.copy_(torch.randn((2, 8, D), device=DEV))
    ln.copy_(ints(900, 250))
    before = cache.weight.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph.replay()
    other = api.kv4_attention(q, cache, table, ln, st, stream=side)
    torch.cuda.synchronize()
    want, add, tol, add_tol = R.attention(q, cache, table, ln, st, D ** -0.5)
    assert torch.all((out.double() - want).abs() <= tol) and torch.equal(out, other)
    total = before.double() + add
    assert torch.all((cache.weight.double() - total).abs() <= add_tol + total * 2.0 ** -21)


# ------------------------------------------------------------------- evict
def check_evict(cache, lens, size, budget, recent, table, first, new_lens_cap=None):
    new_table, pages = R.tables([min(n, budget) for n in lens], size, 21, DEV, first=first)
    old = {n: getattr(cache, n).clone() for n in ("k", "v", "k_scale", "v_scale", "weight")}
    new = api.kv4_evict(cache, table, ints(*lens), new_table, budget, recent)
    torch.cuda.synchronize()
    assert new.tolist() == [min(n, budget) for n in lens]
    want = {n: t.clone() for n, t in old.items()}
    for b, n in enumerate(lens):
        page, slot, _ = R.slots(cache, table, b, n)
        npage, nslot, _ = R.slots(cache, new_table, b, min(n, budget))
        for h in range(cache.kv_heads):
            keep = torch.tensor(R.kept(old["weight"][page, h, slot], n, budget, recent), dtype=torch.long, device=DEV)
            for name, t in old.items():
                want[name][npage, h, nslot] = t[page[keep], h, slot[keep]]
    for name, t in want.items():
        got = getattr(cache, name)
        bits = {1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()]
        assert torch.equal(got.view(bits), t.view(bits)), name


@pytest.mark.parametrize("D,kv,size,lens,budget,recent", [
    (64, 2, 16, [40, 16, 17, 0, 1, 100], 16, 4),
    (128, 8, 64, [1000, 300, 257], 256, 32),
    (256, 1, 32, [129, 128, 127], 127, 127),
    (64, 1, 16, [500, 33], 32, 0),
    (128, 2, 16, [64, 10], 0, 0),
    (64, 1, 64, [50000, 41000], 5000, 100),
    (64, 2, 64, [6000], 5999, 7),
    (64, 1, 64, [50000, 300, 0], 40000, 100),  # more rows a block than it lists at a time, short ones in a wide table
    (128, 1, 32, [44000], 36000, 0),
])
def test_evict(cuda_device, D, kv, size, lens, budget, recent):
    table, pages = R.tables(lens, size, 20, DEV, spare=1)
    room = sum(-(-min(n, budget) // size) for n in lens)
    cache = R.random_cache(api, pages + room + 1, kv, size, D, True, 22, DEV)
    check_evict(cache, lens, size, budget, recent, table, pages)


@pytest.mark.parametrize("kind", ["equal", "few", "zeros", "odd"])
def test_evict_ties_and_odd_weights(cuda_device, kind):
    lens, size, budget, recent = [333, 200], 16, 100, 10
    table, pages = R.tables(lens, size, 20, DEV)
    cache = R.random_cache(api, pages + 20, 2, size, 64, True, 23, DEV)
    w = cache.weight
    if kind == "equal":
        w.fill_(0.25)
    elif kind == "few":
        w.copy_((w * 3).floor())
    elif kind == "zeros":
        w.copy_(torch.where(w > 1, 0.0, -0.0))
    else:
        w.flatten()[::5] = float("nan")
        w.flatten()[1::7] = float("inf")
        w.flatten()[2::9] = float("-inf")
        w.flatten()[3::4] *= -1e-40
    check_evict(cache, lens, size, budget, recent, table, pages)


def test_evict_bad_pages_and_short_table(cuda_device):
    """Tokens on pages that do not exist weigh least and copy nothing; a new table with too few places cuts further."""
    size, kv, D = 16, 1, 64
    cache = R.random_cache(api, 8, kv, size, D, True, 24, DEV)
    keep = {n: getattr(cache, n).clone() for n in ("k", "weight")}
    table = ints(0, -1, 1, 99).view(1, 4)
    new = api.kv4_evict(cache, table, ints(64), ints(4, 9, 5).view(1, 3), budget=40, recent=0)
    torch.cuda.synchronize()
    assert new.tolist() == [40]
    # 32 real tokens, then positions 16..23 of the missing page: kept positions 0..23 and 32..47
    assert torch.equal(cache.k[4, 0], keep["k"][0, 0])  # 16..31 went to page 9, which does not exist
    assert torch.equal(cache.weight[5, 0, :8], keep["weight"][1, 0, 8:16])
    for p in (2, 3, 6, 7):
        assert torch.equal(cache.k[p], keep["k"][p])
    new = api.kv4_evict(cache, ints(0, 1).view(1, 2), ints(32), ints(6).view(1, 1), budget=20, recent=2)
    torch.cuda.synchronize()
    assert new.tolist() == [16]
    w = torch.cat([keep["weight"][0, 0], keep["weight"][1, 0]])
    pos = torch.tensor(R.kept(w, 32, 16, 2), device=DEV)
    assert torch.equal(cache.weight[6, 0], w[pos])


@pytest.mark.parametrize("budget", [2 ** 31 - 1, 2 ** 32 - 1, 2 ** 40])
def test_evict_without_a_bound(cuda_device, budget):
    """Budgets that no table reaches keep everything."""
    lens, size = [70, 5], 16
    table, pages = R.tables(lens, size, 20, DEV)
    cache = R.random_cache(api, pages + 6, 1, size, 64, True, 25, DEV)
    check_evict(cache, lens, size, budget, 3, table, pages)
    new = torch.zeros(2, dtype=torch.int32, device=DEV)
    fresh, _ = R.tables(lens, size, 22, DEV, first=pages)
    ln = ints(*lens)
    seqs = (table.data_ptr(), 2, table.shape[1], ln.data_ptr(), fresh.data_ptr(), fresh.shape[1])
    st = _lib.load().b2sq_kv4_evict(cache._ref, *seqs, budget & 0xffffffff, 0, new.data_ptr(), None)
    torch.cuda.synchronize()
    assert st == 0 and (budget & 0xffffffff == 0 or new.tolist() == lens)


# ------------------------------------------------------------ all together
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_serving_loop(cuda_device, dtype):
    """A prompt is appended, tokens are decoded one by one with their weights added up, the cache is thinned out and
    decoding goes on; the cache always holds what a plain restatement says."""
    kv, heads, D, size, budget, recent = 2, 8, 128, 16, 48, 8
    lens, B = [70, 33, 52], 3
    cache = api.KV4Cache.empty(40, kv, size, D, weights=True, device=DEV)
    table, first = R.tables([96] * B, size, 30, DEV)
    g = torch.Generator(device=DEV)
    g.manual_seed(2)

    def rows(n, h):
        return torch.randn((n, h, D), generator=g, device=DEV).to(dtype)

    counts = list(lens)
    for step in range(6):
        T = sum(counts)
        k, v, q = rows(T, kv), rows(T, kv), rows(T, heads)
        ln, st = ints(*lens), R.starts(counts, DEV)
        api.kv4_append(k, v, cache, table, ln, st)
        before = cache.weight.clone()
        out = api.kv4_attention(q, cache, table, ln, st, max_queries=max(counts), accumulate_weight=True)
        torch.cuda.synchronize()
        want, add, tol, add_tol = R.attention(q, cache, table, ln, st, D ** -0.5)
        assert torch.all((out.double() - want).abs() <= tol)
        total = before.double() + add
        assert torch.all((cache.weight.double() - total).abs() <= add_tol + total * 2.0 ** -20)
        for b in range(B):
            page, slot, ok = R.slots(cache, table, b, lens[b])
            n = counts[b]
            check_append(k, cache.k, cache.k_scale, None, page[-n:], slot[-n:], ok, torch.arange(st[b], st[b] + n, device=DEV))
        if step == 3:
            check = cache.weight.clone()
            fresh, _ = R.tables([budget + 16] * B, size, 31, DEV, first=first)
            new = api.kv4_evict(cache, table, ln, fresh, budget, recent)
            for b in range(B):
                for h in range(kv):
                    page, slot, _ = R.slots(cache, table, b, lens[b])
                    keep = R.kept(check[page, h, slot], lens[b], budget, recent)
                    npage, nslot, _ = R.slots(cache, fresh, b, len(keep))
                    assert torch.equal(cache.weight[npage, h, nslot], check[page[keep], h, slot[keep]])
            lens, table = new.tolist(), fresh
        counts = [1] * B
        lens = [n + 1 for n in lens]
