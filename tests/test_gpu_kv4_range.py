"""The 4-bit cache's attention at the ends of its types' ranges."""
import pytest
import torch

import kv4_ref as R
from optimized_rocwmma_samples_b200 import api
from test_gpu_kv4 import DEV, ints, run_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("mag", [2.0 ** 100, 2.0 ** 115, 2.0 ** 116, 2.0 ** 122, 2.0 ** 127])
def test_huge_bf16_queries(cuda_device, mag, D, accumulate):
    """Scores that 64 bits hold and whose softmax is 0 or 1: the output is one token's value, the weight goes to it.

    Rows are looked at where the best token leads by 2^-10 of the sum of |q k|: scores are off by (D + 8) 2^-23 of that at
    most, 2^-14.9.  A probability of 1 makes each value q * step + base, an fp32 product and sum (2^-22 of either)
    rounded to bf16."""
    kv, group, size, n, batch = 2, 4, 16, 30, 6
    table, pages = R.tables([n] * batch, size, 3, DEV)
    cache = R.random_cache(api, pages, kv, size, D, accumulate, 31, DEV)
    if accumulate:
        cache.weight.zero_()
    g = torch.Generator(device=DEV)
    g.manual_seed(5)
    q = torch.randn((batch, kv * group, D), generator=g, device=DEV)
    q[:, ::2, 1:] = 0
    q = (q / q.abs().amax(-1, keepdim=True)).bfloat16() * torch.tensor(mag, dtype=torch.bfloat16, device=DEV)
    assert torch.isfinite(q).all()
    out = api.kv4_attention(q, cache, table, ints(*[n] * batch), ints(*range(batch + 1)), accumulate_weight=accumulate)
    torch.cuda.synchronize()
    assert torch.isfinite(out).all()
    K, V = R.values(cache)
    Vq = R.values_nibble(cache.v, cache.v_scale)
    looked = 0
    want_w, sure = torch.zeros((pages, kv, size), dtype=torch.float64, device=DEV), torch.ones((batch, kv), dtype=torch.bool)
    for b in range(batch):
        page, slot, _ = R.slots(cache, table, b, n)
        for h in range(kv * group):
            k = K[page, h // group, slot]
            s = k @ q[b, h].double()
            best = s.argmax().item()
            lead = s[best] - torch.cat([s[:best], s[best + 1:]]).max()
            if lead < 2.0 ** -10 * (k.abs() @ q[b, h].double().abs()).max():
                sure[b, h // group] = False
                continue
            looked += 1
            v, vq = V[page[best], h // group, slot[best]], Vq[page[best], h // group, slot[best]]
            tol = 2.0 ** -8 * v.abs() + 2.0 ** -22 * (v.abs() + 2 * vq) * 1.01
            assert torch.all((out[b, h].double() - v).abs() <= tol)
            want_w[page[best], h // group, slot[best]] += 1
    assert looked > batch * kv * group // 2
    if accumulate:
        for b in range(batch):
            page, slot, _ = R.slots(cache, table, b, n)
            for h in range(kv):
                if sure[b, h]:
                    assert torch.equal(cache.weight[page, h, slot].double(), want_w[page, h, slot])


@pytest.mark.parametrize("exponent", [-133, -128, -126, -118, -100])
def test_tiny_bf16_queries(cuda_device, exponent):
    """Queries down to the smallest subnormals, with a scale that brings the scores back."""
    lens, size, kv, D = [100, 37], 16, 2, 64
    table, pages = R.tables(lens, size, 9, DEV)
    cache = R.random_cache(api, pages, kv, size, D, False, 13, DEV)
    g = torch.Generator(device=DEV)
    g.manual_seed(6)
    q = torch.randint(-7, 8, (4, 8, D), generator=g, device=DEV).double() * 2.0 ** exponent
    q = q.bfloat16()
    run_attention(cache, table, lens, [1, 1], 8, D, torch.bfloat16, False, scale=2.0 ** min(127, -exponent - 6), q=q)


def test_largest_scale(cuda_device):
    """A scale near the largest fp32 number, with queries that bring the scores back."""
    lens, size, kv, D = [50], 16, 2, 64
    table, pages = R.tables(lens, size, 9, DEV)
    cache = R.random_cache(api, pages, kv, size, D, False, 13, DEV)
    q = (torch.randn((3, 4, D), device=DEV) * 2.0 ** -130).bfloat16()
    run_attention(cache, table, lens, [1], 4, D, torch.bfloat16, False, scale=1.5 * 2.0 ** 127, q=q)
