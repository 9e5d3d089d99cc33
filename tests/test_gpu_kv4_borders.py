"""Nibbles whose quotient lies on, or by less than fp32 can tell beside, a border between two steps."""
import pytest
import torch

from optimized_rocwmma_samples_b200 import api
from test_gpu_kv4 import DEV, ints

pytestmark = pytest.mark.gpu


def nibbles(x):
    """The cache's nibbles, steps and bases for x [tokens, 1, 64]."""
    T = x.shape[0]
    pages = -(-T // 16)
    cache = api.KV4Cache.empty(pages, 1, 16, 64, device=DEV)
    table = torch.arange(pages, dtype=torch.int32, device=DEV).view(1, pages)
    api.kv4_append(x, x, cache, table, ints(T), ints(0, T))
    torch.cuda.synchronize()
    q = torch.stack([cache.k & 15, cache.k >> 4], -1).flatten(-2).flatten(0, 2)[:T]
    return q.long(), cache.k_scale.flatten(0, 2)[:T, 0]


def exact(x, scale):
    """rint((v - z) / s), ties to even, in whole numbers: v, z and s are multiples of 2^-133 (bf16) or 2^-24 (fp16)."""
    out = torch.zeros(x.shape[0], 64, dtype=torch.long)
    rows, steps = x[:, 0].double().cpu().tolist(), scale.double().cpu().tolist()
    for t, (row, (s, z)) in enumerate(zip(rows, steps)):
        den = int(s * 2.0 ** 140)
        for c, v in enumerate(row):
            num = int(v * 2.0 ** 140) - int(z * 2.0 ** 140)  # exact: Python's whole numbers
            if den == 0:
                continue
            q, r = divmod(num, den)
            q += 2 * r > den or (2 * r == den and q & 1)
            out[t, c] = min(max(q, 0), 15)
    return out.to(x.device)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_ties_that_fp32_cannot_tell(cuda_device, dtype):
    """Base -7.5 s and step s put a border at 0: the smallest numbers beside it lie on one side or the other."""
    rows = []
    smallest = 2.0 ** -24 if dtype == torch.float16 else 2.0 ** -133
    for e in (-6, 0, 3, 9):
        s = 2.0 ** e
        for sign in (1, -1):
            row = torch.zeros(64, dtype=torch.float64)
            row[0], row[1] = -7.5 * s, 7.5 * s
            tiny = torch.tensor([smallest * 2.0 ** (k % 12) for k in range(16)], dtype=torch.float64)
            row[2:18] = sign * tiny
            row[18:34] = -sign * tiny
            row[34:49] = (torch.arange(15, dtype=torch.float64) - 7) * s  # ties, exactly
            rows.append(row)
    x = torch.stack(rows).view(-1, 1, 64).to(DEV).to(dtype)
    q, scale = nibbles(x)
    assert torch.equal(scale[:, 0].double().cpu(), torch.tensor([2.0 ** e for e in (-6, 0, 3, 9) for _ in range(2)], dtype=torch.float64))
    want = exact(x, scale)
    assert torch.equal(q, want)
    assert set(want[:, 2:34].flatten().tolist()) == {7, 8}


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_random_groups_exactly(cuda_device, dtype):
    """Groups of all magnitudes, a wide mix within each, against whole-number arithmetic."""
    g = torch.Generator(device=DEV)
    g.manual_seed(1)
    x = torch.randn((400, 1, 64), generator=g, device=DEV)
    low = -14.0 if dtype == torch.float16 else -30.0
    x *= torch.exp2(torch.empty((400, 1, 1), device=DEV).uniform_(low, 10.0, generator=g))
    x[::2] *= torch.exp2(torch.empty((200, 1, 64), device=DEV).uniform_(-16.0, 0.0, generator=g))
    x = x.to(dtype)
    q, scale = nibbles(x)
    assert torch.equal(q, exact(x, scale))
