"""How exact the 4-bit cache's attention is: error norms against 64 bits, in units of the rounding that the result's type
makes by itself."""
import pytest
import torch

import kv4_ref as R
from optimized_rocwmma_samples_b200 import api

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def norms(out, want):
    """(error, rounding of the exact result) relative to the result."""
    return tuple(((x.double() - want).norm() / want.norm()).item() for x in (out, want.to(out.dtype)))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,kv,group,size,pages", [(128, 8, 4, 64, 64), (64, 16, 1, 32, 64), (256, 4, 4, 16, 64),
                                                   (128, 2, 16, 64, 64), (128, 4, 4, 48, 64)])
def test_long_sums(cuda_device, dtype, D, kv, group, size, pages):
    """64 sequences of 131072 tokens: a warp adds up some thousands of them.

    The tokens repeat (a table may name a page many times), so that their softmax is the short sequence's.  Sums of
    nibbles run to about 15 times the result here.  In fp32 n additions that round are off by about 2^-24 sqrt(n) of the
    sum: with n below 5000, 15 * 2^-24 * 71 = 6.3e-5 of the result.  fp16's own rounding is 2.2e-4, so errors stay below
    1.25 of it (1.25^2 - 1 = 0.75^2 leaves 1.6e-4).  Sums that are cut off are off by n 2^-24 instead, 2e-3 and more."""
    batch, n = 64, 131072 // (pages * size) * pages * size
    cache = R.random_cache(api, pages, kv, size, D, False, 5, DEV)
    g = torch.Generator(device=DEV)
    g.manual_seed(3)
    q = (torch.randn((batch, kv * group, D), generator=g, device=DEV) * 0.1).to(dtype)
    table = torch.arange(pages, dtype=torch.int32, device=DEV).repeat(n // (pages * size)).expand(batch, -1).contiguous()
    out = api.kv4_attention(q, cache, table, torch.full((batch,), n, dtype=torch.int32, device=DEV),
                            torch.arange(batch + 1, dtype=torch.int32, device=DEV))
    k, v = (x.transpose(0, 1).flatten(1, 2) for x in R.values(cache))
    p = torch.softmax(torch.einsum("bhgd,hnd->bhgn", q.double().view(batch, kv, group, D), k) * D ** -0.5, -1)
    want = torch.einsum("bhgn,hnd->bhgd", p, v).reshape(batch, kv * group, D)
    err, rounding = norms(out, want)
    assert err <= 1.25 * rounding, f"{err} against {rounding}"


@pytest.mark.parametrize("every", [2, 16, 32])
def test_long_sums_with_holes(cuda_device, every):
    """The same where each second, 16th or 32nd page is missing: what is set aside for the sums' centre does not pile up."""
    batch, pages, size, D, kv, group = 64, 64, 32, 128, 8, 4
    cache = R.random_cache(api, pages, kv, size, D, False, 8, DEV)
    g = torch.Generator(device=DEV)
    g.manual_seed(3)
    q = (torch.randn((batch, kv * group, D), generator=g, device=DEV) * 0.1).half()
    row = torch.arange(131072 // size, dtype=torch.int32, device=DEV)
    row = torch.where(row % every == every - 1, -1, row % pages).to(torch.int32)
    out = api.kv4_attention(q, cache, row.expand(batch, -1).contiguous(),
                            torch.full((batch,), 131072, dtype=torch.int32, device=DEV),
                            torch.arange(batch + 1, dtype=torch.int32, device=DEV))
    k, v = (x.transpose(0, 1).flatten(1, 2) for x in R.values(cache))
    there = (torch.arange(pages, device=DEV) % every != every - 1).repeat_interleave(size)
    p = torch.softmax(torch.einsum("bhgd,hnd->bhgn", q.double().view(batch, kv, group, D), k[:, there]) * D ** -0.5, -1)
    want = torch.einsum("bhgn,hnd->bhgd", p, v[:, there]).reshape(batch, kv * group, D)
    err, rounding = norms(out, want)
    assert err <= 1.25 * rounding, f"{err} against {rounding}"


def test_fp16_keeps_its_probabilities(cuda_device):
    """Few tokens, fp16: the probabilities that meet the nibbles hold more bits than fp16 has, or the result loses some.

    The kernel's two parts leave 2^-22; one part would be off by as much as the result's rounding, which the oracle below
    shows, and 1.1 of that rounding (0.46 of it beside it) tells them apart."""
    kv, group, size, D, batch, n = 4, 4, 16, 128, 64, 6
    cache = R.random_cache(api, batch, kv, size, D, False, 6, DEV)
    g = torch.Generator(device=DEV)
    g.manual_seed(4)
    q = (torch.randn((batch, kv * group, D), generator=g, device=DEV) * 0.3).half()
    table = torch.arange(batch, dtype=torch.int32, device=DEV).view(batch, 1)
    out = api.kv4_attention(q, cache, table, torch.full((batch,), n, dtype=torch.int32, device=DEV),
                            torch.arange(batch + 1, dtype=torch.int32, device=DEV))
    k, v = (x[:, :, :n] for x in R.values(cache))
    p = torch.softmax(torch.einsum("bhgd,bhnd->bhgn", q.double().view(batch, kv, group, D), k) * D ** -0.5, -1)
    want = torch.einsum("bhgn,bhnd->bhgd", p, v)
    err, rounding = norms(out.view(want.shape), want)
    assert err <= 1.1 * rounding, f"{err} against {rounding}"
    # one part: p times step rounded to fp16
    step, base = (cache.v_scale[:, :, :n, :, i].double() for i in (0, 1))
    nib = torch.stack([cache.v & 15, cache.v >> 4], -1).flatten(-2)[:, :, :n].double().unflatten(-1, (-1, 64))
    ps = torch.einsum("bhgn,bhnr->bhgnr", p, step).half().double()
    one = (torch.einsum("bhgnr,bhnrc->bhgrc", ps, nib) + torch.einsum("bhgn,bhnr->bhgr", p, base)[..., None]).flatten(-2)
    assert norms(one.half(), want)[0] > 1.2 * rounding
