"""The 4-bit cache's operators restated plainly in 64 bits, for the tests."""
import torch

GROUP = 64


def quantise(x):
    """(nibbles, fp16 steps, fp16 bases) of x [..., D] by the cache's rule."""
    y = x.float().clamp(-65504.0, 65504.0).unflatten(-1, (-1, GROUP))
    low, high = y.amin(-1), y.amax(-1)  # NaN stays
    step = torch.div(high - low, torch.full_like(low, 15.0)).half()
    base = low.half()
    s, z = step.double().unsqueeze(-1), base.double().unsqueeze(-1)
    q = torch.where(s > 0, ((y.double() - z) / s).round().clamp(0, 15), torch.zeros_like(s))
    return q.flatten(-2), step, base


def values(cache):
    """(keys, values) of every slot, float64 [pages, heads, page_size, D]."""
    out = []
    for data, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        q = torch.stack([data & 15, data >> 4], -1).flatten(-2).double().unflatten(-1, (-1, GROUP))
        out.append((q * scale[..., 0:1].double() + scale[..., 1:2].double()).flatten(-2))
    return out


def slots(cache, table, b, n):
    """(page, slot, present) of the first n positions of sequence b (positions past the table are left out)."""
    pos = torch.arange(min(n, table.shape[1] * cache.page_size), device=table.device)
    page = table[b].long()[pos // cache.page_size]
    ok = (page >= 0) & (page < cache.pages)
    return page.clamp(0, max(cache.pages - 1, 0)), pos % cache.page_size, ok


def attention(q, cache, table, lens, starts, scale):
    """(out float64, weights added float64, tolerance of out, tolerance of the weights).

    Tolerances, per element: a score's fp32 sum of D products and its scaling is off by at most d =
    (D + 8) 2^-23 scale sum |q| (|q4 s| + |z|); p, a ratio of exponentials, by (2 d + 2^-20) p; the p that
    multiplies the nibbles is rounded to 11 bits, 2^-11 p; the result is rounded once to its type."""
    T, hq, D = q.shape
    hk = cache.kv_heads
    K, V = values(cache)
    Kabs = values_abs(cache, cache.k, cache.k_scale)
    Vq = values_nibble(cache.v, cache.v_scale)
    out = torch.zeros((T, hq, D), dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    add = torch.zeros(cache.k.shape[:3], dtype=torch.float64, device=q.device)
    add_tol = torch.zeros_like(add)
    for b, length in enumerate(lens.tolist()):
        t0, t1 = starts[b].item(), starts[b + 1].item()
        for i in range(t1 - t0):
            see = max(0, length - (t1 - t0) + i + 1)
            page, slot, ok = slots(cache, table, b, see)
            page, slot = page[ok], slot[ok]
            if page.numel() == 0:
                continue
            k, v = K[page, :, slot].transpose(0, 1), V[page, :, slot].transpose(0, 1)  # [hk, n, D]
            qi = q[t0 + i].double().view(hk, hq // hk, D)
            p = torch.softmax(torch.einsum("hgd,hnd->hgn", qi, k) * scale, -1)
            d = torch.einsum("hgd,hnd->hgn", qi.abs(), Kabs[page, :, slot].transpose(0, 1)).amax(-1, keepdim=True)
            rel = 2 * d * abs(scale) * (D + 8) * 2.0 ** -23 + 2.0 ** -20
            o = torch.einsum("hgn,hnd->hgd", p, v)
            err = 2.0 ** -11 * torch.einsum("hgn,hnd->hgd", p, Vq[page, :, slot].transpose(0, 1))
            err += rel * torch.einsum("hgn,hnd->hgd", p, v.abs())
            half = torch.finfo(q.dtype).eps / 2
            out[t0 + i] = o.reshape(hq, D)
            tol[t0 + i] = (half * (o.abs() + err) + err + 2.0 ** -25).reshape(hq, D)  # fp16 subnormals: 2^-25
            add[page, :, slot] += p.sum(1).t()
            add_tol[page, :, slot] += (rel * p).sum(1).t()
    return out, add, tol, add_tol


def values_abs(cache, data, scale):
    q = torch.stack([data & 15, data >> 4], -1).flatten(-2).double().unflatten(-1, (-1, GROUP))
    return (q * scale[..., 0:1].double().abs() + scale[..., 1:2].double().abs()).flatten(-2)


def values_nibble(data, scale):
    q = torch.stack([data & 15, data >> 4], -1).flatten(-2).double().unflatten(-1, (-1, GROUP))
    return (q * scale[..., 0:1].double().abs()).flatten(-2)


def kept(weight, n, budget, recent):
    """Positions that a head of n tokens keeps: a list in order."""
    if n <= budget:
        return list(range(n))
    w = weight[: n - recent].tolist()
    order = sorted(range(n - recent), key=lambda i: (0 if w[i] != w[i] else 1, 0.0 if w[i] != w[i] else -w[i], i))
    return sorted(order[: budget - recent]) + list(range(n - recent, n))


def random_cache(api, pages, heads, size, dim, weights, seed, device, spread=0.3):
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    c = api.KV4Cache.empty(pages, heads, size, dim, weights, device)
    for data, scale in ((c.k, c.k_scale), (c.v, c.v_scale)):
        data.copy_(torch.randint(0, 256, data.shape, generator=g, device=device, dtype=torch.uint8))
        step = torch.empty(scale.shape[:-1], device=device).uniform_(0.3 * spread, 1.7 * spread, generator=g)
        base = -step * torch.empty_like(step).uniform_(5.0, 9.0, generator=g)
        scale.copy_(torch.stack([step, base], -1))
    if weights:
        c.weight.copy_(torch.empty(c.weight.shape, device=device).exponential_(generator=g))
    return c


def tables(lens, size, seed, device, first=0, spare=0):
    """A page table with every sequence's pages in a random order from page `first` on; returns it and the page after."""
    need = [-(-max(n, 0) // size) for n in lens]
    g = torch.Generator()
    g.manual_seed(seed)
    order = (torch.randperm(sum(need), generator=g) + first).to(torch.int32)
    t = torch.full((len(lens), max(need + [1]) + spare), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        t[b, :n] = order[at:at + n]
        at += n
    return t.to(device), first + sum(need)


def starts(counts, device):
    at = [0]
    for n in counts:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device=device)
