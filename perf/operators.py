"""Measured cases of the decode-step operators: a mixture-of-experts layer for a few tokens, and the 4-bit paged key/value
cache (append, attention, eviction).

``run`` computes them in plain torch operations, or, where ``own`` is set, through the package's entry points.
"""
import math

import torch

own = False

QMAX = 127.0
GROUP = 64  # channels that share a step and a base in the 4-bit cache


def _dtype(case):
    return {"fp16": torch.float16, "bf16": torch.bfloat16}[case["dtype"]]


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of a batch: a token's keys and values for each of 16 sequences
        dict(name="append step", op="append", batch=16, tokens=1, kv_heads=8, dim=128, page=64, dtype="bf16"),
        # prompts of different lengths written to the cache at once
        dict(name="append prompts", op="append", batch=7, tokens=4001, kv_heads=8, dim=128, page=64, dtype="fp16"),
        # one short chat: latency
        dict(name="attend short", op="attend", batch=1, length=257, queries=1, heads=32, kv_heads=8, dim=128, page=16,
             dtype="fp16", weights=False),
        # a batch of ordinary, ragged lengths
        dict(name="attend batch", op="attend", batch=16, length=4000, queries=1, heads=32, kv_heads=8, dim=128, page=64,
             dtype="bf16", weights=False),
        # two long documents, eight query heads on each key head
        dict(name="attend long", op="attend", batch=2, length=100001, queries=1, heads=64, kv_heads=8, dim=128, page=64,
             dtype="bf16", weights=False),
        # four drafted tokens a sequence, a head of its own for each query head, weights added up
        dict(name="attend drafts", op="attend", batch=8, length=6001, queries=4, heads=16, kv_heads=16, dim=64, page=32,
             dtype="fp16", weights=True),
        # a full serving batch that adds up the attention weights for a later eviction
        dict(name="attend weights", op="attend", batch=48, length=8192, queries=1, heads=32, kv_heads=8, dim=128,
             page=64, dtype="bf16", weights=True),
        # one sequence just over its budget
        dict(name="evict one", op="evict", batch=1, length=1040, budget=1024, recent=64, kv_heads=8, dim=128, page=16),
        # a batch cut to a quarter
        dict(name="evict batch", op="evict", batch=32, length=8192, budget=2048, recent=256, kv_heads=8, dim=128, page=64),
        # one token through two of eight large experts
        dict(name="moe one token", op="moe", tokens=1, hidden=4096, inter=14336, experts=8, topk=2, dtype="fp16"),
        # a decode batch through the same layer: every expert is read
        dict(name="moe batch", op="moe", tokens=16, hidden=4096, inter=14336, experts=8, topk=2, dtype="bf16"),
        # many smaller experts
        dict(name="moe many experts", op="moe", tokens=24, hidden=4096, inter=1456, experts=32, topk=5, dtype="fp16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "evict", "moe", "moe"])
    dim = rng.choice([64, 128, 128, 256])
    page = rng.choice([16, 32, 64, 128])
    dtype = rng.choice(["fp16", "bf16"])
    if op == "append":
        batch, kv = _log(rng, 1, 64), rng.choice([1, 2, 4, 8, 16])
        most = max(1, 29_000_000 // (batch * kv * dim))
        return dict(op=op, batch=batch, tokens=_log(rng, 1, min(most, 8192)), kv_heads=kv, dim=dim, page=page, dtype=dtype)
    if op == "attend":
        batch, kv = _log(rng, 1, 64), rng.choice([1, 2, 4, 8, 16])
        group = rng.choice([1, 2, 4, 5, 8, 16])
        queries = rng.choice([1, 1, 1, 2, 3, 5, 8])
        most = 200_000_000 // (batch * kv * max(dim, 4 * group * queries))
        return dict(op=op, batch=batch, length=_log(rng, queries, max(queries + 1, min(most, 131072))), queries=queries,
                    heads=kv * group, kv_heads=kv, dim=dim, page=page, dtype=dtype, weights=rng.random() < 0.4)
    if op == "evict":
        batch, kv = _log(rng, 1, 32), rng.choice([1, 2, 4, 8, 16])
        length = _log(rng, 64, max(65, min(65536, 130_000_000 // (batch * kv * dim))))
        budget = max(2, int(length * rng.uniform(0.1, 0.99)))
        return dict(op=op, batch=batch, length=length, budget=budget, recent=rng.randint(0, budget // 2), kv_heads=kv, dim=dim,
                    page=page)
    hidden, inter = 16 * _log(rng, 16, 384), 16 * _log(rng, 8, 896)
    most = max(1, 1_300_000_000 // (3 * hidden * inter))
    experts = rng.choice([e for e in (1, 2, 4, 8, 16, 32, 64, 128) if e <= most])
    return dict(op=op, tokens=_log(rng, 1, 64), hidden=hidden, inter=inter, experts=experts,
                topk=rng.randint(1, min(8, experts)), dtype=dtype)


# ------------------------------------------------------------------------------------------------ sizes
def _lengths(case):
    """Cached tokens of each sequence: the first is the longest, the others spread below it."""
    n, low = case["length"], case.get("queries", 1)
    return [max(low, n - (i * 7919) % max(1, int(0.7 * n))) for i in range(case["batch"])]


def _counts(case):
    """New tokens of each sequence of an append."""
    n = case["tokens"]
    return [max(1, n - (i * 7919) % max(1, int(0.7 * n))) for i in range(case["batch"])]


def _row_bytes(dim):
    return dim // 2 + 4 * (dim // GROUP)  # of a token's keys, or values, in one head


def work(case):
    if case["op"] == "append":
        rows = sum(_counts(case)) * case["kv_heads"]
        return {"bytes": 2 * rows * (4 * case["dim"] + _row_bytes(case["dim"])), "flops": 8 * 2 * rows * case["dim"]}
    if case["op"] == "attend":
        lens, d = _lengths(case), case["dim"]
        seen = sum(n - case["queries"] + i + 1 for n in lens for i in range(case["queries"]))
        per = 2 * _row_bytes(d) + (8 if case["weights"] else 0)
        return {"bytes": sum(lens) * case["kv_heads"] * per + 2 * 2 * len(lens) * case["queries"] * case["heads"] * d,
                "flops": 4 * d * case["heads"] * seen}
    if case["op"] == "evict":
        lens = _lengths(case)
        kept = sum(min(n, case["budget"]) for n in lens)
        return {"bytes": case["kv_heads"] * (4 * sum(lens) + kept * (4 * _row_bytes(case["dim"]) + 4)), "flops": 0}
    t, h, i, e, k = (case[x] for x in ("tokens", "hidden", "inter", "experts", "topk"))
    active = e * (1 - (1 - k / e) ** t)
    return {"bytes": active * (3 * h * i + 4 * (3 * i + 2 * h)) + 4 * t * h, "flops": 2.0 * t * k * 3 * h * i}


# ------------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _table(lens, page, first, g):
    """A page table for sequences of these lengths: pages from `first` on, in a random order. Returns it and the page after."""
    need = [-(-n // page) for n in lens]
    order = torch.randperm(sum(need), generator=g, device="cuda").to(torch.int32) + first
    table = torch.zeros((len(lens), max(need)), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, first + sum(need)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _starts(counts):
    at = [0]
    for n in counts:
        at.append(at[-1] + n)
    return at


def _random_cache(pages, case, g, weights):
    """A filled cache: nibbles of a roughly normal distribution, steps and bases of groups with a spread of about 4 sigma."""
    hk, s, d = case["kv_heads"], case["page"], case["dim"]
    c = {}
    for name in ("k", "v"):
        low = torch.randint(0, 256, (pages, hk, s, d // 2), generator=g, device="cuda", dtype=torch.uint8)
        c[name] = low
        step = torch.empty((pages, hk, s, d // GROUP), device="cuda").uniform_(0.15, 0.45, generator=g)
        base = -step * torch.empty_like(step).uniform_(6.5, 8.0, generator=g)
        c[name + "_scale"] = torch.stack([step, base], -1).to(torch.float16)
    c["weight"] = torch.empty((pages, hk, s), device="cuda").exponential_(generator=g) if weights else None
    return c


def _wrap(c):
    """The package's cache object over these buffers."""
    from optimized_rocwmma_samples_b200 import api
    return api.KV4Cache(k=c["k"], v=c["v"], k_scale=c["k_scale"], v_scale=c["v_scale"], weight=c["weight"])


def prepare(case, seed):
    g = _generator(seed)
    st = {"case": case}
    if case["op"] == "moe":
        t, h, i, e, k = (case[x] for x in ("tokens", "hidden", "inter", "experts", "topk"))
        x = torch.randn((t, h), generator=g, device="cuda")
        x[:, torch.randperm(h, generator=g, device="cuda")[:8]] *= 20.0  # outlier channels, as activations have
        st["x"] = x.to(_dtype(case))
        logits = torch.randn((t, e), generator=g, device="cuda") + torch.randn((1, e), generator=g, device="cuda") * 0.5
        p, ids = torch.softmax(logits, -1).sort(-1, descending=True)
        st["w"], st["ids"] = p[:, :k].contiguous(), ids[:, :k].to(torch.int32).contiguous()

        def matrix(rows, cols):
            return torch.randint(-127, 128, (e, rows, cols), generator=g, device="cuda", dtype=torch.int8)

        def uniform(lo, hi, *shape):
            return torch.empty(shape, device="cuda").uniform_(lo, hi, generator=g)

        st["smooth1"], st["smooth2"] = uniform(0.5, 2.0, e, h), uniform(0.5, 2.0, e, i)
        st["w13"], st["w2"] = matrix(2 * i, h), matrix(h, i)
        one = 1 / 73.0  # the standard deviation of the weights' integers
        st["s13"] = uniform(0.5, 1.5, e, 2 * i) * (one / math.sqrt(h))
        st["s2"] = uniform(0.5, 1.5, e, h) * (one / math.sqrt(i))
        st["out"] = torch.empty((t, h), dtype=_dtype(case), device="cuda")
        return st
    hk, d, page = case["kv_heads"], case["dim"], case["page"]
    if case["op"] == "append":
        counts = _counts(case)
        lens = [n + (37 * b) % 100 for b, n in enumerate(counts)]  # some sequences hold tokens already
        st["table"], pages = _table(lens, page, 0, g)
        st["cache"] = {
            "k": torch.zeros((pages, hk, page, d // 2), dtype=torch.uint8, device="cuda"),
            "v": torch.zeros((pages, hk, page, d // 2), dtype=torch.uint8, device="cuda"),
            "k_scale": torch.zeros((pages, hk, page, d // GROUP, 2), dtype=torch.float16, device="cuda"),
            "v_scale": torch.zeros((pages, hk, page, d // GROUP, 2), dtype=torch.float16, device="cuda"),
            "weight": None}
        total = sum(counts)
        channel = torch.empty((1, hk, d), device="cuda").uniform_(0.3, 3.0, generator=g)  # keys differ by channel
        st["k"] = (torch.randn((total, hk, d), generator=g, device="cuda") * channel).to(_dtype(case))
        st["v"] = torch.randn((total, hk, d), generator=g, device="cuda").to(_dtype(case))
        st["starts"], st["lens"] = _int32(_starts(counts)), _int32(lens)
        st["k_out"], st["v_out"] = torch.empty_like(st["k"]), torch.empty_like(st["v"])
        return st
    lens = _lengths(case)
    st["lens"] = _int32(lens)
    st["table"], pages = _table(lens, page, 0, g)
    if case["op"] == "evict":
        st["first"] = pages
        st["new_table"], pages = _table([min(n, case["budget"]) for n in lens], page, pages, g)
        st["cache"] = _random_cache(pages, case, g, True)
        for name in ("k", "v", "k_scale", "v_scale", "weight"):
            st["cache"][name][st["first"]:] = 0
        st["new_lens"] = torch.empty_like(st["lens"])
        return st
    st["cache"] = _random_cache(pages, case, g, case["weights"])
    n = case["batch"] * case["queries"]
    st["q"] = torch.randn((n, case["heads"], d), generator=g, device="cuda").to(_dtype(case))
    st["starts"] = _int32(_starts([case["queries"]] * case["batch"]))
    st["out"] = torch.empty_like(st["q"])
    return st


# ------------------------------------------------------------------------------------------------ plain forms
def _own(st):
    from optimized_rocwmma_samples_b200 import api
    case = st["case"]
    if case["op"] == "moe":
        return api.moe_layer(st["x"], st["w"], st["ids"], st["smooth1"], st["w13"], st["s13"], st["smooth2"], st["w2"],
                             st["s2"], quant_max=QMAX, out=st["out"])
    if "handle" not in st:  # a program makes this object once, with its cache
        st["handle"] = _wrap(st["cache"])
    cache = st["handle"]
    if case["op"] == "append":
        api.kv4_append(st["k"], st["v"], cache, st["table"], st["lens"], st["starts"], k_out=st["k_out"], v_out=st["v_out"])
        return st["k_out"], st["v_out"]
    if case["op"] == "attend":
        api.kv4_attention(st["q"], cache, st["table"], st["lens"], st["starts"], max_queries=case["queries"],
                          out=st["out"], accumulate_weight=case["weights"])
        return (st["out"], cache.weight) if case["weights"] else st["out"]
    api.kv4_evict(cache, st["table"], st["lens"], st["new_table"], budget=case["budget"], recent=case["recent"],
                  new_lens=st["new_lens"])
    return _evicted(st)


def _evicted(st):
    """The new lengths and the new pages' contents: bits that were copied, not numbers that were computed."""
    c, first = st["cache"], st["first"]
    return {"lens": st["new_lens"], **{name: c[name][first:] for name in ("k", "v", "k_scale", "v_scale", "weight")}}


def run(st):
    if own:
        return _own(st)
    return {"append": _append, "attend": _attend, "evict": _evict, "moe": _moe}[st["case"]["op"]](st)


def _append(st):
    c, page = st["cache"], st["case"]["page"]
    starts, lens = st["starts"].long(), st["lens"].long()
    token = torch.arange(st["k"].shape[0], device="cuda")
    b = torch.searchsorted(starts, token, right=True) - 1
    pos = lens[b] - (starts[b + 1] - starts[b]) + token - starts[b]
    at, slot = st["table"][b, pos // page].long(), pos % page
    for name in ("k", "v"):
        x = st[name].float().clamp(-65504.0, 65504.0).unflatten(-1, (-1, GROUP))
        low, high = x.amin(-1), x.amax(-1)
        step, base = ((high - low) / 15).to(torch.float16), low.to(torch.float16)
        s, z = step.double()[..., None], base.double()[..., None]
        # the quotient in 64 bits: values on the border between two steps go to the even one
        q = torch.where(s > 0, ((x.double() - z) / s).round().clamp(0, 15), 0.0)
        nibble = q.to(torch.uint8).flatten(-2)
        c[name][at, :, slot] = nibble[..., 0::2] | (nibble[..., 1::2] << 4)
        c[name + "_scale"][at, :, slot] = torch.stack([step, base], -1)
        st[name + "_out"].copy_((q * s + z).flatten(-2))
    return st["k_out"], st["v_out"]


def _values(c, name, table):
    """Keys or values of every sequence, [batch, head, position, channel], in 32 bits."""
    raw = c[name][table.long()].permute(0, 2, 1, 3, 4).flatten(2, 3)  # [batch, head, position, bytes]
    q = torch.stack([raw & 15, raw >> 4], -1).flatten(-2).float().unflatten(-1, (-1, GROUP))
    sz = c[name + "_scale"][table.long()].permute(0, 2, 1, 3, 4, 5).flatten(2, 3).float()
    return (q * sz[..., 0:1] + sz[..., 1:2]).flatten(-2)


def _seen(st):
    """[batch, query, position]: which positions a query sees."""
    case, page = st["case"], st["case"]["page"]
    position = torch.arange(st["table"].shape[1] * page, device="cuda")
    last = st["lens"].long()[:, None] - case["queries"] + torch.arange(case["queries"], device="cuda")
    return position <= last[..., None]


def _attend(st):
    case, c, page = st["case"], st["cache"], st["case"]["page"]
    b, n, hq, hk, d = (case[x] for x in ("batch", "queries", "heads", "kv_heads", "dim"))
    q = st["q"].float().view(b, n, hk, hq // hk, d).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [b, hk, group * n, d]
    seen = _seen(st)[:, None, None].expand(b, hk, hq // hk, n, -1).flatten(2, 3)
    score = (q @ _values(c, "k", st["table"]).transpose(-1, -2)) * d ** -0.5
    score = torch.where(seen, score, float("-inf"))
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = p @ _values(c, "v", st["table"])
    st["out"].copy_(o.unflatten(2, (hq // hk, n)).permute(0, 3, 1, 2, 4).reshape(b * n, hq, d))
    if not case["weights"]:
        return st["out"]
    add = p.sum(2).unflatten(-1, (-1, page)).transpose(1, 2)  # [b, page, hk, slot]
    held = torch.arange(st["table"].shape[1], device="cuda") * page < st["lens"][:, None]
    c["weight"][st["table"][held].long()] += add[held]
    return st["out"], c["weight"]


def _evict(st):
    case, c, page = st["case"], st["cache"], st["case"]["page"]
    budget, recent, hk = case["budget"], case["recent"], case["kv_heads"]
    lens = st["lens"].long()
    weight = c["weight"][st["table"].long()].transpose(1, 2).flatten(2)  # [b, hk, position]
    position = torch.arange(weight.shape[-1], device="cuda")
    outside, newest = position >= lens[:, None], position >= lens[:, None] - recent
    key = torch.where(newest[:, None], float("inf"), weight)
    key = torch.where(outside[:, None], float("-inf"), key)
    kept = key.sort(dim=-1, descending=True, stable=True).indices[..., :budget]
    new = lens.clamp(max=budget)
    used = torch.arange(budget, device="cuda") < new[:, None]
    kept = torch.where(used[:, None], kept, weight.shape[-1]).sort(-1).values  # in order, what is not used last
    b, h, j = used[:, None].expand(-1, hk, -1).nonzero(as_tuple=True)
    pos = kept[b, h, j]
    src, dst = st["table"][b, pos // page].long(), st["new_table"][b, j // page].long()
    for name in ("k", "v", "k_scale", "v_scale", "weight"):
        c[name][dst, h, j % page] = c[name][src, h, pos % page]
    st["new_lens"].copy_(new)
    return _evicted(st)


def _quantise(x):
    scale = x.abs().amax(-1, keepdim=True) / QMAX
    inv = torch.where(scale > 0, 1 / scale, 0.0)
    return (x * inv).round().clamp(-QMAX, QMAX), scale


def _moe(st):
    # every expert takes every token; the router's weights, zero where it did not choose, pick the sum
    e, t = st["case"]["experts"], st["case"]["tokens"]
    xq, scale = _quantise(st["x"].float() * st["smooth1"][:, None])
    gate, up = ((xq @ st["w13"].float().transpose(1, 2)) * (scale * st["s13"][:, None])).chunk(2, -1)
    hq, scale = _quantise(gate / (1 + torch.exp(-gate)) * up * st["smooth2"][:, None])
    down = (hq @ st["w2"].float().transpose(1, 2)) * (scale * st["s2"][:, None])
    chosen = torch.zeros((t, e), device="cuda").scatter_add_(1, st["ids"].long(), st["w"])
    st["out"].copy_((chosen.t()[..., None] * down).sum(0))
    return st["out"]


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "append":
        return tuple(_exact_append(st[name]) for name in ("k", "v"))
    if case["op"] == "attend":
        return _exact_attend(st)
    if case["op"] == "moe":
        return _exact_moe(st)
    return _exact_evict(st)


def _exact_append(x):
    y = x.double().clamp(-65504, 65504).reshape(*x.shape[:-1], -1, GROUP)
    z = y.min(-1, keepdim=True).values.half().double()
    s = ((y.max(-1, keepdim=True).values - y.min(-1, keepdim=True).values) / 15).half().double()
    q = torch.clamp(torch.round((y - z) / torch.where(s > 0, s, 1.0)), 0, 15)
    return (torch.where(s > 0, q, 0.0) * s + z).reshape(x.shape)


def _exact_attend(st):
    case, c = st["case"], st["cache"]
    n, hq, hk, d, page = (case[x] for x in ("queries", "heads", "kv_heads", "dim", "page"))
    out = torch.zeros((case["batch"] * n, hq, d), dtype=torch.float64, device="cuda")
    weight = c["weight"].double() if case["weights"] else None
    for b, length in enumerate(_lengths(case)):
        pages = st["table"][b, : -(-length // page)].long()
        kv = []
        for name in ("k", "v"):
            raw = c[name][pages].transpose(0, 1).reshape(hk, -1, d // 2)[:, :length]
            q = torch.empty((hk, length, d), dtype=torch.float64, device="cuda")
            q[..., 0::2], q[..., 1::2] = raw % 16, raw // 16
            sz = c[name + "_scale"][pages].transpose(0, 1).reshape(hk, -1, d // GROUP, 2)[:, :length].double()
            kv.append(q * sz[..., 0].repeat_interleave(GROUP, -1) + sz[..., 1].repeat_interleave(GROUP, -1))
        for i in range(n):
            see = length - n + i + 1
            q = st["q"][b * n + i].double().reshape(hk, hq // hk, d)
            p = torch.softmax(torch.einsum("hgd,htd->hgt", q, kv[0][:, :see]) / math.sqrt(d), -1)
            out[b * n + i] = torch.einsum("hgt,htd->hgd", p, kv[1][:, :see]).reshape(hq, d)
            if weight is not None:
                rows = torch.arange(see, device="cuda")
                weight[pages[rows // page], :, rows % page] += p.sum(1).t()
    return out if weight is None else (out, weight)


def _exact_evict(st):
    case, c = st["case"], st["cache"]
    page, budget, recent = (case[x] for x in ("page", "budget", "recent"))
    for b, length in enumerate(_lengths(case)):
        pages = st["table"][b, : -(-length // page)].long()
        for h in range(case["kv_heads"]):
            old = c["weight"][pages, h].reshape(-1)[: max(0, length - recent)].double()
            most = min(length, budget) - min(length, recent)
            mark = torch.zeros(length, dtype=torch.bool, device="cuda")
            mark[torch.argsort(-old, stable=True)[:most]] = True
            mark[max(0, length - recent):] = True
            src, dst = mark.nonzero().flatten(), torch.arange(min(length, budget), device="cuda")
            to = st["new_table"][b].long()[dst // page]
            for name in ("k_scale", "v_scale", "weight"):
                c[name][to, h, dst % page] = c[name][pages[src // page], h, src % page]
    return {name: (None if name in ("lens", "k", "v") else x.double()) for name, x in _evicted(st).items()}


def _exact_moe(st):
    out = torch.zeros(st["x"].shape, dtype=torch.float64, device="cuda")
    for e in range(st["case"]["experts"]):
        token, slot = (st["ids"] == e).nonzero(as_tuple=True)
        if not len(token):
            continue
        x = st["x"][token].double() * st["smooth1"][e].double()
        step = x.abs().max(1, keepdim=True).values / QMAX
        a = torch.round(x / step) @ st["w13"][e].double().T * step * st["s13"][e].double()
        gate, up = a[:, : a.shape[1] // 2], a[:, a.shape[1] // 2:]
        h = gate * torch.sigmoid(gate) * up * st["smooth2"][e].double()
        step = h.abs().max(1, keepdim=True).values / QMAX
        y = torch.round(h / step) @ st["w2"][e].double().T * step * st["s2"][e].double()
        out.index_add_(0, token, y * st["w"][token, slot].double()[:, None])
    return out
