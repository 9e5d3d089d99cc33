"""The whole mixture-of-experts layer for a few tokens against its formulas in
64 bits.  Quantised activations are integers, so the tolerance counts which of
them lie on a border between two integers, by the computed values."""
import numpy as np
import pytest
import torch

import oracle as O
from optimized_rocwmma_samples_b200 import api, synth

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def make(T, H, I, E, K, dtype, seed=0, ids=None):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)

    def uniform(lo, hi, *shape):
        return torch.empty(shape, device=DEV).uniform_(lo, hi, generator=g)

    x = torch.randn((T, H), generator=g, device=DEV)
    x[:, ::17] *= 10
    logits = torch.randn((T, E), generator=g, device=DEV)
    w, order = torch.softmax(logits, -1).sort(dim=-1, descending=True)
    if ids is None:
        ids = order[:, :K].to(torch.int32).contiguous()
        w = w[:, :K].contiguous()
    else:
        w = uniform(0.1, 1.0, T, K)
    return dict(x=x.to(dtype), topk_weights=w, topk_ids=ids, smooth1=uniform(0.5, 2.0, E, H),
                w13=torch.randint(-127, 128, (E, 2 * I, H), generator=g, device=DEV, dtype=torch.int8),
                s13=uniform(0.5, 1.5, E, 2 * I) / (73.0 * H ** 0.5), smooth2=uniform(0.5, 2.0, E, I),
                w2=torch.randint(-127, 128, (E, H, I), generator=g, device=DEV, dtype=torch.int8),
                s2=uniform(0.5, 1.5, E, H) / (73.0 * I ** 0.5))


def reference(a, qmax=127.0):
    """(out, tolerance) in 64 bits.

    xq and rs1 follow smoothquant's fp32 rule bit for bit.  gate and up are then off by 3 fp32 roundings (2^-22
    of each), h by those, the exponential's argument (|gate| 2^-22), its evaluation and four more roundings: r =
    (8 + |gate|) 2^-22 of h.  h / rs2 is at most qmax, so only integers whose quotient lies within 2 qmax r + 2^-16 of
    a border can differ, by one; rs2 itself is off by r; the sums after that are exact integers and 4 + topk roundings."""
    x, ids = a["x"], a["topk_ids"]
    T, H = x.shape
    out = torch.zeros((T, H), dtype=torch.float64, device=DEV)
    tol = torch.zeros_like(out)
    I = a["w2"].shape[2]
    for t in range(T):
        for k in range(ids.shape[1]):
            e = int(ids[t, k])
            if not 0 <= e < a["w13"].shape[0]:
                continue
            xs = x[t].float() * a["smooth1"][e]
            rs = xs.abs().max() / torch.tensor(qmax, device=DEV)
            inv = 1 / rs if rs > 0 else torch.zeros_like(rs)
            xq = (xs * inv).round().clamp(-qmax, qmax).double()
            gu = (a["w13"][e].double() @ xq) * (rs.double() * a["s13"][e].double())
            gate, up = gu[:I], gu[I:]
            h = gate * torch.sigmoid(gate) * up * a["smooth2"][e].double()
            r = (8 + gate.abs()) * 2.0 ** -22
            top = h.abs().argmax()
            rs2 = h.abs()[top] / qmax
            rr = r[top]
            y = h / rs2 if rs2 > 0 else torch.zeros_like(h)
            hq = y.round().clamp(-qmax, qmax)
            frac = (y.abs() - y.abs().floor() - 0.5).abs()
            near = (frac <= 2 * qmax * (r + rr) + 2.0 ** -16).double()
            w2, s2 = a["w2"][e].double(), a["s2"][e].double()
            d = (w2 @ hq) * (rs2 * s2)
            err = (w2.abs() @ near) * rs2 * s2
            wt = a["topk_weights"][t, k].double().abs()
            out[t] += a["topk_weights"][t, k].double() * d
            tol[t] += wt * (err * (1 + 2.0 ** -10) + d.abs() * (rr + (4 + ids.shape[1]) * 2.0 ** -23))
    half = torch.finfo(x.dtype).eps / 2
    return out, tol + half * (out.abs() + tol) + 2.0 ** -25 + out.abs().amax() * 2.0 ** -22


def check(a, **kw):
    got = api.moe_layer(**a, **kw)
    torch.cuda.synchronize()
    want, tol = reference(a, kw.get("quant_max", 127.0))
    # sums past the type's largest value are infinite (fp16: from 65520 on, half a step above 65504)
    info = torch.finfo(got.dtype)
    edge = info.max * (1 + info.eps / 4)
    fits, over = want.abs() + tol < info.max, want.abs() - tol > edge
    assert torch.isfinite(got[fits]).all() and torch.equal(got[over].double(), want[over].sign() * float("inf"))
    err = torch.where(fits, (got.double() - want).abs(), 0.0)
    assert torch.all(err <= tol), f"err {err.max().item()}, over by {(err - tol).max().item()}"
    return got


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,H,I,E,K", [(1, 256, 512, 8, 2), (3, 1024, 704, 16, 4), (1, 16, 16, 1, 1), (7, 144, 80, 3, 3),
                                       (16, 512, 1456, 4, 2), (33, 272, 336, 64, 8), (64, 128, 256, 2, 1),
                                       (64, 96, 208, 128, 8), (2, 4096, 2048, 4, 2), (5, 8192, 48, 2, 2),
                                       (4, 64, 14336, 2, 1), (200, 64, 64, 5, 2)])
def test_moe_layer(cuda_device, T, H, I, E, K, dtype):
    check(make(T, H, I, E, K, dtype, seed=T + H))


@pytest.mark.parametrize("T,H,I,E,K", [(1, 16384, 32, 2, 2), (20, 16384, 16, 2, 1), (3, 32, 4112, 2, 2), (17, 80, 8208, 3, 2),
                                       (512, 48, 32, 1024, 8), (9, 1040, 12400, 2, 1), (40, 8192, 144, 2, 2)])
def test_moe_layer_far_sizes(cuda_device, T, H, I, E, K):
    """The widest rows, several slices of the inner dimension with ragged ends, many experts, all 4096 routes."""
    check(make(T, H, I, E, K, torch.bfloat16, seed=T + I))


def test_all_tokens_to_one_expert(cuda_device):
    ids = torch.full((50, 1), 5, dtype=torch.int32, device=DEV)
    check(make(50, 320, 336, 7, 1, torch.bfloat16, ids=ids))


def test_ids_outside_and_repeated(cuda_device):
    """Ids outside [0, experts) add nothing, an expert named twice adds twice, a token without any expert gives 0."""
    ids = torch.tensor([[0, 0, 3], [-1, 2, 4], [7, -5, 2 ** 31 - 1], [1, 1, 1]], dtype=torch.int32, device=DEV)
    got = check(make(4, 128, 192, 4, 3, torch.float16, ids=ids))
    assert torch.all(got[2] == 0)
    none = make(3, 64, 64, 2, 1, torch.float16, ids=torch.full((3, 1), -1, dtype=torch.int32, device=DEV))
    assert torch.all(api.moe_layer(**none) == 0)


def test_zero_and_wide_rows(cuda_device):
    a = make(6, 256, 128, 4, 2, torch.float16, seed=3)
    a["x"][0] = 0
    a["x"][1] *= 1000
    a["x"][2] *= 1e-4
    a["x"][3, 1:] = 0
    check(a)
    check(a, quant_max=31.5)


def test_row_pitch_and_given_output(cuda_device):
    a = make(9, 160, 96, 3, 2, torch.bfloat16, seed=4)
    wide = torch.randn((9, 200), device=DEV).bfloat16()
    wide[:, 40:] = a["x"]
    a["x"] = wide[:, 40:]
    out = torch.empty((9, 160), dtype=torch.bfloat16, device=DEV)
    assert check(a, out=out) is out


def test_against_the_operators_for_prompts(cuda_device):
    """The first half equals smoothquant, grouping and the grouped GEMM of the prompt path: with w2 the identity and
    integer-sized steps both give the same h up to its own quantisation (half a step) and the output's rounding."""
    T, H, I, E, K = 12, 256, 256, 4, 2
    a = make(T, H, I, E, K, torch.float16, seed=9)
    count, start, _, perm = api.moe_sorting(a["topk_ids"], E, 16)
    q, rs = api.moe_smoothquant(a["x"], a["smooth1"], a["topk_ids"], row_perm=perm, out_rows=int(start[-1]))
    acc = api.gemm_grouped(q, a["w13"], start, count, rs, a["s13"].reshape(-1), out_dtype=torch.int32)
    torch.cuda.synchronize()
    a["w2"] = torch.eye(I, H, device=DEV).to(torch.int8).expand(E, I, H).contiguous()
    a["s2"] = torch.ones((E, H), device=DEV)
    got = api.moe_layer(**a).double()
    want, tol = torch.zeros((T, H), dtype=torch.float64, device=DEV), torch.zeros((T, 1), dtype=torch.float64, device=DEV)
    for t in range(T):
        for k in range(K):
            e, row = int(a["topk_ids"][t, k]), int(perm[t * K + k])
            gu = acc[row].double() * (rs[row].double() * a["s13"][e].double())
            h = gu[:I] * torch.sigmoid(gu[:I]) * gu[I:] * a["smooth2"][e].double()
            want[t] += a["topk_weights"][t, k].double() * h
            tol[t] += a["topk_weights"][t, k].double() * h.abs().max() / 127 * 0.501
    assert torch.all((got - want).abs() <= tol + want.abs() * 2.0 ** -10)


def test_router_to_layer(cuda_device):
    """Logits through the router and the layer, as a decode step makes them; captured, and replayed with new inputs."""
    T, H, I, E, K = 16, 512, 384, 8, 2
    a = make(T, H, I, E, K, torch.float16, seed=6)
    logits = torch.randn((T, E), device=DEV).half()
    w, ids = torch.zeros((T, K), device=DEV), torch.zeros((T, K), dtype=torch.int32, device=DEV)
    out = torch.empty_like(a["x"])

    def step():
        api.topk_softmax(logits, K, w, ids)
        api.moe_layer(**{**a, "topk_weights": w, "topk_ids": ids}, out=out)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    logits.copy_(torch.randn((T, E), device=DEV))
    a["x"].copy_(torch.randn((T, H), device=DEV))
    graph.replay()
    torch.cuda.synchronize()
    w0, i0 = O.topk_softmax(logits.cpu().numpy(), K)
    assert np.array_equal(ids.cpu().numpy(), i0) and np.array_equal(w.cpu().numpy(), w0)
    want, tol = reference({**a, "topk_weights": w, "topk_ids": ids})
    assert torch.all((out.double() - want).abs() <= tol)


def test_two_streams_and_repeat(cuda_device):
    """Calls that overlap on two streams, and the same call again: the same bits."""
    a, b = make(8, 512, 512, 8, 2, torch.float16, seed=7), make(5, 256, 768, 4, 2, torch.bfloat16, seed=8)
    first, second = check(a), check(b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = [(api.moe_layer(**a), api.moe_layer(**b, stream=side)) for _ in range(5)]
    torch.cuda.synchronize()
    for x, y in outs:
        assert torch.equal(x, first) and torch.equal(y, second)
