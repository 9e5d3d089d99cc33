"""NaN and infinities in the mixture-of-experts layer: they reach the whole output of their token, and no other's."""
import pytest
import torch

from optimized_rocwmma_samples_b200 import api
from test_gpu_moe_layer import DEV, make

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")


def run(a):
    out = api.moe_layer(**a)
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,H,I,E,K", [(5, 144, 80, 4, 2), (40, 2064, 48, 3, 1), (3, 64, 4112, 8, 8)])
def test_in_tokens(cuda_device, T, H, I, E, K, dtype):
    a = make(T, H, I, E, K, dtype, seed=T)
    clean = run(a)
    a["x"][0, 0], a["x"][1, H - 1], a["x"][2, H // 2] = NAN, INF, -INF
    out = run(a)
    assert out[:3].isnan().all()
    assert torch.equal(out[3:], clean[3:])


@pytest.mark.parametrize("bad", [NAN, INF, -INF])
@pytest.mark.parametrize("name", ["smooth1", "s13", "smooth2"])
def test_in_an_expert(cuda_device, name, bad):
    """A bad factor of one expert reaches the tokens that chose it."""
    T, H, I, E, K = 12, 96, 64, 5, 2
    a = make(T, H, I, E, K, torch.float16, seed=2)
    clean = run(a)
    a["w13"][3, 7].fill_(1)  # so that the bad step meets a sum that is not 0
    a["w13"][3, I + 7].fill_(1)
    a[name][3, 7] = bad
    out = run(a)
    hit = (a["topk_ids"] == 3).any(1)
    assert hit.any() and not hit.all()
    assert out[hit].isnan().all() and torch.equal(out[~hit], clean[~hit])


def test_in_a_token_without_an_expert(cuda_device):
    """Nothing of a token is read by a route that has no expert."""
    ids = torch.tensor([[-1], [1]], dtype=torch.int32, device=DEV)
    a = make(2, 64, 48, 2, 1, torch.bfloat16, ids=ids)
    a["x"][0] = NAN
    out = run(a)
    assert torch.all(out[0] == 0) and torch.isfinite(out[1]).all()


def test_sums_that_leave_fp32(cuda_device):
    """h past fp32's range is an infinity, and the token NaN; the definition has no finite value in its type either."""
    a = make(3, 64, 48, 2, 1, torch.bfloat16, seed=5)
    clean = run(a)
    a["x"][1] *= 1e25
    out = run(a)
    assert out[1].isnan().all() and torch.equal(out[[0, 2]], clean[[0, 2]])
