"""moe_route's sigmoids renormalised where all of them are next to nothing: the
definition's ratios stay ordinary numbers, p_j / sum p = r_j / sum r with
r_j = exp(v_j - max) / (1 + exp(v_j)).

Tolerance: as in test_moe_route_gpu.py, an argument rounded once (|v - max| 2^-24
of the result), 16 further roundings, and the sum's: k terms r with arguments of
their own, r |v - max| <= 1 / e each; the smallest normal number for what
underflows."""
import pytest
import torch

pytestmark = pytest.mark.gpu

LOWEST = {t: torch.finfo(t).min for t in (torch.float32, torch.bfloat16, torch.float16)}


@pytest.fixture()
def hg(gpu):
    import hipgemm_amd
    return hipgemm_amd


def rows(dtype):
    low = LOWEST[dtype]
    return torch.tensor([
        [-86, -87, -87.5, -88, -90, -89],          # the last normal sigmoids
        [-95, -100, -96, -103, -104, -110],        # subnormal, then 0
        [-200, -200.5, -201, -230, -400, -300],
        [-60000, -60000, -61000, low, low, -60000],
        [low, low, low, low, low, low],
        [low, -1e4, low, low, -1e4, low],          # two, and masks of the lowest value
        [-0.5, -95, -200, low, -3, -1],            # one ordinary number among them
        [0.25, -95, -200, low, -3, 0],
        [float("-inf"), -100, -101, float("-inf"), float("-inf"), -102],
    ], dtype=torch.float64).to(dtype)


@pytest.mark.parametrize("T", [9, 4500])
@pytest.mark.parametrize("k", [1, 4, 6])
@pytest.mark.parametrize("dtype", list(LOWEST), ids=str)
def test_sigmoids_renormalised_far_below_zero(hg, dtype, k, T):
    l = rows(dtype).repeat(-(-T // 9), 1)[:T].cuda()
    w, ids = hg.moe_route(l, k, scoring="sigmoid", renormalize=True, scale=2.5)
    v, order = l.double().sort(dim=1, descending=True, stable=True)
    v, order = v[:, :k], order[:, :k]
    chosen = v > float("-inf")
    assert torch.equal(ids, torch.where(chosen, order, -1).int())
    away = torch.where(chosen, v[:, :1] - v, 0.0)
    r = torch.where(chosen, torch.exp(-away) / (1 + torch.exp(v)), 0.0)
    want = r / r.sum(1, keepdim=True) * 2.5
    tol = want * (away + 16 + k) * 2.0 ** -24 + 2.0 ** -126
    assert bool(((w.double() - want).abs() <= tol).all()), w[:9]
