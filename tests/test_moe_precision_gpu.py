"""moe_experts' float32 results have float32's precision: the rms error is no larger
than that of the same layer in plain fp32 tensor operations, times 3 (sums in another
order), pair by pair and grouped."""
import pytest
import torch

import hipgemm_amd as hg
import w4util as u
from test_moe_experts_gpu import make, plain

pytestmark = pytest.mark.gpu


def plain32(a, fmt, group):
    x = a["x"].float()
    y = torch.zeros_like(x)
    for e in range(a["w13"].shape[0]):
        t, j = (a["ids"] == e).nonzero(as_tuple=True)
        z13, z2 = ((a[n][e] if a[n] is not None else None) for n in ("zeros13", "zeros2"))
        w13 = u.weights64(a["w13"][e], a["scales13"][e], fmt, group, z13).float()
        w2 = u.weights64(a["w2"][e], a["scales2"][e], fmt, group, z2).float()
        gate, up = (x[t] @ w13.t()).chunk(2, 1)
        h = gate * torch.sigmoid(gate) * up * a["weights"][t, j][:, None]
        y.index_add_(0, t, h @ w2.t())
    return y


@pytest.mark.parametrize("fmt,zeros", [("e4m3", False), ("int4", False), ("int4", True),
                                       ("fp4", False)])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("grouped,T,E,k,D,F", [(False, 3, 8, 2, 1056, 608), (True, 40, 3, 2, 1056, 608),
                                               (True, 64, 5, 4, 416, 1312), (False, 1, 4, 2, 2048, 2048),
                                               (True, 14, 16, 2, 2080, 2336)])
def test_float32_results(gpu, grouped, T, E, k, D, F, dtype, fmt, zeros):
    assert bool(hg.moe_select(T, k, E, D, F, fmt, torch.float32)) == grouped
    a = make(T, T, E, k, D, F, fmt, zeros=zeros, dtype=dtype)
    want, slack = plain(a, fmt, 128, "silu")
    y = hg.moe_experts(**a, format=fmt, out_dtype=torch.float32)
    u.agree(y, want, slack)
    err = (y - want).pow(2).mean().sqrt()
    ref = (plain32(a, fmt, 128) - want).pow(2).mean().sqrt()
    assert err <= 3 * ref, (err / ref).item()
