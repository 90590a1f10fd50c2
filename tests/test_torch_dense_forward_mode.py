"""linear and gated_linear have no forward-mode derivative: a tangent is refused, never taken
for zeros (CPU, with the device calls replaced by host ones)."""
import pytest
import torch
from torch.autograd import forward_ad

import hipgemm_amd as hg
import hipgemm_amd.torch_dense as td

BF = torch.bfloat16


@pytest.fixture
def host(monkeypatch):
    """The device calls in tensor operations."""
    def linear(x, weight, bias=None, activation=None, residual=None, out_dtype=None,
               save_pre=False):
        z = x.float() @ weight.float().t()
        z = z if bias is None else z + bias.float()
        y = torch.nn.functional.silu(z) if activation == "silu" else z
        y = (y if residual is None else y + residual.float()).to(out_dtype or x.dtype)
        return (y, z) if save_pre else y

    def gated(x, weight, bias=None, activation="silu", out_dtype=None, save_pre=False):
        z = x.float() @ weight.float().t()
        g, u = z.chunk(2, 1)
        y = (torch.nn.functional.silu(g) * u).to(out_dtype or x.dtype)
        return (y, z) if save_pre else y

    def back(dy, x, weight, pre, **kw):
        return torch.zeros_like(x), torch.zeros_like(weight), None

    monkeypatch.setattr(td.dense, "linear", linear)
    monkeypatch.setattr(td.dense, "gated_linear", gated)
    monkeypatch.setattr(td.dense, "linear_backward", back)
    g = torch.Generator().manual_seed(0)
    return [torch.randn(s, generator=g).to(BF) for s in ((5, 64), (48, 64), (48,), (5, 48))]


CALLS = {
    "linear": lambda x, w, b, r: td.linear(x, w, b, "silu", r),
    "leading": lambda x, w, b, r: td.linear(x if x.dim() == 3 else x[None], w, b, "silu",
                                            r if r.dim() == 3 else r[None]),
    "gated": lambda x, w, b, r: td.gated_linear(x, w, b),
    "op": lambda x, w, b, r: torch.ops.hipgemm.linear(x, w, b, "silu", r),
    "gated op": lambda x, w, b, r: torch.ops.hipgemm.gated_linear(x, w, b),
}


@pytest.mark.parametrize("which", range(4), ids=("x", "weight", "bias", "residual"))
@pytest.mark.parametrize("name", CALLS)
def test_tangents_are_refused(host, name, which):
    if which == 3 and "gated" in name:
        pytest.skip("no residual")
    call = CALLS[name]

    def of(t):
        return call(*host[:which], t, *host[which + 1:])

    with forward_ad.dual_level(), pytest.raises(hg.HipGemmError, match="forward-mode"):
        of(forward_ad.make_dual(host[which], host[which]))
    with pytest.raises(hg.HipGemmError, match="forward-mode"):
        torch.func.jvp(of, (host[which],), (host[which],))
    with pytest.raises(hg.HipGemmError, match="forward-mode"):
        torch.func.jacfwd(of)(host[which])


@pytest.mark.parametrize("name", ("linear", "leading", "gated"))
def test_constants_beside_tangents(host, name):
    """Forward mode that these inputs take no part in."""
    if name == "leading":
        host[0], host[3] = host[0][None], host[3][None]
    want = CALLS[name](*host)
    with forward_ad.dual_level():
        t = forward_ad.make_dual(host[0], host[0])
        y = CALLS[name](*host)
        assert torch.equal(y, want)
        assert forward_ad.unpack_dual(y.sum() + t).tangent.equal(host[0])
    y, tangent = torch.func.jvp(lambda a: CALLS[name](*host).sum() + a, (host[0],), (host[0],))
    assert torch.equal(y, want.sum() + host[0]) and torch.equal(tangent, host[0])


def test_tangent_of_the_gradient(host):
    """A gradient that carries a tangent into the backward pass."""
    x = host[0].clone().requires_grad_()
    y = td.linear(x, host[1], host[2], "silu", host[3])
    with forward_ad.dual_level():
        dy = forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y))
        with pytest.raises(hg.HipGemmError, match="forward-mode"):
            torch.autograd.grad(y, x, dy, retain_graph=True)
        assert torch.autograd.grad(y, x, torch.ones_like(y))[0].shape == x.shape
