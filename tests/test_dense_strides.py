"""Rows further apart than linear and gated_linear address: copied by the differentiable functions,
refused with the limit's name by the others."""
import pytest
import torch

import hipgemm_amd as hg
import hipgemm_amd.dense as dense
import hipgemm_amd.torch_dense as td

BF = torch.bfloat16


def test_limit_is_named():
    x = torch.empty((1 << 21) + 72, dtype=BF)
    assert dense._operand(x.as_strided((2, 64), (1 << 21, 1)), "x", BF, -1)[0] == 1 << 21
    with pytest.raises(hg.HipGemmError, match="2097152"):
        dense._operand(x.as_strided((2, 64), ((1 << 21) + 8, 1)), "x", BF, -1)
    # one row has no stride
    assert dense._operand(x.as_strided((1, 64), ((1 << 21) + 8, 1)), "x", BF, -1)[0] == 64


def test_far_rows_are_copied():
    x = torch.zeros(1 << 22, dtype=BF)
    for stride, far in ((1 << 21, False), ((1 << 21) + 8, True)):
        t = td._rows(x.as_strided((2, 64), (stride, 1)))
        assert (t.stride(0) == 64) == far and (t.data_ptr() != x.data_ptr()) == far


@pytest.mark.gpu
@pytest.mark.parametrize("gated", (False, True), ids=("linear", "gated"))
def test_last_tokens(gpu, gated):
    """The last token of each of three sequences of 1024 x 4096, forward and backward."""
    g = torch.Generator(device="cuda").manual_seed(0)
    hidden = torch.randn(3, 1024, 4096, generator=g, device="cuda").to(BF)
    w = torch.randn(48, 4096, generator=g, device="cuda").div_(64).to(BF).requires_grad_()
    call = td.gated_linear if gated else (lambda x, w: td.linear(x, w, activation="silu"))
    far = hidden[:, -1]
    assert far.stride(0) > 1 << 21
    near = far.clone().requires_grad_()
    far = far.detach().requires_grad_()
    assert far.stride(0) > 1 << 21
    results = []
    for x in (far, near):
        with torch.no_grad():
            plain = call(x, w)
        y = call(x, w)
        assert torch.equal(y, plain)
        results.append((y, *torch.autograd.grad(y, (x, w), torch.ones_like(y))))
    assert all(torch.equal(a, b) for a, b in zip(*results))
    # a weight of far rows
    wide = torch.zeros(48, (1 << 21) + 8, device="cuda", dtype=BF)[:, :4096]
    wide.copy_(w.detach())
    assert torch.equal(call(near, wide), results[1][0])
