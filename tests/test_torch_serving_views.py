"""The serving modules and operators on views: whatever strides and alignment a
Linear's input may have (GPU), and inputs of another width, which are refused."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import hipgemm_amd as hg
import hipgemm_amd.torch_serving as ts


def test_another_width_is_refused():
    """Twice the features are not twice the rows."""
    lin = ts.W4Linear.from_linear(torch.nn.Linear(64, 40), group_size=32)
    with FakeTensorMode(allow_non_fake_inputs=True) as mode, torch.no_grad():
        assert tuple(lin(mode.from_tensor(torch.zeros(4, 64, dtype=torch.bfloat16))).shape) == (4, 40)
        for shape in ((4, 128), (2, 32), (128,), (2, 3, 32)):
            with pytest.raises(hg.HipGemmError):
                lin(mode.from_tensor(torch.zeros(shape, dtype=torch.bfloat16)))


def views(rows, width):
    """Tensors of (rows, width) or (2, rows / 2, width) whose rows are not as the
    kernels take them."""
    g = torch.Generator(device="cuda").manual_seed(rows)

    def wide(*shape):
        return torch.randn(shape, generator=g, device="cuda").bfloat16()

    yield wide(width, rows).t()
    yield wide(rows, width + 4)[:, 4:]
    yield wide(rows, width + 3)[:, :width]
    yield wide(rows * width + 2)[2:].view(rows, width)
    yield wide(rows, 2 * width)[:, ::2]
    yield wide(1, width).expand(rows, width)
    yield wide(rows // 2, 2, width + 1).transpose(0, 1)[..., 1:]
    yield wide(width, rows // 2, 2).permute(2, 1, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [2, 6, 40])
def test_linear_takes_views(gpu, rows):
    lin = ts.W4Linear.from_linear(torch.nn.Linear(160, 72, device="cuda"), "int4", 32)
    with torch.no_grad():
        for x in views(rows, 160):
            want = lin(x.contiguous().clone())
            assert torch.equal(lin(x), want)
            x2 = x if x.dim() == 2 else x.flatten(0, 1)
            assert torch.equal(torch.ops.hipgemm.w4_gemm(
                x2, lin.weight, lin.scales, group_size=32, bias=lin.bias), want.reshape(rows, 72))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["e4m3", "int4"])
def test_moe_takes_views(gpu, fmt):
    g = torch.Generator(device="cuda").manual_seed(5)

    def rand(*s):
        return torch.randn(s, generator=g, device="cuda") * s[-1] ** -0.5

    moe = ts.MoE.from_weights(rand(8, 96).bfloat16(), rand(8, 128, 96), rand(8, 96, 64), 3, fmt, 32)
    with torch.no_grad():
        for x in views(6, 96):
            x0 = x.contiguous().clone()
            assert torch.equal(moe(x), moe(x0))
            if x.dim() == 2:
                p, ids = hg.moe_route(torch.nn.functional.linear(x0, moe.gate), 3)
                args = (ids, p, moe.w13, moe.scales13, moe.w2, moe.scales2, None, None, fmt, 32)
                assert torch.equal(torch.ops.hipgemm.moe_experts(x, *args), moe(x0))
