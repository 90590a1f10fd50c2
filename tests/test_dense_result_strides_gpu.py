"""Results whose rows lie further apart than an operand's may: as hg.linear(..., out=cache[:, -1])."""
import ctypes

import pytest
import torch

import hipgemm_amd as hg
from denseutil import backward64, check, gated64, linear64

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
FAR = (1 << 21) + 8


def far(rows, cols, dtype=BF):
    """(the storage, rows x cols of it)."""
    full = torch.full((rows, FAR), 7.0, device="cuda", dtype=dtype)
    return full, full[:, 3:3 + cols]


@pytest.mark.parametrize("M", (2, 70))  # a few rows; tiles
@pytest.mark.parametrize("gated", (False, True), ids=("linear", "gated"))
def test_out(gpu, M, gated):
    N, K = 40, 72
    g = torch.Generator(device="cuda").manual_seed(M)
    x = torch.randn(M, K, generator=g, device="cuda").to(BF)
    w = torch.randn(2 * N if gated else N, K, generator=g, device="cuda").div_(8).to(BF)
    full, out = far(M, N)
    if gated:
        _, _, y, ey = gated64(x, w, None, "silu", BF)
        hg.gated_linear(x, w, out=out)
    else:
        res = torch.randn(M, N, generator=g, device="cuda").to(BF)
        out.copy_(res)  # residual and result, in place
        _, _, y, ey = linear64(x, w, None, "silu", res, BF)
        hg.linear(x, w, activation="silu", residual=out, out=out)
    check("y", out, y, ey)
    out.fill_(7.0)
    assert bool((full == 7.0).all())


@pytest.mark.parametrize("M,N,K", ((70, 40, 72), (9, 24, 136)))
def test_descriptors(gpu, M, N, K):
    """z, dx and dw of the C entry points."""
    g = torch.Generator(device="cuda").manual_seed(M)
    x = torch.randn(M, K, generator=g, device="cuda").to(BF)
    w = torch.randn(N, K, generator=g, device="cuda").div_(8).to(BF)
    dy = torch.randn(M, N, generator=g, device="cuda").to(BF)
    y = torch.empty(M, N, device="cuda", dtype=BF)
    silu = hg.ACTIVATIONS["silu"]
    store_z, z = far(M, N, F32)
    d = hg.LinearDesc(size=ctypes.sizeof(hg.LinearDesc), x=x.data_ptr(), weight=w.data_ptr(),
                      y=y.data_ptr(), pre=z.data_ptr(), ldx=K, ldw=K, ldy=N, ldp=FAR, M=M, N=N,
                      K=K, type=1, out_dtype=0, pre_dtype=2, activation=silu)
    need = hg.linear_workspace_size(d)
    memory = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    d.workspace, d.workspace_bytes = memory.data_ptr(), need
    assert hg.linear_raw(d) == 0
    want, bound, _, _ = linear64(x, w, None, "silu", None, BF, F32)
    check("z", z, want, bound)
    store_x, dx = far(M, K)
    store_w, dw = far(N, K)
    b = hg.LinearGradDesc(size=ctypes.sizeof(hg.LinearGradDesc), dy=dy.data_ptr(),
                          x=x.data_ptr(), weight=w.data_ptr(), pre=z.data_ptr(),
                          dx=dx.data_ptr(), dw=dw.data_ptr(), lddy=N, ldx=K, ldw=K, ldp=FAR,
                          lddx=FAR, lddw=FAR, M=M, N=N, K=K, type=1, dy_type=1, pre_type=0,
                          dx_dtype=0, dw_dtype=0, activation=silu)
    need = hg.linear_backward_workspace_size(b)
    memory = torch.empty(need, dtype=torch.uint8, device="cuda")
    b.workspace, b.workspace_bytes = memory.data_ptr(), need
    assert hg.linear_backward_raw(b) == 0
    wants = backward64(dy, x, w, z, "silu", False, BF)
    check("dx", dx, *wants["dx"])
    check("dw", dw, *wants["dw"])
    for full, part in ((store_z, z), (store_x, dx), (store_w, dw)):
        part.fill_(7.0)
        assert bool((full == 7.0).all())
