"""Float32 gradients have float32's precision: dz counts with 24 bits, not with the operands'.

Bounds: dz's own fp32 error (denseutil.dz64); what its parts leave of it, 2^-24 of bf16's three
(half a step of 2^-8 each) and 2^-22 of fp16's two, whose rests are held times 2^11 (2^-36 where
they are subnormal); sums of n fp32 products per part, the parts' magnitudes together 1 + 2^-7
of dz's, and at most 64 slices' and parts' sums added."""
import ctypes

import pytest
import torch

import hipgemm_amd as hg
from denseutil import TINY, U, check, dz64

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
SIZES = [(1, 8, 8), (9, 24, 40), (131, 264, 72), (777, 200, 1032), (2051, 136, 264),
         (300, 1032, 4104), (70, 4104, 136), (1531, 2056, 1032)]


def bounds(dy, x, w, pre, act, gated):
    """{name: (value, bound)} of float32 dx and dw."""
    dz, e = dz64(dy, pre, act, gated)
    e = e + (2.0 ** -24 * dz.abs() + 4 * TINY[BF] if x.dtype == BF
             else 2.0 ** -22 * dz.abs() + 2.0 ** -36)
    xd, wd = x.double(), w.double()
    return {
        "dx": (dz @ wd, e @ wd.abs() + (dz.shape[1] + 64) * 1.01 * U * (dz.abs() @ wd.abs())),
        "dw": (dz.t() @ xd,
               e.t() @ xd.abs() + (dz.shape[0] + 64) * 1.01 * U * (dz.abs().t() @ xd.abs())),
    }


def make(M, N, K, dtype, gated, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0, t=dtype):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(t)

    rows = 2 * N if gated else N
    return (normal(M, K), normal(rows, K, std=K ** -0.5), normal(M, N, std=0.5),
            normal(M, rows, t=F32))


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("dtype", (BF, HF), ids=("bf16", "f16"))
@pytest.mark.parametrize("act,gated", [("silu", False), ("gelu_tanh", True), (None, False)],
                         ids=("linear", "gated", "float32 dy"))
def test_float32_weight_gradient(gpu, M, N, K, dtype, act, gated):
    x, w, dy, pre = make(M, N, K, dtype, gated, M)
    if act is None:
        dy = dy.float() * 1.0001
        pre = None
    back = hg.gated_linear_backward if gated else hg.linear_backward
    kw = dict(activation=act, grad_dtype=F32)
    dx, dw, db = back(dy, x, w, pre, need_bias=True, **kw)
    check("dw", dw, *bounds(dy, x, w, pre, act, gated)["dw"])
    # alone, again, and beside it the gradients that they are without it
    assert torch.equal(dw, back(dy, x, w, pre, need_x=False, **kw)[1])
    other = back(dy, x, w, pre, activation=act, need_bias=True, bias_dtype=F32)
    assert torch.equal(dx, other[0]) and torch.equal(db, other[2])


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("dtype", (BF, HF), ids=("bf16", "f16"))
@pytest.mark.parametrize("gated", (False, True), ids=("linear", "gated"))
def test_float32_descriptor(gpu, M, N, K, dtype, gated):
    """Of the C entry point, which has float32 dx too, into longer rows."""
    x, w, dy, pre = make(M, N, K, dtype, gated, M)
    dx = torch.full((M, K + 3), 7.0, device="cuda")
    dw = torch.full((w.shape[0], K + 5), 7.0, device="cuda")
    d = hg.LinearGradDesc(
        size=ctypes.sizeof(hg.LinearGradDesc), dy=dy.data_ptr(), x=x.data_ptr(),
        weight=w.data_ptr(), pre=pre.data_ptr(), dx=dx.data_ptr(), dw=dw.data_ptr(), lddy=N,
        ldx=K, ldw=K, ldp=w.shape[0], lddx=K + 3, lddw=K + 5, M=M, N=N, K=K, gated=int(gated),
        type=1 if dtype == BF else 2, dy_type=1 if dtype == BF else 2, pre_type=0, dx_dtype=2,
        dw_dtype=2, activation=3)
    need = hg.linear_backward_workspace_size(d)
    memory = torch.full((need + 256,), 255, dtype=torch.uint8, device="cuda")  # NaN
    d.workspace, d.workspace_bytes = memory.data_ptr(), need
    assert hg.linear_backward_raw(d) == 0
    assert bool((memory[need:] == 255).all())
    act = [a for a, c in hg.ACTIVATIONS.items() if c == 3 and a][0]
    want = bounds(dy, x, w, pre, act, gated)
    for name, t in (("dx", dx), ("dw", dw)):
        check(name, t[:, :K], *want[name])
        assert bool((t[:, K:] == 7.0).all())


@pytest.mark.parametrize("dtype", (BF, HF), ids=("bf16", "f16"))
def test_infinities(gpu, dtype):
    """An infinite x against a dz whose rests are zero stays infinite."""
    M, N, K = 70, 40, 72
    x, w, dy, _ = make(M, N, K, dtype, False, 0)
    x[3, 5] = float("inf")
    dy[7, 2] = float("inf")
    x[7, 6] = float("nan")
    dw = hg.linear_backward(dy.float(), x, w, grad_dtype=F32)[1]
    want = dy.double().t() @ x.double()
    bound = (M + 64) * 2 * U * (dy.double().abs().t() @ x.double().abs())
    check("dw", dw, want, bound)
