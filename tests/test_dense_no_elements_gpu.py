"""Sums of nothing, whose operands have no elements: any address and any stride will do."""
import ctypes

import pytest
import torch

import hipgemm_amd as hg

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
STRIDES = (0, 8, 3 << 29, (1 << 31) - 8, -8, -(1 << 40))


@pytest.mark.parametrize("stride", STRIDES)
@pytest.mark.parametrize("M", (1, 40, 300))
@pytest.mark.parametrize("gated", (0, 1), ids=("linear", "gated"))
def test_no_k(gpu, gated, M, stride):
    """y = act(b) + r, act(bg) bu."""
    N = 264
    rows = 2 * N if gated else N
    b = torch.randn(rows, device="cuda")
    r = torch.randn(M, N, device="cuda")
    y = torch.full((M, N), 7.0, device="cuda")
    d = hg.LinearDesc(size=ctypes.sizeof(hg.LinearDesc), bias=b.data_ptr(),
                      residual=0 if gated else r.data_ptr(), y=y.data_ptr(), ldx=stride,
                      ldw=stride, ldr=N, ldy=N, M=M, N=N, K=0, gated=gated, type=1, bias_type=0,
                      residual_type=0, out_dtype=2, activation=hg.ACTIVATIONS["relu"])
    assert hg.linear_workspace_size(d) == 0
    assert hg.linear_raw(d) == 0
    z = b.relu()
    want = (z[:N] * b[N:]).expand(M, N) if gated else z + r
    assert torch.equal(y, want)


@pytest.mark.parametrize("stride", STRIDES)
@pytest.mark.parametrize("gated", (0, 1), ids=("linear", "gated"))
@pytest.mark.parametrize("M,N,K", ((300, 0, 264), (0, 264, 264)))
def test_no_rows_or_columns(gpu, M, N, K, gated, stride):
    """Gradients of zeros."""
    rows = 2 * N if gated else N
    dx = torch.full((M, K), 7.0, device="cuda", dtype=BF)
    dw = torch.full((rows, K), 7.0, device="cuda", dtype=BF)
    db = torch.full((rows,), 7.0, device="cuda", dtype=BF)
    d = hg.LinearGradDesc(size=ctypes.sizeof(hg.LinearGradDesc), dx=dx.data_ptr(),
                          dw=dw.data_ptr(), db=db.data_ptr(), lddy=stride, ldx=stride, ldw=stride,
                          ldp=stride, lddx=K, lddw=K, M=M, N=N, K=K, gated=gated, type=1,
                          dy_type=1, pre_type=0, dx_dtype=0, dw_dtype=0, db_dtype=0)
    need = hg.linear_backward_workspace_size(d)
    memory = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    d.workspace, d.workspace_bytes = memory.data_ptr(), need
    assert hg.linear_backward_raw(d) == 0
    for t in (dx, dw, db):
        assert not bool(t.any())


def test_views(gpu):
    """The same of tensors: a view without columns whose rows lie far apart."""
    x = torch.empty(8, device="cuda", dtype=BF).as_strided((5, 0), (3 << 29, 1))
    w = torch.empty(40, 0, device="cuda", dtype=BF)
    b = torch.randn(40, device="cuda")
    y = hg.linear(x, w, bias=b, out_dtype=F32)
    assert torch.equal(y, b.expand(5, 40))
