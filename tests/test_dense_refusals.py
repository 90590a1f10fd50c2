"""Arguments that linear, gated_linear and their backward passes refuse, on the CPU: checks
come before any GPU call."""
import ctypes

import pytest

import hipgemm_amd as hg

INVALID = 1
FAKE = 1 << 20


def desc(**kw):
    d = hg.LinearDesc()
    d.size = ctypes.sizeof(d)
    for k, v in dict(dict(x=FAKE, weight=FAKE, y=FAKE, ldx=64, ldw=64, ldy=32, M=4, N=32, K=64,
                          type=1, pre_dtype=2), **kw).items():
        setattr(d, k, v)
    return d


def grad(**kw):
    d = hg.LinearGradDesc()
    d.size = ctypes.sizeof(d)
    for k, v in dict(dict(dy=FAKE, x=FAKE, weight=FAKE, dx=FAKE, dw=FAKE, lddy=32, ldx=64, ldw=64,
                          lddx=64, lddw=64, M=4, N=32, K=64, type=1, dy_type=1), **kw).items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw", [
    dict(size=0), dict(M=-1), dict(N=-1), dict(K=-8), dict(K=60), dict(M=(1 << 30) + 1),
    dict(K=(1 << 21) + 8, ldx=1 << 22, ldw=1 << 22), dict(N=(1 << 21) + 1, ldy=1 << 22),
    dict(gated=2), dict(gated=1, N=36, ldy=36), dict(gated=1, residual=FAKE, ldr=32),
    dict(type=0), dict(type=3), dict(out_dtype=3), dict(out_dtype=-1), dict(activation=4),
    dict(bias_type=3), dict(pre_dtype=3), dict(residual_type=3), dict(x=0), dict(weight=0), dict(y=0),
    dict(x=FAKE + 8), dict(weight=FAKE + 2), dict(y=FAKE + 1), dict(ldx=56), dict(ldx=68),
    dict(ldw=60), dict(ldw=(1 << 21) + 8), dict(ldy=31), dict(bias=FAKE + 2),
    dict(residual=FAKE, ldr=31), dict(residual=FAKE + 2, ldr=32), dict(pre=FAKE, ldp=31),
    dict(pre=FAKE + 1, ldp=32), dict(gated=1, pre=FAKE, ldp=63),
])
def test_linear_refuses(kw):
    assert hg.linear_raw(desc(**kw)) == INVALID


@pytest.mark.parametrize("kw", [
    dict(size=0), dict(M=-1), dict(N=-1), dict(K=60), dict(gated=2), dict(type=0),
    dict(dy_type=3), dict(pre_type=3), dict(dx_dtype=3), dict(dw_dtype=3), dict(db_dtype=-1), dict(activation=-1),
    dict(dy=0), dict(dy=FAKE + 1), dict(lddy=31), dict(x=0), dict(weight=0), dict(x=FAKE + 4),
    dict(ldx=60), dict(ldw=56), dict(lddx=63), dict(lddw=63), dict(dx=FAKE + 1), dict(dw=FAKE + 1),
    dict(db=FAKE + 1), dict(activation=1), dict(activation=1, pre=FAKE, ldp=31), dict(activation=1, pre=FAKE + 2, ldp=32),
    dict(gated=1), dict(gated=1, pre=FAKE, ldp=63), dict(gated=1, pre=FAKE, ldp=64),  # no workspace
])
def test_backward_refuses(kw):
    assert hg.linear_backward_raw(grad(**kw)) == INVALID


def test_null_descriptors():
    L = hg.lib()
    assert L.hipgemm_linear(None, None) == INVALID
    assert L.hipgemm_linear_backward(None, None) == INVALID
    assert L.hipgemm_linear_workspace_size(None) == 0
    assert L.hipgemm_linear_backward_workspace_size(None) == 0


def test_no_ops():
    assert hg.linear_raw(desc(M=0, x=0, y=0)) == 0
    assert hg.linear_raw(desc(N=0, weight=0, y=0)) == 0


def test_torch_refusals():
    import torch
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    w = torch.zeros(32, 64, dtype=torch.bfloat16)
    for call in (lambda: hg.linear(x, w), lambda: hg.gated_linear(x, w),
                 lambda: hg.linear_backward(x[:, :32], x, w),
                 lambda: hg.gated_linear_backward(x[:, :16], x, w, x[:, :32])):
        with pytest.raises(hg.HipGemmError):
            call()
