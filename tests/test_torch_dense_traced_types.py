"""Traces of linear and gated_linear refuse the types that the calls refuse (no GPU)."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import hipgemm_amd as hg
import hipgemm_amd.torch_dense as td

BF, HF, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64


def empty(*shape, t=BF, device="cuda"):
    return torch.empty(*shape, dtype=t, device=device)


REFUSED = {
    "float32 x": lambda f: f(empty(5, 64, t=F32), empty(48, 64)),
    "float32 weight": lambda f: f(empty(5, 64), empty(48, 64, t=F32)),
    "float32 both": lambda f: f(empty(5, 64, t=F32), empty(48, 64, t=F32)),
    "two types": lambda f: f(empty(5, 64, t=HF), empty(48, 64)),
    "bias": lambda f: f(empty(5, 64), empty(48, 64), empty(48, t=F64)),
    "out_dtype": lambda f: f(empty(5, 64), empty(48, 64), out_dtype=F64),
    "K": lambda f: f(empty(5, 60), empty(48, 60)),
    "device": lambda f: f(empty(5, 64), empty(48, 64, device="cpu")),
}


@pytest.mark.parametrize("grad", (False, True), ids=("plain", "grad"))
@pytest.mark.parametrize("f", (td.linear, td.gated_linear), ids=("linear", "gated"))
@pytest.mark.parametrize("name", REFUSED)
def test_refused(name, f, grad):
    def call(x, w, *a, **kw):
        return f(x, w.requires_grad_() if grad else w, *a, **kw)

    with FakeTensorMode(), pytest.raises(hg.HipGemmError):
        REFUSED[name](call)


def test_residual():
    with FakeTensorMode():
        x, w = empty(5, 64), empty(48, 64)
        with pytest.raises(hg.HipGemmError):
            td.linear(x, w, residual=empty(5, 48, t=F64))
        for t in (BF, HF, F32):
            assert td.linear(x, w, empty(48, t=t), residual=empty(5, 48, t=t),
                             out_dtype=t).dtype == t
            assert td.gated_linear(x, w, empty(48, t=t), out_dtype=t).shape == (5, 24)
