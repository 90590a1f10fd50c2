"""What the autograd of linear and gated_linear allocates beside its results (no GPU)."""
import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

import hipgemm_amd.torch_dense as td

BF = torch.bfloat16


class Sizes(TorchDispatchMode):
    """Shapes and types of every tensor that an operation returns."""

    def __init__(self):
        super().__init__()
        self.seen = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        out = func(*args, **(kwargs or {}))
        for t in out if isinstance(out, (tuple, list)) else (out,):
            if isinstance(t, torch.Tensor):
                self.seen.append((tuple(t.shape), t.dtype))
        return out


@pytest.mark.parametrize("gated", (False, True), ids=("linear", "gated"))
def test_no_gradient_of_z(gated):
    x = torch.empty(6, 64, dtype=BF, device="meta", requires_grad=True)
    w = torch.empty(48, 64, dtype=BF, device="meta", requires_grad=True)
    y = td.gated_linear(x, w) if gated else td.linear(x, w, activation="silu")
    with Sizes() as sizes:
        dx, dw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
    assert dx.shape == x.shape and dw.shape == w.shape
    assert (x.shape, BF) in sizes.seen
    assert ((6, 48), torch.float32) not in sizes.seen


class Stop(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y):
        return y.sum()

    @staticmethod
    def backward(ctx, dy):
        return None


def test_no_gradient_at_all():
    """A function behind that passes none on: as with torch's own operators there is none."""
    x = torch.empty(6, 64, dtype=BF, device="meta", requires_grad=True)
    w = torch.empty(48, 64, dtype=BF, device="meta")
    assert torch.autograd.grad(Stop.apply(td.linear(x, w, activation="silu")), x,
                               allow_unused=True) == (None,)
    assert torch.autograd.grad(Stop.apply(torch.nn.functional.linear(x, w)), x,
                               allow_unused=True) == (None,)
