"""Products of more tiles, or slices of tiles, than CUs: each workgroup goes from one to the next,
with the next one's operands on their way while the last one's results are stored.  Every kernel
that takes several in turn, at odd sizes whose last step along K is not whole, against 64-bit
forms, with NaN beside and below the operands."""
import pytest
import torch

import hipgemm_amd as hg
from denseutil import backward64, check, gated64, linear64
from test_dense_kernels_gpu import amid, backward_plans, forward_plan, kind_of_plan

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
CUS = 256


def units(plan, M, N, cols=0):
    """Units of the two launches of a plan: of all columns, or those from first_columns on, and of
    the first columns.  cols: result columns of a tile."""
    tile_rows, tile_cols, slices, first = plan
    tile_cols = cols or tile_cols
    big = 128 if cols == plan[1] // 2 else 256
    return (-(-M // tile_rows) * -(-(N - first) // tile_cols) * slices,
            -(-M // 256) * (first // big))


# (tile rows, tile columns, in slices, first columns apart), sizes of linear, of gated
FORWARD = [
    ((64, 128, False, False), (131, 16389, 264), (131, 8200, 264)),
    ((64, 128, True, False), (131, 4101, 4104), (131, 2056, 4104)),
    ((64, 128, False, True), (777, 32997, 200), (777, 16392, 200)),
    ((128, 128, False, False), (77, 32997, 264), (77, 16392, 264)),
    ((128, 128, True, False), (77, 16389, 4104), (77, 8200, 4104)),
    ((128, 128, False, True), (4099, 8197, 200), (4099, 4104, 200)),
    ((256, 128, False, False), (32999, 261, 264), (32999, 136, 264)),
    ((256, 128, False, True), (2051, 16389, 328), (2051, 8200, 328)),
    ((256, 256, False, False), (6001, 4101, 200), (2307, 5000, 200)),
    ((256, 256, False, False), (6001, 4101, 1000), (2307, 5000, 1000)),
]


@pytest.mark.parametrize("kind", ("linear", "residual", "gated"))
@pytest.mark.parametrize("want,linear,gated", FORWARD)
def test_sizes_forward(want, linear, gated, kind):
    M, N, K = gated if kind == "gated" else linear
    p = forward_plan(M, N, K, kind)
    assert kind_of_plan(p) == want
    assert max(units(p, M, N, p[1] // 2 if kind == "gated" else p[1])) > CUS


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ("linear", "residual", "gated"))
@pytest.mark.parametrize("want,linear,gated", FORWARD)
def test_forward(gpu, want, linear, gated, kind):
    M, N, K = gated if kind == "gated" else linear
    for i, dtype in enumerate((BF, HF)):
        g = torch.Generator(device="cuda").manual_seed(M + i)
        rows = 2 * N if kind == "gated" else N
        x, w = amid(M, K, 1.0, dtype, g), amid(rows, K, K ** -0.5, dtype, g)
        b = torch.randn(rows, generator=g, device="cuda").to((dtype, F32)[i])
        act = ("gelu_tanh", "silu")[i]
        # results of the operands' type without pre, with it in fp32, and others
        for out, held in ((dtype, None), (dtype, F32), (F32, dtype)):
            kw = dict(bias=b, activation=act, out_dtype=out, save_pre=held or False)
            if kind == "gated":
                z, ez, y, ey = gated64(x, w, b, act, out, held or F32)
                got = hg.gated_linear(x, w, **kw)
            else:
                r = amid(M, N, 1.0, (dtype, F32)[i], g, beside=5) if kind == "residual" else None
                z, ez, y, ey = linear64(x, w, b, act, r, out, held or F32)
                got = hg.linear(x, w, residual=r, **kw)
            if held:
                got, pre = got
                check("pre", pre, z, ez)
            check("y", got, y, ey)
            del z, ez, y, ey, got


# "dx" or "dw", its kernel, gated, sizes
BACKWARD = [
    ("dx", (128, 128, False, False), False, (16387, 133, 520)),
    ("dx", (128, 128, False, False), True, (16387, 136, 520)),
    ("dx", (128, 128, True, False), True, (333, 4104, 4104)),
    ("dx", (128, 128, False, True), False, (8197, 133, 4104)),
    ("dx", (256, 128, False, False), False, (32999, 261, 264)),
    ("dx", (256, 128, False, False), True, (32999, 264, 264)),
    ("dx", (256, 128, True, False), False, (8197, 8197, 264)),
    ("dx", (256, 256, False, False), False, (6001, 133, 4104)),
    ("dx", (256, 256, False, False), True, (6001, 264, 4104)),
    ("dx", (256, 256, True, False), True, (2051, 4104, 4104)),
    ("dw", (128, 128, False, False), False, (77, 16389, 520)),
    ("dw", (128, 128, False, False), True, (131, 33000, 8)),
    ("dw", (128, 128, True, False), True, (4099, 264, 4104)),
    ("dw", (128, 128, False, True), True, (131, 4104, 4104)),
    ("dw", (256, 128, False, False), True, (777, 16392, 264)),
    ("dw", (256, 128, True, False), True, (4099, 4104, 520)),
    ("dw", (256, 256, False, False), False, (131, 32997, 1000)),
    ("dw", (256, 256, False, False), True, (777, 5000, 4104)),
    ("dw", (256, 256, True, False), True, (8197, 4104, 1000)),
]


def of(which, gated, size):
    """(its plan, M and N of the product)."""
    M, N, K = size
    rows = 2 * N if gated else N
    plan = backward_plans(M, N, K, gated)[which == "dw"]
    return plan, (rows, K) if which == "dw" else (M, K)


@pytest.mark.parametrize("which,want,gated,size", BACKWARD)
def test_sizes_backward(which, want, gated, size):
    plan, (m, n) = of(which, gated, size)
    assert kind_of_plan(plan) == want
    assert max(units(plan, m, n)) > CUS


@pytest.mark.gpu
@pytest.mark.parametrize("which,want,gated,size", BACKWARD)
def test_backward(gpu, which, want, gated, size):
    M, N, K = size
    back = hg.gated_linear_backward if gated else hg.linear_backward
    rows = 2 * N if gated else N
    for i, dtype in enumerate((BF, HF)):
        g = torch.Generator(device="cuda").manual_seed(M + i)
        x, w = amid(M, K, 1.0, dtype, g), amid(rows, K, K ** -0.5, dtype, g)
        pre = amid(M, rows, 1.0, (F32, dtype)[i], g)
        dy = amid(M, N, 1.0, dtype, g, beside=(0, 3)[i])
        dx, dw, _ = back(dy, x, w, pre, activation="silu", need_x=which == "dx",
                         need_weight=which == "dw")
        got = dw if which == "dw" else dx
        check(which, got, *backward64(dy, x, w, pre, "silu", gated, dtype)[which])
        # a float32 weight's gradient: a launch for each part of dz
        if which == "dw":
            got = back(dy, x, w, pre, activation="silu", need_x=False, grad_dtype=F32)[1]
            check(which, got, *backward64(dy, x, w, pre, "silu", gated, F32)[which])
