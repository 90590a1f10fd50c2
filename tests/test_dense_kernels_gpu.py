"""Every kernel that linear, gated_linear and their backward passes take for some sizes,
against 64-bit forms: the kernel of few rows, each tile, whole, in slices along K and with a
launch of its own for the first columns, at odd sizes, with NaN beside and below the operands."""
import ctypes

import pytest
import torch

import hipgemm_amd as hg
from denseutil import backward64, check, gated64, linear64

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
NAN = float("nan")


def amid(rows, cols, std, dtype, g, beside=8):
    """rows x cols of normals inside a larger tensor of NaN."""
    full = torch.full((rows + 3, cols + beside), NAN, device="cuda", dtype=dtype)
    v = full[:rows, :cols]
    v.copy_(torch.randn((rows, cols), generator=g, device="cuda") * std)
    return v


def forward_plan(M, N, K, kind):
    """kind: linear, residual, gated."""
    return hg.linear_select(hg.LinearDesc(
        size=ctypes.sizeof(hg.LinearDesc), M=M, N=N, K=K, gated=int(kind == "gated"), type=1,
        residual=int(kind == "residual")))


def backward_plans(M, N, K, gated):
    return hg.linear_backward_select(hg.LinearGradDesc(
        size=ctypes.sizeof(hg.LinearGradDesc), M=M, N=N, K=K, gated=int(gated), type=1, dx=1,
        dw=1))


# (tile rows, tile columns, in slices, first columns apart): sizes, of linear and of gated
FORWARD = [
    ((0, 0, False, False), (5, 517, 1032), (5, 520, 1032)),
    ((0, 0, False, False), (23, 261, 520), (23, 264, 520)),
    ((0, 0, False, False), (61, 517, 264), (61, 520, 264)),
    ((0, 0, True, False), (45, 133, 4104), (45, 136, 4104)),
    ((64, 128, False, False), (77, 133, 264), (77, 136, 264)),
    ((64, 128, True, False), (131, 261, 2056), (131, 264, 2056)),
    ((64, 128, False, False), (45, 14341, 520), (45, 8200, 200)),  # 64 rows at most
    ((64, 128, True, False), (45, 4101, 2056), (45, 2056, 2056)),
    ((128, 128, False, False), (201, 8197, 264), (77, 8200, 264)),
    ((128, 128, True, False), (2051, 133, 4104), (77, 2056, 4104)),
    ((128, 128, False, True), (2051, 8197, 264), (2051, 4104, 200)),
    ((256, 128, False, False), (777, 4997, 200), (201, 8200, 200)),
    ((256, 128, True, False), (2307, 517, 4104), (201, 4104, 4104)),
    ((256, 128, True, True), (2051, 8197, 4104), (2051, 4104, 4104)),
    ((256, 256, False, False), (777, 10245, 200), (777, 5000, 200)),
    ((256, 256, True, False), (2051, 2053, 4104), (131, 8200, 4104)),
]


def kind_of_plan(p):
    return (p[0], p[1], p[2] > 1, p[3] > 0)


@pytest.mark.parametrize("kind", ("linear", "residual", "gated"))
@pytest.mark.parametrize("want,linear,gated", FORWARD)
def test_forward_kernels(gpu, want, linear, gated, kind):
    M, N, K = gated if kind == "gated" else linear
    assert kind_of_plan(forward_plan(M, N, K, kind)) == want
    for i, dtype in enumerate((BF, HF)):
        g = torch.Generator(device="cuda").manual_seed(M + i)
        rows = 2 * N if kind == "gated" else N
        x, w = amid(M, K, 1.0, dtype, g), amid(rows, K, K ** -0.5, dtype, g)
        b = torch.randn(rows, generator=g, device="cuda").to((F32, dtype)[i])
        r = amid(M, N, 1.0, (dtype, F32)[i], g, beside=(0, 5)[i]) if kind == "residual" else None
        act = ("silu", "gelu_tanh")[i]
        full = torch.full((M + 2, N + 7), 7.0, device="cuda", dtype=(dtype, F32)[i])
        out = full[1:M + 1, (3, 0)[i]:(3, 0)[i] + N]
        if kind == "gated":
            z, ez, y, ey = gated64(x, w, b, act, out.dtype, F32)
            _, pre = hg.gated_linear(x, w, bias=b, activation=act, out=out, save_pre=True)
            plain = hg.gated_linear(x, w, bias=b, activation=act, out_dtype=out.dtype)
        else:
            z, ez, y, ey = linear64(x, w, b, act, r, out.dtype, F32)
            _, pre = hg.linear(x, w, bias=b, activation=act, residual=r, out=out, save_pre=True)
            plain = hg.linear(x, w, bias=b, activation=act, residual=r, out_dtype=out.dtype)
        check("y", out, y, ey)
        check("pre", pre, z, ez)
        assert torch.equal(plain, out)
        out.fill_(7.0)
        assert bool((full == 7.0).all())


# (kernel of dx or None, of dw or None), gated, sizes; kernels as above
BACKWARD = [
    (((64, 128, False, False), (128, 128, True, False)), True, (2307, 520, 264)),
    (((64, 128, True, False), None), True, (131, 1032, 264)),
    (((64, 128, True, False), None), False, (333, 4101, 264)),
    (((64, 128, False, False), (128, 128, True, False)), False, (4099, 1029, 200)),
    (((128, 128, False, False), None), False, (2051, 133, 1032)),
    (((128, 128, True, False), None), True, (77, 2056, 4104)),
    (((256, 128, False, False), None), False, (2051, 133, 2056)),
    (((256, 128, True, False), None), True, (2307, 2056, 520)),
    (((256, 256, False, False), None), False, (2051, 133, 4104)),
    (((256, 256, True, False), None), True, (2051, 2056, 2056)),
    (((128, 128, False, True), None), True, (2051, 264, 8200)),
    ((None, (256, 128, False, False)), True, (77, 8200, 200)),
    ((None, (256, 256, False, False)), True, (77, 10248, 520)),
    ((None, (256, 256, True, False)), True, (2051, 8200, 200)),
    ((None, (128, 128, False, True)), True, (131, 2056, 4104)),
    ((None, (128, 128, True, True)), True, (1531, 2056, 4104)),
]


@pytest.mark.parametrize("want,gated,size", BACKWARD)
def test_backward_kernels(gpu, want, gated, size):
    M, N, K = size
    for got, kind in zip(backward_plans(M, N, K, gated), want):
        assert kind is None or kind_of_plan(got) == kind
    f = hg.gated_linear_backward if gated else hg.linear_backward
    for i, dtype in enumerate((BF, HF)):
        g = torch.Generator(device="cuda").manual_seed(M + i)
        rows = 2 * N if gated else N
        x, w = amid(M, K, 1.0, dtype, g), amid(rows, K, K ** -0.5, dtype, g)
        pre = amid(M, rows, 1.0, (F32, dtype)[i], g, beside=(0, 8)[i])
        dy = amid(M, N, 1.0, dtype, g, beside=(0, 3)[i])
        grad = (dtype, F32)[i]
        # what the call's memory holds before it is written: NaN
        torch.cuda.empty_cache()
        scratch = torch.full((1 << 28,), NAN, device="cuda")
        del scratch
        grads = f(dy, x, w, pre, activation="silu", need_bias=True, grad_dtype=grad)
        bounds = backward64(dy, x, w, pre, "silu", gated, grad)
        for name, t in zip(("dx", "dw", "db"), grads):
            check(name, t, *bounds[name])


@pytest.mark.parametrize("M,N,K,gated", ((5, 5, 200, False), (1029, 605, 264, False),
                                         (77, 5, 4104, False), (777, 136, 1000, True),
                                         (1531, 2001, 1000, False), (1, 8, 8, True)))
def test_both_products_in_one_launch(gpu, M, N, K, gated):
    """Whole tiles of 128 x 128 with a CU each; a gradient alone has the same bits."""
    plans = backward_plans(M, N, K, gated)
    assert plans == ((128, 128, 1, 0),) * 2
    rows = 2 * N if gated else N
    assert (-(-M // 128) + -(-rows // 128)) * -(-K // 128) <= 256
    f = hg.gated_linear_backward if gated else hg.linear_backward
    for i, dtype in enumerate((BF, HF)):
        g = torch.Generator(device="cuda").manual_seed(M + i)
        x, w = amid(M, K, 1.0, dtype, g), amid(rows, K, K ** -0.5, dtype, g)
        pre, dy = amid(M, rows, 1.0, F32, g), amid(M, N, 1.0, dtype, g, beside=3)
        grad = (F32, dtype)[i]
        torch.cuda.empty_cache()
        scratch = torch.full((1 << 28,), NAN, device="cuda")
        del scratch
        both = f(dy, x, w, pre, activation="silu", need_bias=True, grad_dtype=grad)
        bounds = backward64(dy, x, w, pre, "silu", gated, grad)
        for name, t in zip(("dx", "dw", "db"), both):
            check(name, t, *bounds[name])
        dx, _, _ = f(dy, x, w, pre, activation="silu", need_weight=False, grad_dtype=grad)
        _, dw, _ = f(dy, x, w, pre, activation="silu", need_x=False, grad_dtype=grad)
        assert torch.equal(dx, both[0]) and torch.equal(dw, both[1])


@pytest.mark.parametrize("M,N,K", ((70, 72, 136), (777, 200, 1032), (9, 1032, 264)))
def test_backward_reads_dy(gpu, M, N, K):
    """Without an activation the products read dy itself, with NaN beside and below it."""
    for dtype in (BF, HF):
        g = torch.Generator(device="cuda").manual_seed(M)
        x, w = amid(M, K, 1.0, dtype, g), amid(N, K, K ** -0.5, dtype, g)
        dy = amid(M, N, 1.0, dtype, g)
        bounds = backward64(dy, x, w, None, None, False, dtype)
        for name, t in zip(("dx", "dw", "db"), hg.linear_backward(dy, x, w, need_bias=True)):
            check(name, t, *bounds[name])


def test_results_past_4_gib(gpu):
    """Offsets in y, pre, dz, x and dx past 32 bits: 600000 rows of 4096 columns."""
    M, N, K = 600000, 4096, 8
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(M, K, generator=g, device="cuda").to(BF)
    w = torch.randn(N, K, generator=g, device="cuda").to(BF)
    rows = torch.tensor([0, 1, 262143, 262144, 524287, 524288, 524289, 599999], device="cuda")
    y, pre = hg.linear(x, w, activation="silu", save_pre=True)
    z, ez, want, ey = linear64(x[rows], w, None, "silu", None, BF, F32)
    check("y", y[rows], want, ey)
    check("pre", pre[rows], z, ez)
    # gradients: of the listed rows alone (y, as dy, is zero in the others)
    keep = torch.zeros(M, 1, device="cuda", dtype=BF)
    keep[rows] = 1
    y.mul_(keep)
    del keep
    dx, dw, _ = hg.linear_backward(y, x, w, pre, activation="silu")
    bounds = backward64(y[rows], x[rows], w, pre[rows], "silu", False, BF)
    check("dx", dx[rows], *bounds["dx"])
    # (zeros add no error, but the sum has M terms)
    value, bound = bounds["dw"]
    check("dw", dw, value, bound)
    assert int(dx.any(1).sum()) == rows.numel()


def test_operands_past_4_gib(gpu):
    """x and dx of 600000 rows of 4096 columns."""
    M, N, K = 600000, 16, 4096
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.empty(M, K, device="cuda", dtype=BF).normal_(generator=g)
    w = (torch.randn(N, K, generator=g, device="cuda") / 64).to(BF)
    rows = torch.tensor([0, 262144, 524287, 524288, 599999], device="cuda")
    y = hg.linear(x, w)
    _, _, want, ey = linear64(x[rows], w, None, None, None, BF)
    check("y", y[rows], want, ey)
    dy = torch.zeros(M, N, device="cuda", dtype=BF)
    dy[rows] = torch.randn(rows.numel(), N, generator=g, device="cuda").to(BF)
    dx, dw, _ = hg.linear_backward(dy, x, w)
    bounds = backward64(dy[rows], x[rows], w, None, None, False, BF)
    check("dx", dx[rows], *bounds["dx"])
    check("dw", dw, *bounds["dw"])


def test_two_streams_and_two_graphs(gpu):
    """Calls with workspaces on two streams at once, and two captured graphs of them replayed
    at once: everything as one after the other."""
    sizes = ((131, 261, 2056), (45, 133, 4104))
    g = torch.Generator(device="cuda").manual_seed(3)
    args = []
    for M, N, K in sizes:
        assert forward_plan(M, N, K, "linear")[2] > 1
        x, w = amid(M, K, 1.0, BF, g), amid(N, K, K ** -0.5, BF, g)
        args.append((x, w, amid(M, N, 1.0, BF, g, beside=0)))

    def run(x, w, dy):
        y, pre = hg.linear(x, w, activation="silu", save_pre=True)
        return (y, *hg.linear_backward(dy, x, w, pre, activation="silu", need_bias=True))

    want = [run(*a) for a in args]
    streams = [torch.cuda.Stream() for _ in args]
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        for s, a in zip(streams, args):
            with torch.cuda.stream(s):
                got.append(run(*a))
    torch.cuda.synchronize()
    for i, out in enumerate(got):
        assert all(torch.equal(p, q) for p, q in zip(out, want[i % 2])), i
    graphs, static = [], []
    for s, a in zip(streams, args):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            static.append([run(*a) for _ in range(4)])
        graphs.append(graph)
    for n in range(3):
        for outs in static:
            for out in outs:
                for t in out:
                    t.zero_()
        torch.cuda.synchronize()
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for i, outs in enumerate(static):
            for out in outs:
                assert all(torch.equal(p, q) for p, q in zip(out, want[i])), (n, i)
