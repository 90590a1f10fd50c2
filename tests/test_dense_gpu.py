"""Products of 16-bit operands with epilogues (linear, gated_linear) and their backward
passes against 64-bit forms."""
import pytest
import torch

import hipgemm_amd as hg
from denseutil import act64, backward64, check, dz64, gated64, linear64

pytestmark = pytest.mark.gpu

ACTS = (None, "relu", "silu", "gelu_tanh")
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def make(M, N, K, dtype, seed=0, gated=False, bias=None, residual=None, pad=0):
    """x, weight, bias, residual, dy; pad: further columns of the rows' storage."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(rows, cols, std, t):
        v = torch.randn((rows, cols + pad), generator=g, device="cuda") * std
        return v.to(t)[:, :cols]

    rows = 2 * N if gated else N
    x, w = normal(M, K, 1.0, dtype), normal(rows, K, max(K, 1) ** -0.5, dtype)
    b = normal(1, rows, 0.3, bias)[0] if bias else None
    r = normal(M, N, 1.0, residual) if residual else None
    return x, w, b, r, normal(M, N, 1.0, dtype)


SIZES = [
    (1, 1, 8), (1, 8, 8), (1, 4096, 512), (2, 33, 64), (3, 5, 16), (5, 130, 72), (16, 256, 1024),
    (17, 96, 136), (33, 200, 64), (64, 512, 520), (65, 129, 128), (128, 128, 64), (129, 257, 200),
    (200, 1000, 328), (257, 300, 1032), (300, 2001, 96), (513, 136, 2056), (700, 640, 64),
]


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("dtype", (BF, HF), ids=("bf16", "f16"))
def test_linear(gpu, M, N, K, dtype):
    for i, act in enumerate(ACTS):
        bias = (None, dtype, F32, None)[i]
        res = (dtype, None, F32, HF if dtype == BF else BF)[i]
        out = (dtype, F32, dtype, dtype)[i]
        x, w, b, r, _ = make(M, N, K, dtype, i, bias=bias, residual=res)
        held = (F32, dtype, F32, dtype)[i]
        z, ez, y, ey = linear64(x, w, b, act, r, out, held)
        got, pre = hg.linear(x, w, bias=b, activation=act, residual=r, out_dtype=out,
                             save_pre=True if held == F32 else held)
        assert got.dtype == out and pre.dtype == held
        check(f"y {act}", got, y, ey)
        check(f"pre {act}", pre, z, ez)
        # without pre: the same values
        assert torch.equal(got, hg.linear(x, w, bias=b, activation=act, residual=r,
                                          out_dtype=out))


@pytest.mark.parametrize("M,N,K", [(m, (n + 7) // 8 * 8, k) for m, n, k in SIZES])
@pytest.mark.parametrize("dtype", (BF, HF), ids=("bf16", "f16"))
def test_gated(gpu, M, N, K, dtype):
    for i, act in enumerate(("silu", "gelu_tanh", "relu", None)):
        out = (dtype, F32, dtype, dtype)[i]
        x, w, b, _, _ = make(M, N, K, dtype, i, gated=True, bias=(None, F32, dtype, None)[i])
        held = (F32, dtype, F32, dtype)[i]
        z, ez, y, ey = gated64(x, w, b, act, out, held)
        got, pre = hg.gated_linear(x, w, bias=b, activation=act, out_dtype=out, save_pre=held)
        check(f"y {act}", got, y, ey)
        check(f"pre {act}", pre, z, ez)
        assert torch.equal(got, hg.gated_linear(x, w, bias=b, activation=act, out_dtype=out))


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("dtype", (BF, HF), ids=("bf16", "f16"))
def test_linear_backward(gpu, M, N, K, dtype):
    for i, act in enumerate(ACTS):
        grad = (dtype, F32, dtype, F32)[i]
        x, w, b, _, dy = make(M, N, K, dtype, i, bias=dtype)
        if i == 3:
            dy = dy.float()
        pre = None
        if act:
            _, pre = hg.linear(x, w, bias=b, activation=act, save_pre=(F32, dtype)[i % 2])
        want = backward64(dy, x, w, pre, act, False, grad)
        got = hg.linear_backward(dy, x, w, pre, activation=act, need_bias=True, grad_dtype=grad)
        for name, t in zip(("dx", "dw", "db"), got):
            assert t.dtype == (dtype if name == "dx" else grad)
            check(f"{name} {act}", t, *want[name])


@pytest.mark.parametrize("M,N,K", [(m, (n + 7) // 8 * 8, k) for m, n, k in SIZES])
@pytest.mark.parametrize("dtype", (BF, HF), ids=("bf16", "f16"))
def test_gated_backward(gpu, M, N, K, dtype):
    for i, act in enumerate(("silu", "gelu_tanh", "relu", None)):
        grad = (dtype, F32, F32, dtype)[i]
        x, w, b, _, dy = make(M, N, K, dtype, i, gated=True, bias=dtype)
        _, pre = hg.gated_linear(x, w, bias=b, activation=act, save_pre=(F32, dtype)[i % 2])
        want = backward64(dy, x, w, pre, act, True, grad)
        got = hg.gated_linear_backward(dy, x, w, pre, activation=act, need_bias=True,
                                       grad_dtype=grad)
        for name, t in zip(("dx", "dw", "db"), got):
            check(f"{name} {act}", t, *want[name])


@pytest.mark.parametrize("gated", (False, True), ids=("linear", "gated"))
def test_needs(gpu, gated):
    """Each gradient alone is the one that comes with the others."""
    f = hg.gated_linear if gated else hg.linear
    back = hg.gated_linear_backward if gated else hg.linear_backward
    x, w, b, _, dy = make(150, 136, 264, BF, gated=gated, bias=BF)
    _, pre = f(x, w, bias=b, activation="silu", save_pre=True)
    all3 = back(dy, x, w, pre, activation="silu", need_bias=True)
    for i in range(3):
        need = [j == i for j in range(3)]
        one = back(dy, x, w, pre, activation="silu", need_x=need[0], need_weight=need[1],
                   need_bias=need[2])
        for j in range(3):
            assert (one[j] is None) == (j != i)
        assert torch.equal(one[i], all3[i])


@pytest.mark.parametrize("dtype", (BF, HF), ids=("bf16", "f16"))
def test_views(gpu, dtype):
    """Rows longer than the matrix, results and residuals into and from views of any
    alignment; what lies beside them stays."""
    M, N, K = 70, 131, 136
    x, w, b, r, dy = make(M, N, K, dtype, 1, bias=F32, residual=dtype, pad=8)
    _, _, y, ey = linear64(x, w, b, "silu", r, dtype)
    for off, width in ((0, N), (1, N + 3), (8, N + 21)):
        full = torch.full((M + 2, off + width), 7.0, device="cuda", dtype=dtype)
        out = full[1:M + 1, off:off + N]
        assert hg.linear(x, w, bias=b, activation="silu", residual=r, out=out) is out
        check("out", out, y, ey)
        full[1:M + 1, off:off + N] = 7.0
        assert bool((full == 7.0).all())
        # in place on the residual
        full[1:M + 1, off:off + N] = r
        hg.linear(x, w, bias=b, activation="silu", residual=out, out=out)
        check("in place", out, y, ey)
    # gradients of views
    _, pre = hg.linear(x, w, bias=b, activation="silu", save_pre=True)
    want = backward64(dy, x, w, pre, "silu", False, dtype)
    big = torch.zeros(M, N + 5, device="cuda", dtype=F32)
    big[:, 3:N + 3] = pre
    for name, t in zip(("dx", "dw", "db"),
                       hg.linear_backward(dy, x, w, big[:, 3:N + 3], activation="silu",
                                          need_bias=True)):
        check(name, t, *want[name])


def test_empty(gpu):
    for M, N, K in ((0, 16, 8), (4, 0, 8), (4, 16, 0), (0, 0, 0)):
        for gated in (False, True):
            x, w, b, r, dy = make(M, N, K, BF, gated=gated, bias=BF, residual=BF)
            if gated:
                y, pre = hg.gated_linear(x, w, bias=b, save_pre=True)
                _, _, want, bound = gated64(x, w, b, "silu", BF)
                grads = hg.gated_linear_backward(dy, x, w, pre, need_bias=True)
            else:
                y, pre = hg.linear(x, w, bias=b, activation="silu", residual=r, save_pre=True)
                _, _, want, bound = linear64(x, w, b, "silu", r, BF)
                grads = hg.linear_backward(dy, x, w, pre, activation="silu", need_bias=True)
            check("y", y, want, bound)
            wants = backward64(dy, x, w, pre, "silu", gated, BF)
            for name, t in zip(("dx", "dw", "db"), grads):
                check(name, t, *wants[name])


@pytest.mark.parametrize("M", (1, 3, 40, 200))
def test_nonfinite_rows(gpu, M):
    """An infinity or NaN in a row of x reaches that row's results only; one in a row of
    the weight that column's.  (Finite elsewhere, sums' ends included: K is no multiple of a
    step.)"""
    N, K = 200, 72
    x, w, b, r, _ = make(M, N, K, BF, 2, bias=F32, residual=BF)
    clean = hg.linear(x, w, bias=b, residual=r)
    x2, w2 = x.clone(), w.clone()
    x2[M // 2, K - 1] = float("nan")
    w2[7, 0] = float("inf")
    got = hg.linear(x2, w2, bias=b, residual=r)
    rows = torch.arange(M, device="cuda") != M // 2
    cols = torch.arange(N, device="cuda") != 7
    assert bool(got[M // 2].isnan().all())
    assert bool((~got[rows][:, 7].isfinite()).all())
    assert torch.equal(got[rows][:, cols], clean[rows][:, cols])


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("gated", (False, True), ids=("linear", "gated"))
def test_slopes_far_out(gpu, act, gated):
    """Slopes and activations of large, infinite and NaN sums: the limits, no NaN from
    products of their parts."""
    if gated and act is None:
        pytest.skip("the linear case")
    v = torch.tensor([0.0, -0.0, 1e-30, 1.0, -1.0, 11.0, -11.0, 100.0, -100.0, 3e4, -3e4, 1e19,
                      -1e19, 3e38, -3e38, float("inf"), -float("inf"), float("nan")],
                     device="cuda").to(BF)
    n = v.numel()
    N = 24
    x = torch.zeros(n, 8, device="cuda", dtype=BF)
    w = torch.zeros(2 * N if gated else N, 8, device="cuda", dtype=BF)
    pre = torch.ones(n, 2 * N if gated else N, device="cuda", dtype=BF)
    pre[:, :N] = v[:, None]
    dy = torch.ones(n, N, device="cuda", dtype=BF)
    back = hg.gated_linear_backward if gated else hg.linear_backward
    # dx of a weight that picks one column of dz
    w[0, 0] = 1
    dx, _, _ = back(dy, x, w, pre, activation=act)
    # Slopes are constant past +-1e30; activations are not (an infinite du times a weight of
    # zero is NaN).
    lim = pre.double().clamp(-1e30, 1e30) if act else pre.double()
    want, e = dz64(dy, lim, act, gated)
    if gated:
        want[:, N:] = act64(pre[:, :N].double(), act)
    want = (want @ w.double())[:, 0]
    keep = ~v.isnan()
    check("slope", dx[keep, 0], want[keep], (e[:, 0] + 2.0 ** -8 * want.abs() + 2.0 ** -133)[keep])
    if act:
        assert bool(dx[~keep, 0].isnan().all())


@pytest.mark.parametrize("gated", (False, True), ids=("linear", "gated"))
def test_against_differences(gpu, gated):
    """The gradients along random directions are the differences of the 64-bit form.  The
    operands are quarters and the biases sixteenths, so that fp16 holds z exactly and the
    gradients' own bounds are all there is (1e-6 of the terms for the differences)."""
    M, N, K, act = 40, 48, 56, "gelu_tanh"
    g = torch.Generator(device="cuda").manual_seed(9)
    rows = 2 * N if gated else N

    def grid(*shape, steps, of):
        return torch.randint(-steps, steps + 1, shape, generator=g, device="cuda").double() / of

    base = [grid(M, K, steps=2, of=4), grid(rows, K, steps=1, of=4), grid(rows, steps=8, of=16)]
    dy = torch.randn(M, N, generator=g, device="cuda").to(HF)
    x, w, b = base[0].to(HF), base[1].to(HF), base[2].float()
    f = hg.gated_linear if gated else hg.linear
    back = hg.gated_linear_backward if gated else hg.linear_backward
    _, pre = f(x, w, bias=b, activation=act, save_pre=True)
    grads = back(dy, x, w, pre, activation=act, need_bias=True, grad_dtype=F32)
    bounds = backward64(dy, x, w, pre, act, gated, F32)

    def loss(x, w, b):
        z = x @ w.t() + b
        y = act64(z[:, :N], act) * z[:, N:] if gated else act64(z, act)
        return float((y * dy.double()).sum())

    for i, name in enumerate(("dx", "dw", "db")):
        d = torch.randn(base[i].shape, generator=g, device="cuda", dtype=torch.float64)
        h = 1e-5
        up, down = list(base), list(base)
        up[i], down[i] = base[i] + h * d, base[i] - h * d
        diff = (loss(*up) - loss(*down)) / (2 * h)
        along = float((grads[i].double() * d).sum())
        value, bound = bounds[name]
        room = float((bound * d.abs()).sum()) + 1e-6 * float((value * d).abs().sum())
        assert abs(along - diff) <= room, (name, along, diff, room)


@pytest.mark.parametrize("gated", (False, True), ids=("linear", "gated"))
def test_same_bits_twice(gpu, gated):
    f = hg.gated_linear if gated else hg.linear
    back = hg.gated_linear_backward if gated else hg.linear_backward
    for M, N, K in ((300, 256, 2048), (2048, 128, 256), (8, 4096, 4096)):
        x, w, b, _, dy = make(M, N, K, BF, 5, gated=gated, bias=BF)
        first = None
        for _ in range(3):
            y, pre = f(x, w, bias=b, activation="silu", save_pre=True)
            now = (y, pre, *back(dy, x, w, pre, activation="silu", need_bias=True))
            if first:
                assert all(torch.equal(a, c) for a, c in zip(first, now))
            first = now


def test_streams_and_graphs(gpu):
    """On a stream of the caller's, and captured: replays give the eager results, with
    eager calls in between."""
    M, N, K = 96, 512, 1024
    x, w, b, r, dy = make(M, N, K, BF, 6, gated=False, bias=BF, residual=BF)
    wg = torch.cat((w, w.flip(0)))
    side = torch.cuda.Stream()

    def run(stream=None):
        y, pre = hg.linear(x, w, bias=b, activation="silu", residual=r, save_pre=True,
                           stream=stream)
        h, z = hg.gated_linear(x, wg, save_pre=True, stream=stream)
        return (y, *hg.linear_backward(dy, x, w, pre, activation="silu", need_bias=True,
                                       stream=stream), h,
                *hg.gated_linear_backward(dy, x, wg, z, need_bias=True, stream=stream))

    want = run()
    torch.cuda.synchronize()
    got = run(side)
    side.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = run()
    for i in range(3):
        for t in static:
            t.zero_()
        x.add_(0.25)
        eager = run()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(eager, static)), i
