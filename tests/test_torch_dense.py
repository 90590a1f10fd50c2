"""torch.library operators, autograd and modules over linear and gated_linear (CPU: schemas,
shapes, tracing, refusals before any GPU call; GPU: gradients, strides, graphs, a block of both
together, the example)."""
import os
import sys

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import hipgemm_amd as hg
import hipgemm_amd.torch_dense as td
from denseutil import HALF, U, act64, check, gated64, linear64

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def test_fake_shapes():
    with FakeTensorMode():
        x = torch.empty(5, 64, dtype=BF, device="cuda", requires_grad=True)
        w = torch.empty(48, 64, dtype=BF, device="cuda", requires_grad=True)
        b = torch.empty(48, dtype=F32, device="cuda")
        r = torch.empty(5, 48, dtype=BF, device="cuda")
        y = torch.ops.hipgemm.linear(x, w, b, "relu", r)
        assert y.shape == (5, 48) and y.dtype == BF
        assert torch.ops.hipgemm.linear(x, w, out_dtype=F32).dtype == F32
        assert torch.ops.hipgemm.gated_linear(x, w).shape == (5, 24)
        y, pre = torch.ops.hipgemm.linear_with_pre(x, w, b, "silu", None, None, True)
        assert y.shape == (5, 24) and pre.shape == (5, 48) and pre.dtype == F32
        assert y.requires_grad
    x = torch.empty(5, 64, dtype=BF, device="meta", requires_grad=True)
    w = torch.empty(48, 64, dtype=BF, device="meta", requires_grad=True)
    b = torch.empty(48, dtype=F32, device="meta", requires_grad=True)
    g = torch.autograd.grad(td.gated_linear(x, w, b).sum(), (x, w, b))
    assert [(t.shape, t.dtype) for t in g] == [(t.shape, t.dtype) for t in (x, w, b)]


@pytest.mark.parametrize("call", [
    lambda x, w: td.linear(x, w[:, :32]),
    lambda x, w: td.linear(x, w, activation="tanh"),
    lambda x, w: td.linear(x, w, bias=torch.zeros(47, device="meta")),
    lambda x, w: td.linear(x, w, residual=torch.zeros(5, 47, device="meta")),
    lambda x, w: td.gated_linear(x, w[:40]),
    lambda x, w: td.DenseLinear(60, 8, device="meta"),
    lambda x, w: td.DenseLinear(64, 8, activation="tanh", device="meta"),
    lambda x, w: td.DenseLinear(128, 8, device="meta")(x),
    lambda x, w: td.GatedMLP(64, 60, device="meta"),
    lambda x, w: td.GatedMLP(128, 64, device="meta")(x),
])
def test_refusals(call):
    x = torch.empty(5, 64, dtype=BF, device="meta")
    w = torch.empty(48, 64, dtype=BF, device="meta")
    with pytest.raises(hg.HipGemmError):
        call(x, w)


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(4, 64, dtype=BF), torch.zeros(32, 64, dtype=BF)
    with pytest.raises(hg.HipGemmError):
        td.linear(x, w)
    with pytest.raises(hg.HipGemmError):
        td.gated_linear(x, w.requires_grad_())


def leaves(M, N, K, dtype, gated, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0, t=dtype):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(t).requires_grad_()

    rows = 2 * N if gated else N
    return (normal(M, K), normal(rows, K, std=K ** -0.5), normal(rows, std=0.3, t=F32),
            normal(M, N))


def reference(x, w, b, r, act, gated, dy):
    """Gradients in 64 bits, and bounds: dz rounded to the operands' type (half a step), sums of
    fp32 products, z's fp32 error times the slope's slope (2 at most)."""
    ts = [t.detach().double().requires_grad_() for t in (x, w, b, r)]
    z = ts[0] @ ts[1].t() + ts[2]
    if gated:
        n = z.shape[1] // 2
        y = act64(z[:, :n], act) * z[:, n:] + ts[3]
    else:
        y = act64(z, act) + ts[3]
    dz, *g = torch.autograd.grad(y, [z, *ts], dy.double())
    h = HALF[x.dtype]
    e = dz.abs() * h + 64 * U * (dy.double().abs().amax() + dz.abs())
    X, W = ts[0].detach().abs(), ts[1].detach().abs()
    ex = e @ W + (W.shape[0] + 1) * U * (dz.abs() @ W)
    ew = e.t() @ X + (X.shape[0] + 1) * U * (dz.abs().t() @ X)
    eb = 64 * U * (dz.abs() + dy.double().abs().amax()).sum(0) * 2
    return g, [ex + h * (g[0].abs() + ex), ew + h * (g[1].abs() + ew), eb + U * g[2].abs(),
               h * g[3].abs()]


@pytest.mark.gpu
@pytest.mark.parametrize("gated", (False, True), ids=("linear", "gated"))
@pytest.mark.parametrize("act", (None, "silu", "gelu_tanh"))
@pytest.mark.parametrize("M,N,K", [(1, 8, 8), (37, 56, 72), (130, 264, 136)])
def test_gradients(gpu, gated, act, M, N, K):
    for dtype in (BF, HF):
        x, w, b, r = leaves(M, N, K, dtype, gated)
        dy = torch.randn(M, N, device="cuda").to(dtype)
        if gated:
            y = td.gated_linear(x, w, b, act) + r
        else:
            y = td.linear(x, w, b, act, residual=r)
        got = torch.autograd.grad(y, (x, w, b, r), dy)
        want, bound = reference(x, w, b, r, act, gated, dy)
        for name, t, a, e, leaf in zip(("dx", "dw", "db", "dr"), got, want, bound, (x, w, b, r)):
            assert t.dtype == leaf.dtype and t.shape == leaf.shape
            check(f"{name} {act}", t, a, e)


@pytest.mark.gpu
def test_some_leaves_only(gpu):
    x, w, b, r = leaves(20, 48, 64, BF, False)
    dy = torch.randn(20, 48, device="cuda").to(BF)
    full = torch.autograd.grad(td.linear(x, w, b, "silu", r), (x, w, b, r), dy)
    for i in range(4):
        ts = [t.detach() for t in (x, w, b, r)]
        ts[i].requires_grad_()
        y = td.linear(ts[0], ts[1], ts[2], "silu", ts[3])
        got, = torch.autograd.grad(y, ts[i], dy)
        assert torch.equal(got, full[i])
    with torch.no_grad():
        assert not td.linear(x, w, b, "silu", r).requires_grad
    # a gradient that comes broadcast, and one in another layout
    y = td.linear(x, w, b, "silu", r)
    one, = torch.autograd.grad(y.sum(), x, retain_graph=True)
    same, = torch.autograd.grad(y, x, torch.ones(48, 20, device="cuda", dtype=BF).t())
    assert torch.equal(one, same)


@pytest.mark.gpu
def test_strides_and_shapes(gpu):
    """Views that the kernels do not take are copied; leading dimensions come back."""
    g = torch.Generator(device="cuda").manual_seed(3)
    big = torch.randn(6, 9, 80, generator=g, device="cuda").to(BF)
    x = big[:, ::2, 3:67]
    w = torch.randn(64, 48, generator=g, device="cuda").to(BF).t()
    b = torch.randn(96, generator=g, device="cuda").to(BF)[::2]
    r = torch.randn(48, 6, 5, generator=g, device="cuda").to(BF).permute(1, 2, 0)
    y = td.linear(x, w, b, "relu", r)
    assert y.shape == (6, 5, 48)
    _, _, want, bound = linear64(x.reshape(-1, 64), w.contiguous(), b.contiguous(), "relu",
                                 r.reshape(-1, 48), BF)
    check("y", y.reshape(-1, 48), want, bound)
    h = td.gated_linear(x, w, b)
    assert h.shape == (6, 5, 24)
    _, _, want, bound = gated64(x.reshape(-1, 64), w.contiguous(), b.contiguous(), "silu", BF)
    check("h", h.reshape(-1, 24), want, bound)
    m = td.DenseLinear.from_linear(torch.nn.Linear(64, 48, device="cuda", dtype=BF), "silu")
    assert m(x).shape == (6, 5, 48) and m(x[0, 0]).shape == (48,)


@pytest.mark.gpu
def test_block(gpu):
    """gated_linear, then linear with the residual: the block's output and its gradients,
    against 64 bits with h rounded where the block rounds it."""
    torch.manual_seed(0)
    dim, hidden, M = 136, 264, 75
    block = td.GatedMLP(dim, hidden, device="cuda")
    x = torch.randn(M, dim, device="cuda").to(BF).requires_grad_()
    y = block(x, residual=x)
    with torch.no_grad():
        _, _, h64, eh = gated64(x, block.w13, None, "silu", BF)
        h = td.gated_linear(x, block.w13)
        check("h", h, h64, eh)
        _, _, want, bound = linear64(h, block.w2, None, None, x, BF)
        check("y", y, want, bound)
    dy = torch.randn(M, dim, device="cuda").to(BF)
    dx, dw13, dw2 = torch.autograd.grad(y, (x, block.w13, block.w2), dy)
    # the parts, one call each, make the same gradients
    dh, dw2b, _ = hg.linear_backward(dy, h, block.w2.detach())
    _, pre = hg.gated_linear(x.detach(), block.w13.detach(), save_pre=True)
    dxb, dw13b, _ = hg.gated_linear_backward(dh, x.detach(), block.w13.detach(), pre)
    assert torch.equal(dw2, dw2b) and torch.equal(dw13, dw13b)
    assert torch.equal(dx, dxb + dy)


@pytest.mark.gpu
def test_captured_step(gpu):
    """A training step of a block in a graph: each replay gives the eager step's gradients, also
    while an eager graph of the same parameters lives."""
    torch.manual_seed(1)
    block = td.GatedMLP(128, 256, device="cuda")
    x = torch.randn(64, 128, device="cuda").to(BF)
    dy = torch.randn(64, 128, device="cuda").to(BF)

    # Leaves of the captured pass' own, over the same memory: capturing a backward pass into
    # leaves that an eager graph alive has too ends the process inside torch.
    w13, w2 = (p.detach().requires_grad_() for p in (block.w13, block.w2))

    def step():
        y = td.linear(td.gated_linear(x, w13), w2, residual=x)
        return (y, *torch.autograd.grad(y, (w13, w2), dy))

    alive = block(x, residual=x)  # an eager graph of the block's own leaves
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()
    for _ in range(3):
        with torch.no_grad():
            x.mul_(0.5)
            block.w2.add_(0.01)
        eager = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, static))
    assert alive.requires_grad


@pytest.mark.gpu
def test_example(gpu):
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    try:
        import train_block as ex
    finally:
        sys.path.pop(0)
    block, goal = ex.make(64, 128, 0), ex.make(64, 128, 1)
    x = torch.randn(96, 64, device="cuda").to(BF)
    with torch.no_grad():
        target = goal(x, residual=x)
    loss, grads = ex.gradients(block, x, target)
    # the same loss in 64 bits: within the roundings of y (2^-8) and of h through w2
    w13, w2, x64 = block.w13.detach().double(), block.w2.detach().double(), x.double()
    w13.requires_grad_(), w2.requires_grad_()
    z = x64 @ w13.t()
    y = x64 + (act64(z[:, :128], "silu") * z[:, 128:]) @ w2.t()
    want = (y - target.double()).square().mean()
    g = torch.autograd.grad(want, (w13, w2))
    # Rounding errors are independent: relative to the whole gradient each of the six
    # roundings on its way (y, dy, dh, dz, h, the gradient) is 2^-8 at most; y's is relative to
    # y, and the difference from the target is smaller than y.
    room = 2.0 ** -8 * float(y.detach().norm() / (y.detach() - target.double()).norm()) + 5 * 2.0 ** -8
    assert abs(float(loss) - float(want)) <= 2 * room * float(want)
    for a, b in zip(grads, g):
        assert float((a.double() - b).norm()) <= room * float(b.norm())
    assert len(ex.train(block, x, target, 3)) == 3
    step, sx, sy = ex.capture(block, 64)
    sx.copy_(x[:1])
    for _ in range(2):
        step()
        with torch.no_grad():
            assert torch.equal(sy, block(x[:1], residual=x[:1]))


def test_leading_dimensions():
    """Those of the residual are x's own, not any that hold as many rows."""
    w = torch.empty(48, 64, dtype=BF, device="meta")
    x = torch.empty(2, 3, 64, dtype=BF, device="meta")
    for shape in ((3, 2, 48), (6, 48), (1, 3, 48)):
        with pytest.raises(hg.HipGemmError, match="residual"):
            td.linear(x, w, residual=torch.empty(shape, dtype=BF, device="meta"))
    r = torch.empty(2, 3, 48, dtype=BF, device="meta")
    assert td.linear(x, w, residual=r).shape == (2, 3, 48)
    assert td.linear(x[0, 0], w, residual=torch.empty(48, dtype=BF, device="meta")).shape == (48,)
    # and of no elements
    for lead, k in (((0, 3), 64), ((2, 0), 64), ((2, 3), 0)):
        y = td.gated_linear(torch.empty(*lead, k, dtype=BF, device="meta"), w[:, :k])
        assert y.shape == (*lead, 24)


def test_differentiable_once():
    x = torch.empty(5, 64, dtype=BF, device="meta", requires_grad=True)
    w = torch.empty(48, 64, dtype=BF, device="meta", requires_grad=True)
    g, = torch.autograd.grad(td.gated_linear(x, w).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), w)
