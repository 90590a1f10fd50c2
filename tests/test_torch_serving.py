"""torch.library operators and modules over the serving operators, the weights'
quantiser, and the C ABI's refusals (CPU: schemas, shapes, tracing, refusals
before any GPU call; GPU: results, graphs, the example)."""
import ctypes
import os
import sys

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import hipgemm_amd as hg
import hipgemm_amd.torch_serving as ts
from hipgemm_amd import serving
from w4util import ROUND, act64, agree, generator, weights64

INVALID = 1    # hipErrorInvalidValue
FAKE = 1 << 20  # an aligned address that nothing reads


def _w4_desc(**kw):
    d = dict(size=ctypes.sizeof(serving.W4Desc), x=FAKE, weight=FAKE, scales=FAKE,
             zeros=0, y=FAKE, bias=0, M=4, N=8, K=64, group_size=32, ldx=64, ldw=32,
             lds=2, ldy=8, x_type=1, format=0, scale_type=1, out_dtype=0, activation=0)
    d.update(kw)
    return serving.W4Desc(**d)


@pytest.mark.parametrize("bad", [
    dict(size=8), dict(M=-1), dict(N=-1), dict(K=-32), dict(K=48), dict(K=1 << 27),
    dict(group_size=0), dict(group_size=48), dict(x_type=0), dict(x_type=3),
    dict(format=2), dict(format=-1), dict(scale_type=4), dict(out_dtype=9),
    dict(activation=9), dict(format=1, zeros=FAKE), dict(x=0), dict(weight=0),
    dict(scales=0), dict(y=0), dict(x=FAKE + 8), dict(weight=FAKE + 8),
    dict(scales=FAKE + 1), dict(y=FAKE + 1), dict(bias=FAKE + 2), dict(ldx=56),
    dict(ldx=68), dict(ldw=16), dict(ldw=40), dict(ldw=1 << 26), dict(lds=1),
    dict(lds=1 << 26), dict(ldy=7)], ids=str)
def test_w4_refusals(bad):
    assert serving.w4_gemm_raw(_w4_desc(**bad)) == INVALID


def test_w4_nothing_to_do():
    assert serving.w4_gemm_raw(_w4_desc(M=0, x=0, y=0)) == 0
    assert serving.w4_gemm_raw(_w4_desc(N=0, weight=0, scales=0, y=0)) == 0
    assert hg.lib().hipgemm_w4_gemm(None, None) == INVALID


def _moe_desc(w13=None, w2=None, **kw):
    m13 = dict(weight=FAKE, scales=FAKE, zeros=0, ldw=64, expert_w=64 * 128, lds=1,
               expert_s=128)
    m2 = dict(weight=FAKE, scales=FAKE, zeros=0, ldw=64, expert_w=64 * 64, lds=1, expert_s=64)
    m13.update(w13 or {})
    m2.update(w2 or {})
    d = dict(size=ctypes.sizeof(serving.MoeDesc), x=FAKE, ids=FAKE, weights=FAKE, y=FAKE,
             workspace=FAKE, workspace_bytes=serving.moe_workspace_size(2, 2, 4, 64, 64),
             ldx=64, ldy=64, T=2, k=2, E=4, D=64, F=64, group_size=32, x_type=1, format=2,
             scale_type=0, out_dtype=0, activation=3)
    d.update(kw)
    return serving.MoeDesc(w13=serving.MoeMatrix(**m13), w2=serving.MoeMatrix(**m2), **d)


@pytest.mark.parametrize("bad", [
    dict(size=8), dict(T=-1), dict(k=0), dict(k=65), dict(E=0), dict(E=1025), dict(D=0),
    dict(D=48), dict(F=0), dict(F=80), dict(x_type=0), dict(format=3), dict(scale_type=1),
    dict(out_dtype=9), dict(activation=-1), dict(x=0), dict(ids=0), dict(weights=0),
    dict(y=0), dict(x=FAKE + 2), dict(ids=FAKE + 1), dict(workspace=0),
    dict(workspace=FAKE + 8), dict(workspace_bytes=16), dict(ldx=32), dict(ldx=68),
    dict(ldy=32), dict(w13=dict(weight=0)), dict(w13=dict(ldw=32)),
    dict(w2=dict(scales=0)), dict(w2=dict(ldw=72)), dict(format=0, group_size=16)], ids=str)
def test_moe_experts_refusals(bad):
    assert serving.moe_experts_raw(_moe_desc(**bad)) == INVALID


def test_moe_nothing_to_do():
    assert serving.moe_experts_raw(_moe_desc(T=0, x=0)) == 0
    assert serving.moe_workspace_size(0, 2, 4, 64, 64) == 0
    assert serving.moe_workspace_size(4, 2, 4, 64, 64) >= 4 * 2 * 64 * 4


@pytest.mark.parametrize("args", [
    dict(type=3), dict(type=-1), dict(T=-1), dict(E=0), dict(E=1025), dict(k=0),
    dict(k=65), dict(k=17), dict(ld=15), dict(scoring=2), dict(logits=0),
    dict(weights=0), dict(ids=0)], ids=str)
def test_moe_route_refusals(args):
    d = dict(logits=FAKE, type=0, T=2, E=16, k=2, ld=16, scoring=0, renorm=1, scale=1.0,
             weights=FAKE, ids=FAKE)
    d.update(args)
    assert hg.lib().hipgemm_moe_route(*d.values(), None) == INVALID


def test_fake_shapes_and_errors():
    op = torch.ops.hipgemm
    with FakeTensorMode():
        x = torch.empty(5, 96, dtype=torch.bfloat16)
        w, s = torch.empty(40, 48, dtype=torch.uint8), torch.empty(40, 3)
        y = op.w4_gemm(x, w, s, group_size=32)
        assert tuple(y.shape) == (5, 40) and y.dtype == torch.bfloat16
        assert op.w4_gemm(x, w, s, group_size=32, out_dtype=torch.float32).dtype == torch.float32
        for bad in (dict(group_size=64), dict(group_size=16), dict(group_size=32, format="int5"),
                    dict(group_size=32, activation="tanh")):
            with pytest.raises(hg.HipGemmError):
                op.w4_gemm(x, w, s, **bad)
        p, ids = op.moe_route(torch.empty(5, 8), 2)
        assert tuple(p.shape) == tuple(ids.shape) == (5, 2) and ids.dtype == torch.int32
        with pytest.raises(hg.HipGemmError):
            op.moe_route(torch.empty(5, 8), 2, scoring="max")
        f8 = torch.float8_e4m3fn
        args = (torch.empty(8, 128, 96, dtype=f8), torch.empty(8, 128),
                torch.empty(8, 96, 64, dtype=f8), torch.empty(8, 96))
        assert tuple(op.moe_experts(x, ids, p, *args).shape) == (5, 96)
        with pytest.raises(hg.HipGemmError):
            op.moe_experts(x, ids, p, *args, format="int4")


def test_modules_trace_as_operators():
    from torch.fx.experimental.proxy_tensor import make_fx
    lin = ts.W4Linear.from_linear(torch.nn.Linear(64, 40), group_size=32)
    moe = ts.MoE.from_weights(torch.randn(4, 64), torch.randn(4, 64, 64),
                              torch.randn(4, 64, 32), 2, "int4", 32)
    with FakeTensorMode(allow_non_fake_inputs=True) as mode, torch.no_grad():
        gm = make_fx(lambda x: moe(lin(x).new_empty(6, 64)), tracing_mode="fake")(
            mode.from_tensor(torch.randn(2, 3, 64).to(torch.bfloat16)))
    names = [str(n.target) for n in gm.graph.nodes if n.op == "call_function"]
    for op in ("w4_gemm", "moe_route", "moe_experts"):
        assert names.count(f"hipgemm.{op}.default") == 1, names


def test_modules_refuse():
    w, s = torch.zeros(8, 32, dtype=torch.uint8), torch.ones(8, 2)
    for kw in (dict(format="int5"), dict(activation="tanh"), dict(group_size=48),
               dict(group_size=64)):
        with pytest.raises(hg.HipGemmError):
            ts.W4Linear(w, s, **{"group_size": 32, **kw})
    g = torch.zeros(4, 64)
    with pytest.raises(hg.HipGemmError):
        ts.MoE.from_weights(g, torch.zeros(4, 64, 64), torch.zeros(4, 64, 32), 5)
    with pytest.raises(hg.HipGemmError):
        ts.MoE.from_weights(torch.zeros(3, 64), torch.zeros(4, 64, 64),
                            torch.zeros(4, 64, 32), 2)
    with pytest.raises(hg.HipGemmError):
        ts.quantize_w4(torch.zeros(4, 40))


@pytest.mark.parametrize("scale", [torch.float32, torch.bfloat16, torch.float16, torch.uint8],
                         ids=str)
@pytest.mark.parametrize("fmt,group,K", [("int4", 32, 96), ("int4", 64, 160), ("fp4", 32, 64),
                                         ("fp4", 128, 96)])
def test_quantize_w4_error(fmt, group, K, scale):
    """Within half a step of the grid at each weight, plus what the scale's own
    rounding takes from the largest (a clamped code)."""
    w = torch.randn(7, K, generator=torch.Generator().manual_seed(3))
    w[2] = 0
    q, s = ts.quantize_w4(w, fmt, group, scale)
    assert q.dtype == torch.uint8 and tuple(q.shape) == (7, K // 2)
    assert s.dtype == scale and tuple(s.shape) == (7, -(-K // group))
    got = weights64(q, s, fmt, group)
    amax = torch.nn.functional.pad(w, (0, -K % group)).unflatten(-1, (-1, group)).abs().amax(-1)
    amax = amax.double().repeat_interleave(group, -1)[:, :K]
    up = 2.0 if scale == torch.uint8 else 1 + 2.0 ** -8
    # int4: steps of s <= up amax / 7;  fp4: of 2 s at most
    half = 0.5 * up * amax / 7 if fmt == "int4" else up * amax / 6
    assert ((got - w.double()).abs() <= half + amax * 2.0 ** -8).all()
    assert (got[2] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("fmt", ["int4", "fp4"])
def test_w4_linear_gpu(fmt, dtype):
    g = generator(11)
    lin = torch.nn.Linear(160, 72, device="cuda", dtype=dtype)
    layer = ts.W4Linear.from_linear(lin, fmt, 32, torch.float32, activation="silu")
    w = weights64(layer.weight, layer.scales, fmt, 32)
    for shape in ((160,), (3, 160), (2, 5, 160)):
        x = torch.randn(shape, generator=g, device="cuda").to(dtype)
        x2 = x.reshape(-1, 160)
        with torch.no_grad():
            y = layer(x)
        assert y.shape == (*shape[:-1], 72) and y.dtype == dtype
        assert torch.equal(y.reshape(-1, 72), torch.ops.hipgemm.w4_gemm(
            x2, layer.weight, layer.scales, format=fmt, group_size=32, bias=layer.bias,
            activation="silu"))
        z = x2.double() @ w.T + layer.bias.double()
        # fp32 sums in any order: K + 2 roundings of the sum of magnitudes; SiLU's
        # slope is at most 1.1, its own error a few ulp.
        mag = x2.double().abs() @ w.abs().T + layer.bias.double().abs()
        agree(y.reshape(-1, 72), act64(z, "silu"), 1.1 * 162 * 2.0 ** -24 * mag + 2.0 ** -20 * z.abs())


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["e4m3", "int4", "fp4"])
@pytest.mark.parametrize("T", [1, 6])
def test_moe_gpu(fmt, T):
    g = generator(12)
    E, D, F, k = 8, 96, 64, 3
    rand = lambda *s: torch.randn(s, generator=g, device="cuda") * s[-1] ** -0.5
    moe = ts.MoE.from_weights(rand(E, D).bfloat16(), rand(E, 2 * F, D), rand(E, D, F), k, fmt,
                              32, torch.float32)
    x = torch.randn(2, T, D, generator=g, device="cuda").bfloat16()
    with torch.no_grad():
        y = moe(x)
    assert y.shape == x.shape and y.dtype == x.dtype
    x2 = x.reshape(-1, D)
    # the choice from the module's own logits, then all in 64 bits
    logits = torch.nn.functional.linear(x2, moe.gate)
    p = logits.double().softmax(-1)
    top, ids = p.topk(k, -1)
    top = top / top.sum(-1, keepdim=True)
    w13 = weights64(moe.w13, moe.scales13, fmt, 32)
    w2 = weights64(moe.w2, moe.scales2, fmt, 32)
    want = torch.zeros(2 * T, D, dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(want)
    for t in range(2 * T):
        for j in range(k):
            e = ids[t, j]
            a, b = (w13[e] @ x2[t].double()).chunk(2)
            h = act64(a, "silu") * b
            m = w13[e].abs() @ x2[t].double().abs()
            # error of h: sums of D terms, one rounding to 16 bits
            dh = (D + 4) * 2.0 ** -24 * (1.1 * m[:F] * b.abs() + a.abs() * m[F:]) \
                + 2.0 ** -16 * h.abs()
            want[t] += top[t, j] * (w2[e] @ h)
            mag[t] += top[t, j] * (w2[e].abs() @ (dh + (F + k + 8) * 2.0 ** -24 * h.abs()))
    agree(y.reshape(-1, D), want, mag + 1e-12)


@pytest.mark.gpu
def test_opcheck_gpu():
    g = generator(13)
    x = torch.randn(5, 64, generator=g, device="cuda").bfloat16()
    w, s = ts.quantize_w4(torch.randn(24, 64, device="cuda"), group_size=32)
    checks = ("test_schema", "test_faketensor")
    torch.library.opcheck(torch.ops.hipgemm.w4_gemm.default, (x, w, s, None, "int4", 32),
                          test_utils=checks)
    logits = torch.randn(5, 8, generator=g, device="cuda")
    torch.library.opcheck(torch.ops.hipgemm.moe_route.default, (logits, 2), test_utils=checks)
    p, ids = hg.moe_route(logits, 2)
    m = ts.MoE.from_weights(torch.randn(8, 64, device="cuda"), torch.randn(8, 64, 64, device="cuda"),
                            torch.randn(8, 64, 32, device="cuda"), 2, "int4", 32)
    torch.library.opcheck(torch.ops.hipgemm.moe_experts.default,
                          (x, ids, p, m.w13, m.scales13, m.w2, m.scales2, None, None, "int4", 32),
                          test_utils=checks)


@pytest.mark.gpu
def test_rows_far_apart_gpu():
    """Rows of x too far apart for one buffer's range go four at a time."""
    g = generator(14)
    M, K, N, ld = 6, 64, 40, (1 << 24) + 64
    x = torch.empty(M * ld, dtype=torch.bfloat16, device="cuda").as_strided((M, K), (ld, 1))
    x.copy_(torch.randn(M, K, generator=g, device="cuda"))
    w, s = ts.quantize_w4(torch.randn(N, K, generator=g, device="cuda"), group_size=32)
    got = hg.w4_gemm(x, w, s, group_size=32, out_dtype=torch.float32)
    w64 = weights64(w, s, "int4", 32)
    mag = x.double().abs() @ w64.abs().T
    agree(got, x.double() @ w64.T, (K + 2) * 2.0 ** -24 * mag)


@pytest.mark.gpu
def test_example_gpu():
    """The block of the example: eager against the formula, a graph of it against
    eager, replay by replay."""
    sys.path.insert(0, os.path.join(os.path.dirname(__file__), "..", "examples"))
    import moe_block
    with torch.no_grad():
        block = moe_block.Block(256, 160, 8, 2, group_size=32)
        step, x, y = moe_block.capture(block, 3, 256)
        for seed in (1, 2, 3):
            x.copy_(torch.randn(3, 256, generator=generator(seed), device="cuda"))
            want = block(x)
            step()
            torch.cuda.synchronize()
            assert torch.equal(y, want)
        # a prompt of the same tokens and others: the same rows
        w = {n: weights64(m.weight, m.scales, "int4", 32)
             for n, m in (("gate", block.gate), ("up", block.up), ("down", block.down))}
        x64 = x.double()
        r = lambda t: t.to(torch.bfloat16).double()
        h = r(r(act64(x64 @ w["gate"].T, "silu")) * r(x64 @ w["up"].T))
        plain = x64 + r(h @ w["down"].T) + block.moe(x).double()
        # four roundings to bf16 on the way, of values up to `size`; and h's three
        # through the product
        size = plain.abs() + x64.abs() + block.moe(x).double().abs() + (h @ w["down"].T).abs()
        bound = 4 * ROUND[torch.bfloat16] * size + 6 * ROUND[torch.bfloat16] * (
            h.abs() @ w["down"].abs().T)
        assert ((y.double() - plain).abs() <= bound).all()
