"""w4_gemm against its definition in 64 bits.

Tolerance: the output type's rounding, and fp32's on the sums.  A term passes
through the additions of its lane's 32, of its group, of the blocks of K (one in
128), of lanes and of waves: fewer than K / 128 + 64 roundings of 2^-24 of the
sum of magnitudes.  int4's magnitudes are those of the shifted codes (q + 128
and z + 128, so q + z + 256 at most).  Activations change by at most 1.13 times
the change of their argument, and carry 8 roundings of their own.
"""
import pytest
import torch

import w4util as u

pytestmark = pytest.mark.gpu


def plain(x, w, s, z, fmt, group, bias, act):
    wd = u.weights64(w, s, fmt, group, z)
    v = x.double() @ wd.t()
    if bias is not None:
        v = v + bias.double()
    q = u.unpack(w).double()
    mag = (q + (8 if z is None else z.double().repeat_interleave(group, 1)[:, :q.shape[1]])
           + 256 if fmt == "int4" else u.codes64(w, fmt, None, group).abs())
    mag = mag * u.scales64(s).abs().repeat_interleave(group, 1)[:, :q.shape[1]]
    slack = (x.double().abs() @ mag.t()) * ((x.shape[1] / 128 + 64) * 2.0 ** -24)
    if bias is not None:
        slack = slack + (v.abs() + bias.double().abs()) * 2.0 ** -24
    y = u.act64(v, act)
    if act not in (None, "none"):
        slack = 1.13 * slack + 8 * 2.0 ** -24 * y.abs()
    return y, slack


def case(hg, M, N, K, fmt="int4", group=128, scale="bfloat16", zeros=False,
         dtype="bfloat16", bias=False, act=None, out_dtype=None, seed=0, x=None, **kw):
    g = u.generator(seed)
    if x is None:
        x = torch.randn((M, K), generator=g, device="cuda").to(getattr(torch, dtype))
    w, s, z = u.four_bit(g, (N,), K, fmt, group, scale, zeros)
    b = torch.randn(N, generator=g, device="cuda") if bias else None
    y = hg.w4_gemm(x, w, s, z, format=fmt, group_size=group, bias=b, activation=act,
                   out_dtype=out_dtype, **kw)
    assert y.shape == (M, N) and y.dtype == (out_dtype or x.dtype)
    want, slack = plain(x, w, s, z, fmt, group, b, act)
    u.agree(y, want, slack)
    return y


@pytest.fixture()
def hg(gpu):
    import hipgemm_amd
    return hipgemm_amd


SHAPES = [(1, 1, 32), (1, 7, 64), (1, 4096, 4096), (2, 33, 2336), (3, 100, 1056),
          (4, 129, 8192), (5, 48, 96), (7, 31, 128), (16, 64, 4128), (17, 100, 256),
          (33, 65, 1952), (64, 32, 160), (65, 70, 512), (100, 130, 2080), (1, 300, 28672),
          (16, 40, 14336), (129, 257, 384), (300, 200, 1184)]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("fmt", ["int4", "fp4"])
def test_shapes(hg, M, N, K, fmt):
    case(hg, M, N, K, fmt, zeros=fmt == "int4" and N % 2 == 0, seed=M + N + K)


# Columns enough for tiles of 32, 48 and 64 rows, of 32 columns and of 64.
@pytest.mark.parametrize("M,N", [(20, 4104), (37, 5000), (20, 8200), (40, 8200), (64, 4100),
                                 (64, 8216), (90, 8200)])
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("fmt,scale", [("int4", "bfloat16"), ("fp4", "e8m0"), ("fp4", "float16")])
def test_tall_tiles(hg, M, N, group, fmt, scale):
    for dtype, zeros in (("bfloat16", False), ("float16", fmt == "int4")):
        case(hg, M, N, 1120, fmt, group, scale, zeros, dtype, seed=M + N)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("scale", ["bfloat16", "float16", "float32", "e8m0"])
@pytest.mark.parametrize("group", [32, 64, 96, 128, 256, 4096])
@pytest.mark.parametrize("M", [1, 4, 9, 40, 140])
def test_groups_and_types(hg, M, group, scale, dtype):
    for fmt in ("int4", "fp4"):
        # 1120 = 8 blocks of 128 and 96: a short last group for most sizes
        case(hg, M, 72, 1120, fmt, group, scale, fmt == "int4", dtype, seed=group + M)


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu_tanh"])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M", [1, 3, 20, 150])
def test_epilogue(hg, M, out, act):
    case(hg, M, 95, 512, bias=True, act=act, out_dtype=out, zeros=True, seed=M)
    case(hg, M, 95, 512, "fp4", act=act, out_dtype=out, dtype="float16", seed=M)


@pytest.mark.parametrize("M", [1, 4, 6, 50, 200])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_strides_and_guards(hg, M, dtype):
    """Rows inside wider tensors; nothing written outside the output's window."""
    g = u.generator(M)
    N, K = 77, 416
    x = torch.randn((M, K + 40), generator=g, device="cuda").to(getattr(torch, dtype))[:, 8:8 + K]
    w, s, z = u.four_bit(g, (N,), K, "int4", 64, "float16", True, pad=48)
    ss = torch.full((N, s.shape[1] + 3), 7.0, device="cuda", dtype=torch.float16)
    ss[:, :s.shape[1]] = s
    big = torch.full((M + 2, N + 5), -77.0, device="cuda", dtype=x.dtype)
    out = big[1:1 + M, 2:2 + N]
    hg.w4_gemm(x, w, ss[:, :s.shape[1]], z, group_size=64, out=out)
    want, slack = plain(x, w, s, z, "int4", 64, None, None)
    u.agree(out.contiguous(), want, slack)
    keep = torch.ones_like(big, dtype=torch.bool)
    keep[1:1 + M, 2:2 + N] = False
    assert bool((big[keep] == -77.0).all())


@pytest.mark.parametrize("M", [1, 2, 5, 40, 140])
@pytest.mark.parametrize("fmt", ["int4", "fp4"])
def test_infinities_and_nan(hg, M, fmt):
    """An infinite activation gives infinities (NaN where its weight is 0), a NaN
    one NaN, as the products do; other rows are untouched by it."""
    g = u.generator(7)
    K, N = 512, 64
    x = torch.randn((M, K), generator=g, device="cuda").bfloat16()
    x[0, 300] = float("inf")
    if M > 1:
        x[M - 1, 5] = float("nan")
    w, s, z = u.four_bit(g, (N,), K, fmt, 128, "bfloat16", False)
    y = hg.w4_gemm(x, w, s, z, format=fmt)
    wd = u.weights64(w, s, fmt, 128, z)
    col = wd[:, 300]
    assert torch.equal(torch.isnan(y[0]), col == 0)
    assert torch.equal(y[0].double()[col != 0], torch.sign(col[col != 0]) * float("inf"))
    if M > 1:
        assert bool(torch.isnan(y[M - 1]).all())
    if M > 2:
        want, slack = plain(x[1:M - 1], w, s, z, fmt, 128, None, None)
        u.agree(y[1:M - 1], want, slack)


@pytest.mark.parametrize("M", [1, 3, 9, 150])
@pytest.mark.parametrize("fmt", ["int4", "fp4"])
def test_large_activations(hg, M, fmt):
    """Activations whose product with an unscaled code overflows fp32, while the
    results do not."""
    g = u.generator(3)
    K, N = 256, 40
    x = torch.zeros((M, K), device="cuda", dtype=torch.bfloat16)
    x[:, 17] = 2.0 ** 126
    x[:, 100] = -2.0 ** 125
    w, s, z = u.four_bit(g, (N,), K, fmt, 64, "bfloat16", fmt == "int4")
    y = hg.w4_gemm(x, w, s, z, format=fmt, group_size=64)
    wd = u.weights64(w, s, fmt, 64, z)
    u.agree(y, x.double() @ wd.t(), (x.double().abs() @ wd.t().abs()) * 4 * 2.0 ** -24)


def test_e8m0_ends(hg):
    """2^-127 (byte 0) is a number, 255 is NaN."""
    for M in (1, 8):
        for dtype in (torch.bfloat16, torch.float16):
            x = torch.zeros((M, 64), device="cuda", dtype=dtype)
            x[:, 3] = 2.0 ** 15
            w = torch.full((3, 32), 0x77, device="cuda", dtype=torch.uint8)  # 6.0
            s = torch.tensor([[0, 127], [255, 127], [127, 127]], device="cuda",
                             dtype=torch.uint8)
            y = hg.w4_gemm(x, w, s, format="fp4", group_size=32, out_dtype=torch.float32)
            assert bool(torch.isnan(y[:, 1]).all())
            assert bool((y[:, 2] == 6.0 * 2 ** 15).all())
            assert bool((y[:, 0] == 6.0 * 2.0 ** (15 - 127)).all()), y[:, 0]


def test_empty(hg):
    for M, N, K in ((0, 8, 64), (3, 0, 64), (2, 5, 0), (30, 5, 0)):
        x = torch.empty((M, K), device="cuda", dtype=torch.bfloat16)
        w = torch.empty((N, K // 2), device="cuda", dtype=torch.uint8)
        s = torch.empty((N, -(-K // 128)), device="cuda", dtype=torch.bfloat16)
        b = torch.arange(N, device="cuda", dtype=torch.float32)
        y = hg.w4_gemm(x, w, s, bias=b)
        assert y.shape == (M, N)
        assert torch.equal(y, b.bfloat16().expand(M, N))


def test_other_stream_and_graph(hg):
    g = u.generator(11)
    w, s, z = u.four_bit(g, (512,), 1024, "int4", 128, "bfloat16", True)
    side = torch.cuda.Stream()
    for M in (1, 12, 150):
        x = torch.randn((M, 1024), generator=g, device="cuda").bfloat16()
        ref = hg.w4_gemm(x, w, s, z)
        out = torch.zeros_like(ref)
        side.wait_stream(torch.cuda.current_stream())
        hg.w4_gemm(x, w, s, z, out=out, stream=side)
        torch.cuda.synchronize()
        assert torch.equal(out, ref)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = hg.w4_gemm(x, w, s, z)
        for seed in range(3):
            x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
            ref = hg.w4_gemm(x, w, s, z)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, ref)


def test_repeats_are_equal(hg):
    g = u.generator(5)
    w, s, z = u.four_bit(g, (1000,), 4096, "int4", 32, "float16", True)
    for M in (1, 16, 200):
        x = torch.randn((M, 4096), generator=g, device="cuda").half()
        a, b = (hg.w4_gemm(x, w, s, z, group_size=32) for _ in range(2))
        assert torch.equal(a, b)


@pytest.mark.parametrize("change", [
    dict(x=lambda t: t.float()), dict(x=lambda t: t[0]), dict(x=lambda t: t[:, :96]),
    dict(x=lambda t: t.cpu()), dict(x=lambda t: t.t().contiguous().t()),
    dict(w=lambda t: t.int()), dict(w=lambda t: t.cpu()), dict(w=lambda t: t[:, 1:]),
    dict(w=lambda t: t.t().contiguous().t()),
    dict(s=lambda t: t.double()), dict(s=lambda t: t[:, :1]), dict(s=lambda t: t[1:]),
    dict(z=lambda t: t.int()), dict(z=lambda t: t[1:]), dict(z=lambda t: t.cpu()),
    dict(group_size=48), dict(group_size=0), dict(group_size=-32),
    dict(format="int8"), dict(activation="tanh"), dict(out_dtype=torch.float64),
    dict(bias=torch.zeros(3)), dict(format="fp4"),
])
def test_refusals(hg, change):
    g = u.generator(1)
    a = dict(x=torch.zeros((4, 128), device="cuda", dtype=torch.bfloat16))
    a["w"], a["s"], a["z"] = u.four_bit(g, (6,), 128, "int4", 64, "bfloat16", True)
    kw = dict(group_size=64)
    hg.w4_gemm(a["x"], a["w"], a["s"], a["z"], **kw)
    for k, f in change.items():
        if k in a:
            a[k] = f(a[k])
        else:
            kw[k] = f
    with pytest.raises(hg.HipGemmError):
        hg.w4_gemm(a["x"], a["w"], a["s"], a["z"], **kw)


def test_refuses_misaligned_rows(hg):
    g = u.generator(1)
    w, s, z = u.four_bit(g, (6,), 128, "int4", 128, "bfloat16", True)
    x = torch.zeros((4, 132), device="cuda", dtype=torch.bfloat16)
    for bad in (x[:, :128], torch.zeros(4 * 128 + 4, device="cuda",
                                        dtype=torch.bfloat16)[4:].view(4, 128)):
        with pytest.raises(hg.HipGemmError):
            hg.w4_gemm(bad, w, s, z)
