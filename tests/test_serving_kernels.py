"""The kernels behind w4_gemm and moe_experts that sizes choose: each test names the
kernel that it is about and asks the library (w4_select, moe_select) whether its
sizes reach it, so that a rule that changes does not leave a kernel untested.

Oracles and tolerances as in test_w4_gpu.py and test_moe_experts_gpu.py."""
import ctypes

import pytest
import torch

import hipgemm_amd as hg
import w4util as u
from hipgemm_amd import serving
from test_moe_experts_gpu import check, make, plain as moe_plain
from test_w4_gpu import case, plain

gpu_test = pytest.mark.gpu
FAKE = 1 << 20


def w4_kernel(M, N, K, ldx=None, group=128):
    d = serving.W4Desc(size=ctypes.sizeof(serving.W4Desc), x=FAKE, weight=FAKE, scales=FAKE,
                       y=FAKE, M=M, N=N, K=K, group_size=group, ldx=ldx or K, ldw=K // 2,
                       lds=-(-K // group), ldy=N, x_type=1, scale_type=1)
    return hg.w4_select(d)


# ---- which kernels (no GPU) ------------------------------------------------

# 128 x 128 tiles: ragged rows and columns, fewer tiles than workgroups and more.
TILES = [(97, 28600, 160), (193, 12300, 1120), (300, 10300, 96), (1030, 7400, 32),
         (1100, 2700, 416)]
# As many of the large tiles, and nearly as many, that run on the split kernel's.
NEAR = [(97, 24500, 160), (129, 12300, 1120), (300, 8200, 96), (129, 16600, 224)]
# Tiles of 16 rows of 64 columns, and of each height.
SPLIT = [((5, 8200, 1120), 16, 64), ((16, 8300, 160), 16, 64), ((11, 16400, 32), 16, 64),
         ((7, 100, 416), 16, 32), ((20, 8200, 544), 32, 64), ((37, 5000, 160), 48, 32),
         ((40, 8200, 96), 48, 64), ((64, 4100, 416), 64, 32), ((90, 8200, 160), 48, 64),
         ((64, 8216, 32), 64, 64)]
# moe_experts grouped: (T, E, k, D, F).
GROUPED = [(40, 3, 2, 1056, 608), (12, 3, 2, 2080, 1120), (24, 2, 2, 4128, 544),
           (64, 5, 4, 416, 1312), (300, 3, 2, 1056, 608), (9, 8, 2, 544, 8224),
           (20, 2, 2, 96, 18592), (64, 24, 6, 512, 384), (33, 2, 2, 8192, 128),
           (14, 16, 2, 2080, 2336)]
# Where LDS holds one row of x (the widest model) and where it holds a few; the widest
# expert.
LIMITS = [(20, 1, 1, 37120, 64), (20, 1, 1, 28960, 96), (9, 2, 2, 96, 65536),
          (8, 1, 1, 128, 65504)]


def moe_kernels(size, fmt):
    T, E, k, D, F = size
    return hg.moe_select(T, k, E, D, F, fmt)


def test_sizes_reach_their_kernels():
    for M, N, K in TILES:
        assert w4_kernel(M, N, K) == ("tiles", 128, 128)
    assert any(-(-M // 128) * -(-N // 128) > 512 for M, N, K in TILES)
    for size in NEAR:
        assert w4_kernel(*size)[0] == "split"
    for size, rows, columns in SPLIT:
        assert w4_kernel(*size) == ("split", rows, columns), size
    assert w4_kernel(4, 8200, 64)[0] == w4_kernel(40, 100, 0, 64)[0] == "vectors"
    assert w4_kernel(40, 100, 64, (1 << 24) + 64)[0] == "vectors"
    for fmt in ("e4m3", "int4"):
        plans = [moe_kernels(s, fmt) for s in GROUPED]
        assert all(plans), [s for s, p in zip(GROUPED, plans) if not p]
        for name, values in (("up_rows", {16, 32}), ("up_waves", {2, 8}), ("down_rows", {16, 32}),
                             ("down_waves", {2, 8})):
            assert {p[name] for p in plans} == values, (fmt, name)
        assert min(p["parts"] for p in plans) == 1 and max(p["parts"] for p in plans) > 8
        assert all(moe_kernels(s, fmt) for s in LIMITS)
    assert any(T * k > 512 for T, E, k, D, F in GROUPED)
    assert hg.moe_select(1, 2, 8, 256, 512) == {} == hg.moe_select(6, 1, 1, 37152, 32)


def test_select_refuses():
    d = serving.W4Desc(size=8)
    with pytest.raises(hg.HipGemmError):
        hg.w4_select(d)
    assert hg.lib().hipgemm_w4_select(None, None) == 1
    for bad in ((0, 1, 2, 64, 64), (1, 0, 2, 64, 64), (1, 65, 2, 64, 64), (1, 1, 0, 64, 64),
                (1, 1, 1025, 64, 64), (1, 1, 2, 48, 64), (1, 1, 2, 64, 0)):
        with pytest.raises(hg.HipGemmError):
            hg.moe_select(*bad)
    with pytest.raises(hg.HipGemmError):
        hg.moe_select(1, 2, 1, 64, 64, "int8")


# ---- products of many rows --------------------------------------------------

@gpu_test
@pytest.mark.parametrize("M,N,K", TILES + NEAR)
@pytest.mark.parametrize("group", [32, 96, 128, 256])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_w4_tiles(gpu, M, N, K, group, dtype):
    for fmt, zeros, scales in (("int4", False, ("bfloat16", "float32", "e8m0")),
                               ("int4", True, ("float16", "float32", "e8m0")),
                               ("fp4", False, ("bfloat16", "float16", "float32", "e8m0"))):
        for scale in scales:
            case(hg, M, N, K, fmt, group, scale, zeros, dtype, seed=M + group)


@gpu_test
@pytest.mark.parametrize("size,rows,columns", SPLIT)
@pytest.mark.parametrize("group", [32, 96, 128])
def test_w4_split(gpu, size, rows, columns, group):
    for fmt, zeros, scale, dtype in (("int4", False, "bfloat16", "bfloat16"),
                                     ("int4", True, "float32", "float16"),
                                     ("int4", True, "e8m0", "bfloat16"),
                                     ("fp4", False, "e8m0", "bfloat16"),
                                     ("fp4", False, "float16", "float16")):
        case(hg, *size, fmt, group, scale, zeros, dtype, seed=size[0])


@gpu_test
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu_tanh"])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float16, torch.float32])
def test_w4_tiles_epilogue(gpu, out, act):
    for M, N in ((129, 12300), (193, 12300)):
        case(hg, M, N, 512, bias=True, act=act, out_dtype=out, zeros=True, seed=1)
    for M, N in ((300, 8200), (300, 10300)):
        case(hg, M, N, 224, "fp4", 32, "e8m0", bias=True, act=act, out_dtype=out, seed=2)


@gpu_test
@pytest.mark.parametrize("M,N", [(129, 12300), (193, 12300), (1100, 2700), (13, 8300)])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_w4_strides_and_guards(gpu, M, N, dtype):
    """Rows inside wider tensors; nothing written outside the output's window."""
    g = u.generator(M)
    K = 416
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


@gpu_test
@pytest.mark.parametrize("M", [129, 193])
@pytest.mark.parametrize("fmt", ["int4", "fp4"])
def test_w4_tiles_large_activations(gpu, fmt, M):
    """Activations whose product with an unscaled code overflows fp32, while the
    results do not."""
    g = u.generator(3)
    N, K = 12300, 256
    x = torch.zeros((M, K), device="cuda", dtype=torch.bfloat16)
    x[:, 17] = 2.0 ** 126
    x[:, 100] = -2.0 ** 125
    w, s, z = u.four_bit(g, (N,), K, fmt, 64, "bfloat16", fmt == "int4")
    y = hg.w4_gemm(x, w, s, z, format=fmt, group_size=64)
    wd = u.weights64(w, s, fmt, 64, z)
    u.agree(y, x.double() @ wd.t(), (x.double().abs() @ wd.t().abs()) * 4 * 2.0 ** -24)


@gpu_test
@pytest.mark.parametrize("M,N", [(129, 12300), (193, 12300), (1030, 7400), (16, 8300)])
def test_w4_stream_graph_and_repeats(gpu, M, N):
    g = u.generator(11)
    w, s, z = u.four_bit(g, (N,), 1024, "int4", 128, "bfloat16", True)
    x = torch.randn((M, 1024), generator=g, device="cuda").bfloat16()
    ref = hg.w4_gemm(x, w, s, z)
    assert torch.equal(hg.w4_gemm(x, w, s, z), ref)
    side = torch.cuda.Stream()
    out = torch.zeros_like(ref)
    side.wait_stream(torch.cuda.current_stream())
    hg.w4_gemm(x, w, s, z, out=out, stream=side)
    torch.cuda.synchronize()
    assert torch.equal(out, ref)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = hg.w4_gemm(x, w, s, z)
    for _ in range(3):
        x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        ref = hg.w4_gemm(x, w, s, z)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ref)


# ---- experts, grouped --------------------------------------------------------

@gpu_test
@pytest.mark.parametrize("T,E,k,D,F", GROUPED + LIMITS)
@pytest.mark.parametrize("fmt,zeros", [("e4m3", False), ("int4", False), ("int4", True),
                                       ("fp4", False)])
def test_experts(gpu, T, E, k, D, F, fmt, zeros):
    check(hg, make(T + E + k, T, E, k, D, F, fmt, zeros=zeros), fmt)


@gpu_test
@pytest.mark.parametrize("size", GROUPED + LIMITS)
@pytest.mark.parametrize("fmt", ["e4m3", "int4", "fp4"])
def test_experts_float32(gpu, size, fmt):
    """h in three parts: fewer rows of it in LDS, more parts of F."""
    T, E, k, D, F = size
    assert hg.moe_select(T, k, E, D, F, fmt, torch.float32)
    for group in (128,) if fmt == "e4m3" else (32, 128):
        check(hg, make(T + E + k, *size, fmt, group, "e8m0" if fmt == "fp4" else "float16"), fmt,
              group, out_dtype=torch.float32)


@gpu_test
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("scale", ["bfloat16", "float16", "float32", "e8m0"])
@pytest.mark.parametrize("group", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("T,E,k,D,F", [GROUPED[0], GROUPED[1]])
def test_experts_groups_and_types(gpu, T, E, k, D, F, group, scale, dtype):
    for fmt, zeros in (("int4", False), ("int4", True), ("fp4", False)):
        check(hg, make(group, T, E, k, D, F, fmt, group, scale, zeros, dtype), fmt, group)


@gpu_test
@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu_tanh"])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("fmt", ["e4m3", "int4", "fp4"])
def test_experts_epilogue(gpu, act, out, fmt):
    a = make(3, *GROUPED[0], fmt, dtype="float16" if fmt == "fp4" else "bfloat16")
    check(hg, a, fmt, act=act, out_dtype=out)


@gpu_test
@pytest.mark.parametrize("fmt", ["e4m3", "int4", "fp4"])
def test_experts_skipped_and_repeated_ids(gpu, fmt):
    """Ids outside [0, E) contribute nothing; one expert for all tokens, twice each."""
    a = make(9, *GROUPED[0], fmt)
    a["ids"][0] = -1
    a["ids"][1, 1] = 3
    a["ids"][2, 0] = 2 ** 31 - 1
    a["ids"][3, :2] = -2 ** 31
    y = check(hg, a, fmt)
    assert bool((y[0] == 0).all()) and bool((y[3] == 0).all())
    a["ids"].fill_(1)
    check(hg, a, fmt)
    a["ids"].fill_(-1)
    assert bool((hg.moe_experts(**a, format=fmt) == 0).all())


@gpu_test
@pytest.mark.parametrize("fmt", ["e4m3", "int4"])
def test_experts_strides_and_guards(gpu, fmt):
    T, E, k, D, F = GROUPED[0]
    a = make(8, T, E, k, D, F, fmt, 64, zeros=True)
    big = torch.zeros((T, D + 24), device="cuda", dtype=torch.bfloat16)
    big[:, 8:8 + D] = a["x"]
    a["x"] = big[:, 8:8 + D]
    for n in ("13", "2"):
        w = a["w" + n]
        wide = torch.zeros((E + 1, w.shape[1] + 3, w.shape[2] + 32), device="cuda",
                           dtype=torch.uint8)
        wide[1:, 1:-2, 16:-16] = w.view(torch.uint8)
        a["w" + n] = wide[1:, 1:-2, 16:-16].view(w.dtype)
    guard = torch.full((T + 2, D + 6), -77.0, device="cuda", dtype=torch.bfloat16)
    out = guard[1:-1, 3:-3]
    hg.moe_experts(**a, format=fmt, group_size=64, out=out)
    want, slack = moe_plain(a, fmt, 64, "silu")
    u.agree(out.contiguous(), want, slack)
    keep = torch.ones_like(guard, dtype=torch.bool)
    keep[1:-1, 3:-3] = False
    assert bool((guard[keep] == -77.0).all())


@gpu_test
def test_experts_nan_codes_of_others(gpu):
    """Nothing of another expert's rows is read into the sums: K ends inside a unit,
    and the neighbours' codes are NaN."""
    a = make(4, *GROUPED[0])
    a["ids"].fill_(1)
    for n in ("w13", "w2"):
        a[n].view(torch.uint8)[0] = 0x7F
        a[n].view(torch.uint8)[2:] = 0x7F
    y = hg.moe_experts(**a)
    assert bool(torch.isfinite(y).all())
    for n in ("w13", "w2"):
        a[n].view(torch.uint8)[0] = 0
        a[n].view(torch.uint8)[2:] = 0
    check(hg, a)


@gpu_test
@pytest.mark.parametrize("fmt", ["e4m3", "int4", "fp4"])
@pytest.mark.parametrize("size", [GROUPED[0], GROUPED[2], GROUPED[3]])
def test_experts_nan_and_inf_rows_stay_apart(gpu, fmt, size):
    """A token of NaN or infinities leaves the other tokens' results as they are."""
    a = make(6, *size, fmt)
    ref = hg.moe_experts(**a, format=fmt)
    a["x"][2] = float("nan")
    a["x"][5, 7] = float("inf")
    y = hg.moe_experts(**a, format=fmt)
    rest = [t for t in range(size[0]) if t not in (2, 5)]
    assert torch.equal(y[rest], ref[rest])
    assert bool(torch.isnan(y[2]).all()) and not bool(torch.isfinite(y[5]).any())


@gpu_test
def test_experts_h_next_to_the_largest(gpu):
    """A gate times up that is finite in fp32 and infinite in bf16 gives an infinity,
    no NaN."""
    T, E, k, D, F = GROUPED[0]
    a = make(5, T, E, k, D, F)
    a["x"].fill_(1.0)
    for n in ("w13", "w2"):
        a[n].copy_(torch.ones_like(a[n], dtype=torch.float32))
    a["scales13"].fill_(float((2.0 ** 128 * (1 - 2.0 ** -12)) ** 0.5 / D))
    a["scales2"].fill_(1.0)
    a["weights"].fill_(1.0)
    assert bool((hg.moe_experts(**a, activation=None) == float("inf")).all())


@gpu_test
@pytest.mark.parametrize("size,fmt", [(GROUPED[0], "int4"), (GROUPED[4], "fp4"), (GROUPED[6], "e4m3"),
                                      (GROUPED[7], "int4")])
def test_experts_stream_graph_and_workspace(gpu, size, fmt):
    T, E, k, D, F = size
    a = make(12, *size, fmt)
    ref = hg.moe_experts(**a, format=fmt)
    assert torch.equal(hg.moe_experts(**a, format=fmt), ref)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    y = hg.moe_experts(**a, format=fmt, stream=side)
    torch.cuda.synchronize()
    assert torch.equal(y, ref)
    ws = torch.full((hg.moe_workspace_size(T, k, E, D, F),), 255, dtype=torch.uint8, device="cuda")
    assert torch.equal(hg.moe_experts(**a, format=fmt, workspace=ws), ref)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = hg.moe_experts(**a, format=fmt, workspace=ws)
    g = u.generator(1)
    for _ in range(3):
        a["x"].copy_(torch.randn(a["x"].shape, generator=g, device="cuda"))
        a["ids"].copy_(torch.rand((T, E), generator=g, device="cuda").topk(k, 1).indices)
        ref = hg.moe_experts(**a, format=fmt)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ref)
