"""moe_experts against its definition in 64 bits.

Tolerance: fp32 sums as for w4_gemm, fewer than K / 128 + 64 roundings of 2^-24
of the sum of magnitudes each; the gate's and up's pass through the activation
(its slope is below 1.13) and the product; h's two parts leave 2^-16 of it; the
routing weights' products and the sum over k add 4 + k roundings."""
import pytest
import torch

import w4util as u

pytestmark = pytest.mark.gpu


def make(seed, T, E, k, D, F, fmt="e4m3", group=128, scale="bfloat16", zeros=False,
         dtype="bfloat16"):
    g = u.generator(seed)
    a = dict(x=torch.randn((T, D), generator=g, device="cuda").to(getattr(torch, dtype)),
             ids=torch.rand((T, E), generator=g, device="cuda").topk(k, 1).indices.int(),
             weights=torch.rand((T, k), generator=g, device="cuda"))
    for name, rows, K in (("13", 2 * F, D), ("2", D, F)):
        if fmt == "e4m3":
            a["w" + name] = (torch.randn((E, rows, K), generator=g, device="cuda") * 60).to(
                torch.float8_e4m3fn)
            a["scales" + name] = torch.rand((E, rows), generator=g, device="cuda") * 1e-3 + 1e-4
            a["zeros" + name] = None
        else:
            a["w" + name], a["scales" + name], a["zeros" + name] = u.four_bit(
                g, (E, rows), K, fmt, group, scale, zeros)
    return a


def plain(a, fmt, group, act):
    x = a["x"].double()
    y, slack = torch.zeros_like(x), torch.zeros_like(x)
    E, F = a["w13"].shape[0], a["w13"].shape[1] // 2
    T, k = a["ids"].shape
    unit = 2.0 ** -24

    def magnitudes(name, e):
        w, s, z = a["w" + name][e], a["scales" + name][e], a["zeros" + name]
        if fmt == "e4m3":
            return w.double().abs() * s.double()[:, None]
        q = u.unpack(w).double()
        if fmt == "fp4":
            m = u.codes64(w, fmt, None, group).abs()
        else:
            m = q + 256 + (8 if z is None else
                           z[e].double().repeat_interleave(group, 1)[:, :q.shape[1]])
        return m * u.scales64(s).repeat_interleave(group, 1)[:, :q.shape[1]]

    for e in range(E):
        t, j = (a["ids"] == e).nonzero(as_tuple=True)
        if not len(t):
            continue
        z13, z2 = ((a[n][e] if a[n] is not None else None) for n in ("zeros13", "zeros2"))
        w13 = u.weights64(a["w13"][e], a["scales13"][e], fmt, group, z13)
        w2 = u.weights64(a["w2"][e], a["scales2"][e], fmt, group, z2)
        gu = x[t] @ w13.t()
        dgu = x[t].abs() @ magnitudes("13", e).t() * ((x.shape[1] / 128 + 64) * unit)
        gate, dgate = u.act64(gu[:, :F], act), 1.13 * dgu[:, :F]
        dgate = dgate + 8 * unit * gate.abs()
        r = a["weights"][t, j].double()[:, None]
        h = gate * gu[:, F:] * r
        dh = (dgate * gu[:, F:].abs() + gate.abs() * dgu[:, F:] + dgate * dgu[:, F:]) * r.abs()
        dh = dh + h.abs() * (2.0 ** -16 + 4 * unit)
        y.index_add_(0, t, h @ w2.t())
        slack.index_add_(0, t, dh @ w2.abs().t() + h.abs() @ magnitudes("2", e).t()
                         * ((F / 128 + 64 + k) * unit))
    return y, slack


def check(hg, a, fmt="e4m3", group=128, act="silu", **kw):
    y = hg.moe_experts(**a, format=fmt, group_size=group, activation=act, **kw)
    assert y.shape == a["x"].shape
    want, slack = plain(a, fmt, group, act)
    u.agree(y, want, slack)
    return y


@pytest.fixture()
def hg(gpu):
    import hipgemm_amd
    return hipgemm_amd


SHAPES = [(1, 1, 1, 32, 32), (1, 8, 2, 256, 512), (1, 64, 8, 2048, 1024), (2, 5, 3, 96, 160),
          (3, 30, 3, 1056, 288), (16, 16, 4, 512, 256), (33, 4, 2, 384, 96),
          (64, 40, 8, 256, 128), (64, 128, 8, 128, 64), (100, 6, 1, 64, 224),
          (200, 9, 4, 96, 64), (7, 512, 64, 64, 32)]


@pytest.mark.parametrize("T,E,k,D,F", SHAPES)
@pytest.mark.parametrize("fmt", ["e4m3", "int4", "fp4"])
def test_shapes(hg, T, E, k, D, F, fmt):
    check(hg, make(T + E + k, T, E, k, D, F, fmt, zeros=fmt == "int4" and T % 2 == 0), fmt)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("scale", ["bfloat16", "float16", "float32", "e8m0"])
@pytest.mark.parametrize("group", [32, 64, 96, 256])
@pytest.mark.parametrize("T", [2, 40])
def test_groups_and_types(hg, T, group, scale, dtype):
    for fmt in ("int4", "fp4"):
        check(hg, make(group, T, 3, 2, 416, 352, fmt, group, scale, fmt == "int4", dtype),
              fmt, group)


@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu_tanh"])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float16, torch.float32])
def test_epilogue(hg, act, out):
    for fmt in ("e4m3", "int4"):
        check(hg, make(3, 5, 7, 3, 256, 128, fmt), fmt, act=act, out_dtype=out)


def test_skipped_ids(hg):
    """Ids outside [0, E) contribute nothing; a token without any gives zeros."""
    for T in (1, 6, 70):
        a = make(T, T, 6, 3, 160, 96)
        a["ids"][0] = -1
        if T > 1:
            a["ids"][1, 1] = 6
            a["ids"][2, 0] = 2 ** 31 - 1
            a["ids"][3, :2] = -2 ** 31
        y = check(hg, a)
        assert bool((y[0] == 0).all())
    a["ids"].fill_(-1)
    assert bool((hg.moe_experts(**a) == 0).all())


def test_one_expert_for_all_and_twice(hg):
    for T in (1, 16, 17, 64):
        a = make(T, T, 9, 2, 128, 96, "int4")
        a["ids"].fill_(4)
        check(hg, a, "int4")


@pytest.mark.parametrize("fmt", ["e4m3", "int4"])
def test_strides_and_guards(hg, fmt):
    T, E, k, D, F = 10, 5, 2, 224, 160
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
    want, slack = plain(a, fmt, 64, "silu")
    u.agree(out.contiguous(), want, slack)
    keep = torch.ones_like(guard, dtype=torch.bool)
    keep[1:-1, 3:-3] = False
    assert bool((guard[keep] == -77.0).all())


def test_nan_codes_of_other_experts(hg):
    """Nothing of another expert's rows is read into the sums: K ends inside a
    block of 128, and the neighbours' codes are NaN."""
    a = make(4, 3, 4, 2, 160, 96)
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


def test_nan_and_inf_rows_stay_apart(hg):
    """A token of NaN or infinities leaves the other tokens' results as they are."""
    for fmt in ("e4m3", "int4", "fp4"):
        a = make(6, 9, 3, 2, 128, 64, fmt)
        ref = hg.moe_experts(**a, format=fmt)
        a["x"][2] = float("nan")
        a["x"][5, 7] = float("inf")
        y = hg.moe_experts(**a, format=fmt)
        rest = [0, 1, 3, 4, 6, 7, 8]
        assert torch.equal(y[rest], ref[rest])
        assert bool(torch.isnan(y[2]).all()) and not bool(torch.isfinite(y[5]).any())


def test_other_stream_graph_and_workspace(hg):
    a = make(12, 4, 16, 4, 512, 256, "int4")
    ref = hg.moe_experts(**a, format="int4")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    y = torch.zeros_like(ref)
    hg.moe_experts(**a, format="int4", out=y, stream=side)
    torch.cuda.synchronize()
    assert torch.equal(y, ref)
    ws = torch.full((hg.moe_workspace_size(4, 4, 16, 512, 256),), 255, dtype=torch.uint8,
                    device="cuda")
    assert torch.equal(hg.moe_experts(**a, format="int4", workspace=ws), ref)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits = a["x"].float() @ torch.ones((512, 16), device="cuda")
        y = hg.moe_experts(**a, format="int4", workspace=ws)
    g = u.generator(1)
    for _ in range(3):
        a["x"].copy_(torch.randn(a["x"].shape, generator=g, device="cuda"))
        a["ids"].copy_(torch.rand((4, 16), generator=g, device="cuda").topk(4, 1).indices)
        ref = hg.moe_experts(**a, format="int4")
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ref)


def test_results_belong_to_the_stream(hg):
    """Without `out`, results (and an experts' call's workspace) are memory of the
    stream that writes them, not what the current stream has just freed."""
    a = make(3, 4, 16, 4, 256, 128, "int4", zeros=True)
    wide = a["zeros13"][0].t().contiguous().t()  # (of other strides: copied)
    want = (hg.moe_experts(**a, format="int4"), *hg.moe_route(a["x"][:, :16], 4),
            hg.w4_gemm(a["x"], a["w13"][0], a["scales13"][0], wide))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = (hg.moe_experts(**a, format="int4", stream=side),
           *hg.moe_route(a["x"][:, :16], 4, stream=side),
           hg.w4_gemm(a["x"], a["w13"][0], a["scales13"][0], wide, stream=side))
    torch.cuda.synchronize()
    segments = torch.cuda.memory_snapshot()
    for x, y in zip(want, got):
        assert torch.equal(x, y)
        p = y.data_ptr()
        owner = [s["stream"] for s in segments
                 if s["address"] <= p < s["address"] + s["total_size"]]
        assert owner == [side.cuda_stream]


# Sizes of which a workgroup's LDS holds few rows, or none: many tokens of wide
# experts, parts of F, and the way pair by pair beyond.
@pytest.mark.parametrize("fmt", ["e4m3", "int4"])
@pytest.mark.parametrize("T,E,k,D,F", [(16, 2, 1, 256, 14336), (40, 2, 1, 96, 14368),
                                       (7, 2, 2, 64, 18592), (5, 1, 1, 128, 65568),
                                       (33, 2, 2, 8192, 64), (20, 1, 1, 28960, 32),
                                       (6, 1, 1, 37120, 32), (6, 1, 1, 37152, 32)])
def test_wide(hg, T, E, k, D, F, fmt):
    check(hg, make(T + F, T, E, k, D, F, fmt, zeros=fmt == "int4"), fmt)


def test_h_next_to_the_largest(hg):
    """A gate times up that is finite in fp32 and infinite in bf16 gives an
    infinity, no NaN."""
    a = make(5, 4, 2, 2, 32, 32)
    a["x"].fill_(1.0)
    for n in ("w13", "w2"):
        a[n].copy_(torch.ones_like(a[n], dtype=torch.float32))
    a["scales13"].fill_(float((2.0 ** 128 * (1 - 2.0 ** -12)) ** 0.5 / 32))
    a["scales2"].fill_(1.0)
    a["weights"].fill_(1.0)
    for T in (1, 4):  # pair by pair, grouped
        y = hg.moe_experts(a["x"][:T], a["ids"][:T], a["weights"][:T], a["w13"], a["scales13"],
                           a["w2"], a["scales2"], activation=None)
        assert bool((y == float("inf")).all())


def test_repeats_are_equal(hg):
    for T in (1, 64):
        a = make(T, T, 24, 6, 512, 384, "fp4")
        x, y = (hg.moe_experts(**a, format="fp4") for _ in range(2))
        assert torch.equal(x, y)


def test_empty(hg):
    a = make(1, 1, 4, 2, 64, 32)
    a.update(x=a["x"][:0], ids=a["ids"][:0], weights=a["weights"][:0])
    assert hg.moe_experts(**a).shape == (0, 64)


@pytest.mark.parametrize("change", [
    dict(x=lambda t: t.float()), dict(x=lambda t: t.cpu()), dict(x=lambda t: t[:, :32]),
    dict(ids=lambda t: t.long()), dict(ids=lambda t: t[:, :1]), dict(ids=lambda t: t.cpu()),
    dict(weights=lambda t: t.double()), dict(weights=lambda t: t[:1]),
    dict(weights=lambda t: t.t().contiguous().t()),
    dict(w13=lambda t: t[:, 1:]), dict(w13=lambda t: t.float()), dict(w13=lambda t: t[0]),
    dict(w2=lambda t: t[:-1]), dict(w2=lambda t: t[:, :, :32]), dict(w2=lambda t: t.cpu()),
    dict(scales13=lambda t: t.half()), dict(scales2=lambda t: t[:, 1:]),
    dict(format="int8"), dict(format="int4"), dict(activation="tanh"),
    dict(out_dtype=torch.int32), dict(workspace=torch.empty(4, dtype=torch.uint8)),
])
def test_refusals(hg, change):
    a = make(2, 3, 4, 2, 64, 96)
    hg.moe_experts(**a)
    kw = {}
    for k, f in change.items():
        if k in a:
            a[k] = f(a[k])
        else:
            kw[k] = f
    with pytest.raises(hg.HipGemmError):
        hg.moe_experts(**a, **kw)


def test_refuses_small_workspace(hg):
    a = make(2, 3, 4, 2, 64, 96)
    ws = torch.empty(hg.moe_workspace_size(3, 2, 4, 64, 96) - 1, dtype=torch.uint8, device="cuda")
    with pytest.raises(hg.HipGemmError):
        hg.moe_experts(**a, workspace=ws)
