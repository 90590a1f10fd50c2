"""Products with 4-bit weights, the router's choice and the layer of experts,
as measured calls: listed() names twelve, draw() gives further ones of the same
ranges; prepare() makes what a program holds before the call, run() is one pass
(the framework's entry points where `own`, elementary fp32 tensor operations
otherwise), exact() the same result in 64 bits.

Kinds:
  w4       hipgemm_amd.w4_gemm: 16-bit activations (M x K) by 4-bit weights
           (N x K) with one scale per group of weights along K.
  route    hipgemm_amd.moe_route: the k largest of each token's router logits,
           and their weights.
  experts  hipgemm_amd.moe_experts: gated MLP of each token's chosen experts
           (E experts of width F over a model width D), summed with the
           routing weights.
"""
import math

import torch

own = False

E4M3 = torch.float8_e4m3fn
#: Values of the sixteen E2M1 codes.
FP4 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0,
       -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)
DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16,
          "float32": torch.float32}
#: The largest listed cases bound what a drawn one may cost.
MAX_FLOPS = 2.0 * 2048 * 14336 * 4096
MAX_WEIGHTS = 28672 * 8192
MAX_EXPERT_WEIGHTS = 128 * 3 * 4096 * 1536


def listed():
    return [
        # One token through a square projection: what one call costs.
        dict(name="w4 one token", kind="w4", M=1, N=4096, K=4096, format="int4",
             group=128, scale="bfloat16", zeros=False, dtype="bfloat16",
             bias=False, act="none"),
        # One token through the largest projection, with zero points: a pass
        # over the weights.
        dict(name="w4 one token, large", kind="w4", M=1, N=28672, K=8192,
             format="int4", group=128, scale="float16", zeros=True,
             dtype="float16", bias=False, act="none"),
        # Decode of 16 sequences through an up projection, microscaled fp4.
        dict(name="w4 decode 16", kind="w4", M=16, N=14336, K=4096, format="fp4",
             group=32, scale="e8m0", zeros=False, dtype="bfloat16", bias=False,
             act="silu"),
        # Odd sizes on every side, small groups, bias.
        dict(name="w4 ragged", kind="w4", M=37, N=5000, K=3584, format="int4",
             group=64, scale="float16", zeros=True, dtype="bfloat16", bias=True,
             act="gelu_tanh"),
        # A prefill chunk through an up projection.
        dict(name="w4 prefill", kind="w4", M=2048, N=14336, K=4096,
             format="int4", group=128, scale="bfloat16", zeros=False,
             dtype="bfloat16", bias=False, act="none"),
        # The choice for one token.
        dict(name="route one token", kind="route", T=1, E=64, k=8,
             dtype="float32", scoring="softmax", renormalize=True, masked=False),
        # The choice for a long prefill, some experts switched off.
        dict(name="route prefill", kind="route", T=16384, E=256, k=8,
             dtype="bfloat16", scoring="sigmoid", renormalize=True, masked=True),
        # One token, two of eight wide experts in e4m3.
        dict(name="experts one token, wide", kind="experts", T=1, E=8, k=2,
             D=4096, F=14336, format="e4m3", group=0, dtype="bfloat16",
             act="silu"),
        # One token, eight of 64 narrow experts in int4: latency.
        dict(name="experts one token, narrow", kind="experts", T=1, E=64, k=8,
             D=2048, F=1024, format="int4", group=128, dtype="bfloat16",
             act="silu"),
        # A small decode batch over e4m3 experts.
        dict(name="experts decode 16", kind="experts", T=16, E=64, k=4, D=4096,
             F=2048, format="e4m3", group=0, dtype="bfloat16", act="silu"),
        # Odd sizes, microscaled fp4.
        dict(name="experts ragged", kind="experts", T=5, E=30, k=3, D=2336,
             F=1056, format="fp4", group=32, dtype="float16", act="gelu_tanh"),
        # A decode batch that reaches nearly every expert.
        dict(name="experts decode 64", kind="experts", T=64, E=128, k=8, D=4096,
             F=1536, format="int4", group=128, dtype="bfloat16", act="silu"),
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of step, log-uniform between lo and hi."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(step, int(round(v / step)) * step)


def draw(rng):
    kind = rng.choice(("w4", "w4", "route", "experts", "experts"))
    dtype = rng.choice(("bfloat16", "bfloat16", "float16"))
    # One case in three has sizes that are no multiples of tiles.
    odd = rng.random() < 0.34
    while True:
        if kind == "w4":
            fmt = rng.choice(("int4", "int4", "fp4"))
            c = dict(kind=kind, M=_log(rng, 1, 2048),
                     N=_log(rng, 256, 28672, 1 if odd else 128),
                     K=_log(rng, 256, 28672, 32 if odd else 128), format=fmt,
                     group=rng.choice((32, 64, 128, 128, 256)),
                     scale=rng.choice(("bfloat16", "float16", "float32", "e8m0")),
                     zeros=fmt == "int4" and rng.random() < 0.5, dtype=dtype,
                     bias=rng.random() < 0.3,
                     act=rng.choice(("none", "none", "relu", "silu", "gelu_tanh")))
            if rng.random() < 0.3:
                c["M"] = rng.choice((1, 1, 2, 3, 4))
            if (2.0 * c["M"] * c["N"] * c["K"] <= MAX_FLOPS
                    and c["N"] * c["K"] <= MAX_WEIGHTS):
                return c
        elif kind == "route":
            E = _log(rng, 8, 512, 1 if odd else 8)
            return dict(kind=kind, T=_log(rng, 1, 16384), E=E,
                        k=rng.randint(1, min(16, E)),
                        dtype=rng.choice(("float32", "bfloat16", "float16")),
                        scoring=rng.choice(("softmax", "softmax", "sigmoid")),
                        renormalize=rng.random() < 0.7,
                        masked=rng.random() < 0.3)
        else:
            fmt = rng.choice(("e4m3", "e4m3", "int4", "fp4"))
            E = _log(rng, 4, 256, 1 if odd else 4)
            c = dict(kind=kind, T=_log(rng, 1, 64), E=E,
                     k=rng.randint(1, min(8, E)),
                     D=_log(rng, 256, 8192, 32 if odd else 128),
                     F=_log(rng, 256, 14336, 32 if odd else 128), format=fmt,
                     group=0 if fmt == "e4m3" else rng.choice((32, 64, 128)),
                     dtype=dtype, act=rng.choice(("silu", "silu", "gelu_tanh")))
            if 3 * E * c["D"] * c["F"] <= MAX_EXPERT_WEIGHTS:
                return c


# ---- inputs ---------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)


def _normal(g, *shape, std=1.0, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda").mul_(std).to(dtype)


def _activations(g, rows, cols, dtype):
    """Unit normal rows whose channels differ in scale, as a norm with learned
    weights leaves them."""
    channel = torch.randn(cols, generator=g, device="cuda").mul_(0.5).exp_()
    return (torch.randn((rows, cols), generator=g, device="cuda") * channel).to(dtype)


def _groups(K, group):
    return -(-K // group)


def _four_bit(g, shape, K, fmt, group, scale, zeros):
    """Codes, scales and zero points of normal weights of variance 1 / K,
    quantised by groups of `group`: the largest of a group is near the end of the
    codes' range. Codes are drawn as such (a group's rounded normals)."""
    n = torch.randn((*shape, K), generator=g, device="cuda", dtype=torch.float16)
    if fmt == "int4":
        code = n.mul_(2.7).add_(7.5).round_().clamp_(0, 15).to(torch.uint8)
        step = K ** -0.5 / 2.7
    else:
        mid = torch.tensor((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0), device="cuda",
                           dtype=torch.float16)
        n.mul_(2.2)
        code = torch.bucketize(n.abs(), mid, out_int32=True).to(torch.uint8)
        code |= (n < 0).to(torch.uint8) << 3
        step = K ** -0.5 / 2.2
    del n
    packed = code[..., 0::2] | (code[..., 1::2] << 4)
    del code
    s = torch.randn((*shape, _groups(K, group)), generator=g, device="cuda")
    s = s.mul_(0.2).exp_().mul_(step)
    if scale == "e8m0":
        s = torch.log2(s).round_().add_(127).clamp_(0, 254).to(torch.uint8)
    else:
        s = s.to(DTYPES[scale])
    z = None
    if zeros:
        z = torch.randint(5, 11, s.shape, generator=g, device="cuda",
                          dtype=torch.uint8)
    return packed, s, z


def _e4m3(g, shape, K):
    """e4m3 weights of variance 1 / K, each row's largest near 448, and the rows'
    scales."""
    n = torch.randn((*shape, K), generator=g, device="cuda", dtype=torch.float16)
    q = n.mul_(110.0).clamp_(-448, 448).to(E4M3)
    s = torch.randn(shape, generator=g, device="cuda").mul_(0.2).exp_()
    return q, s.mul_(K ** -0.5 / 110.0)


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case)
    if case["kind"] == "w4":
        M, N, K = case["M"], case["N"], case["K"]
        s["x"] = _activations(g, M, K, DTYPES[case["dtype"]])
        s["w"], s["s"], s["z"] = _four_bit(g, (N,), K, case["format"],
                                           case["group"], case["scale"],
                                           case["zeros"])
        s["b"] = _normal(g, N, std=0.2) if case["bias"] else None
        return s
    if case["kind"] == "route":
        s["logits"] = _normal(g, case["T"], case["E"], std=1.5,
                              dtype=DTYPES[case["dtype"]])
        if case["masked"]:  # one expert in eight is switched off
            off = torch.rand(case["E"], generator=g, device="cuda") < 0.125
            s["logits"][:, off] = float("-inf")
        return s
    T, E, k, D, F = (case[v] for v in ("T", "E", "k", "D", "F"))
    s["x"] = _activations(g, T, D, DTYPES[case["dtype"]])
    # Each token's own choice, and weights that sum to one.
    top = torch.rand((T, E), generator=g, device="cuda").topk(k, dim=1)
    s["ids"] = top.indices.to(torch.int32)
    s["weights"] = torch.softmax(_normal(g, T, k), 1)
    if case["format"] == "e4m3":
        s["w13"], s["s13"] = _e4m3(g, (E, 2 * F), D)
        s["w2"], s["s2"] = _e4m3(g, (E, D), F)
    else:
        scale = "e8m0" if case["format"] == "fp4" else "bfloat16"
        s["w13"], s["s13"], _ = _four_bit(g, (E, 2 * F), D, case["format"],
                                          case["group"], scale, False)
        s["w2"], s["s2"], _ = _four_bit(g, (E, D), F, case["format"],
                                        case["group"], scale, False)
    return s


# ---- one pass -------------------------------------------------------------

def run(s):
    if own:
        return _run_own(s)
    return {"w4": _plain_w4, "route": _plain_route,
            "experts": _plain_experts}[s["kind"]](s)


def _run_own(s):
    import hipgemm_amd as hg
    if s["kind"] == "w4":
        return hg.w4_gemm(s["x"], s["w"], s["s"], s["z"], format=s["format"],
                          group_size=s["group"], bias=s["b"],
                          activation=s["act"])
    if s["kind"] == "route":
        w, ids = hg.moe_route(s["logits"], s["k"], scoring=s["scoring"],
                              renormalize=s["renormalize"])
        return {"weights": w, "ids": ids}
    return hg.moe_experts(s["x"], s["ids"], s["weights"], s["w13"], s["s13"],
                          s["w2"], s["s2"], format=s["format"],
                          group_size=s["group"], activation=s["act"])


def _act(v, act):
    if act == "relu":
        return torch.where(v < 0, torch.zeros_like(v), v)
    if act == "silu":
        return v / (1 + torch.exp(-v))
    if act == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v)))
    return v


def _weights32(w, s, z, fmt, group):
    """Quantised weights as fp32 values."""
    if fmt == "e4m3":
        return w.float() * s[..., None]
    code = torch.stack((w & 15, w >> 4), -1).flatten(-2)
    if fmt == "fp4":
        v = torch.tensor(FP4, device=w.device)[code.int()]
    else:
        v = code.float()
    K = v.shape[-1]
    s = torch.exp2(s.float() - 127) if s.dtype == torch.uint8 else s.float()
    if fmt == "int4":
        v -= 8.0 if z is None else z.float().repeat_interleave(group, -1)[..., :K]
    return v.mul_(s.repeat_interleave(group, -1)[..., :K])


def _plain_w4(s):
    w = _weights32(s["w"], s["s"], s["z"], s["format"], s["group"])
    v = s["x"].float() @ w.t()
    if s["b"] is not None:
        v += s["b"]
    return _act(v, s["act"]).to(s["x"].dtype)


def _plain_route(s):
    l = s["logits"].float()
    vals, idx = torch.sort(l, dim=1, descending=True, stable=True)
    vals, idx = vals[:, :s["k"]], idx[:, :s["k"]]
    chosen = vals > float("-inf")
    if s["scoring"] == "softmax":
        p = torch.exp(vals - vals[:, :1])
        total = torch.exp(l - vals[:, :1]).sum(1, keepdim=True)
    else:
        p = 1 / (1 + torch.exp(-vals))
        total = torch.ones_like(p[:, :1])
    p = torch.where(chosen, p, torch.zeros_like(p))
    if s["renormalize"]:
        total = p.sum(1, keepdim=True)
    w = torch.where(chosen, p / total, torch.zeros_like(p))
    return {"weights": w, "ids": torch.where(chosen, idx, -1).to(torch.int32)}


def _plain_experts(s):
    x, F, fmt, group = s["x"].float(), s["F"], s["format"], s["group"]
    T, k = s["ids"].shape
    ids = s["ids"].long()
    if T * k <= s["E"]:
        # Few choices: each one's own copy of its expert's weights.
        e = ids.flatten()
        w13 = _weights32(s["w13"][e], s["s13"][e], None, fmt, group)
        gu = torch.bmm(w13, x.repeat_interleave(k, 0)[:, :, None])[:, :, 0]
        h = _act(gu[:, :F], s["act"]) * gu[:, F:]
        del w13
        w2 = _weights32(s["w2"][e], s["s2"][e], None, fmt, group)
        y = torch.bmm(w2, h[:, :, None])[:, :, 0].view(T, k, -1)
        return (y * s["weights"][:, :, None]).sum(1).to(s["x"].dtype)
    # Many: every expert on every token, with weight zero where not chosen.
    r = torch.zeros((T, s["E"]), device=x.device).scatter_(1, ids, s["weights"])
    w13 = _weights32(s["w13"], s["s13"], None, fmt, group)
    gu = torch.matmul(x, w13.flatten(0, 1).t()).view(T, s["E"], 2 * F)
    del w13
    h = _act(gu[..., :F], s["act"]) * gu[..., F:]
    w2 = _weights32(s["w2"], s["s2"], None, fmt, group)
    y = torch.bmm(w2, h.permute(1, 2, 0).contiguous())  # (E, D, T)
    return (y * r.t()[:, None, :]).sum(0).t().to(s["x"].dtype)


# ---- what a pass cannot do without ---------------------------------------

def _weight_bytes(n, K, fmt, group, scale, zeros):
    """Of n rows of K weights."""
    if fmt == "e4m3":
        return n * (K + 4.0)
    size = {"e8m0": 1, "float32": 4}.get(scale, 2) + (1 if zeros else 0)
    return n * (K / 2.0 + size * _groups(K, group))


def work(case):
    if case["kind"] == "w4":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": _weight_bytes(N, K, case["format"], case["group"],
                                       case["scale"], case["zeros"])
                + 2.0 * M * K + 2.0 * M * N + (4.0 * N if case["bias"] else 0.0),
                "flops": 2.0 * M * N * K}
    if case["kind"] == "route":
        T, E, k = case["T"], case["E"], case["k"]
        size = 4.0 if case["dtype"] == "float32" else 2.0
        return {"bytes": size * T * E + 8.0 * T * k, "flops": 4.0 * T * E}
    T, E, k, D, F = (case[v] for v in ("T", "E", "k", "D", "F"))
    # Experts that at least one token chooses, on average.
    active = E * (1.0 - (1.0 - k / E) ** T)
    scale = "e8m0" if case["format"] == "fp4" else "bfloat16"
    one = (_weight_bytes(2 * F, D, case["format"], case["group"], scale, False)
           + _weight_bytes(D, F, case["format"], case["group"], scale, False))
    return {"bytes": active * one + 4.0 * T * D + 8.0 * T * k,
            "flops": 6.0 * T * k * D * F}


# ---- the same in 64 bits --------------------------------------------------

def _act64(v, act):
    if act == "relu":
        return v.clamp_min(0)
    if act == "silu":
        return v * torch.sigmoid(v)
    if act == "gelu_tanh":
        return torch.nn.functional.gelu(v, approximate="tanh")
    return v


def _weights64(w, s, z, fmt, group):
    """Values of a (rows, K) matrix of quantised weights."""
    if fmt == "e4m3":
        return w.double() * s.double()[:, None]
    rows, K = w.shape[0], 2 * w.shape[1]
    v = torch.empty((rows, K), dtype=torch.float64, device=w.device)
    for half in (0, 1):
        code = (w >> (4 * half)) % 16
        if fmt == "int4":
            v[:, half::2] = code.double()
        else:
            mag = (code % 8).double()
            # E2M1: subnormal below 2, then (2 + m) 2^(e - 2)
            e, m = torch.floor(mag / 2), mag % 2
            mag = torch.where(e == 0, m / 2, (2 + m) * torch.exp2(e - 2))
            v[:, half::2] = torch.where(code >= 8, -mag, mag)
    s = torch.exp2(s.double() - 127) if s.dtype == torch.uint8 else s.double()
    at = torch.arange(K, device=w.device) // group
    if fmt == "int4":
        v -= 8.0 if z is None else z.double()[:, at]
    return v * s[:, at]


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "w4":
        v = s["x"].double() @ _weights64(s["w"], s["s"], s["z"], case["format"],
                                         case["group"]).t()
        if s["b"] is not None:
            v += s["b"].double()
        return _act64(v, case["act"])
    if case["kind"] == "route":
        l = s["logits"].double()
        vals = l.topk(case["k"], dim=1).values  # the values, whatever the ties
        if case["scoring"] == "softmax":
            p = torch.softmax(l, 1).nan_to_num(0.0)
            p = p.topk(case["k"], dim=1).values
        else:
            p = torch.sigmoid(vals)
        if case["renormalize"]:
            p = p / p.sum(1, keepdim=True)
        return {"weights": p.nan_to_num(0.0), "ids": None}
    x, F = s["x"].double(), case["F"]
    y = torch.zeros_like(x)
    for e in s["ids"].unique().tolist():
        t, j = (s["ids"] == e).nonzero(as_tuple=True)
        w13 = _weights64(s["w13"][e], s["s13"][e], None, case["format"], case["group"])
        gu = x[t] @ w13.t()
        h = _act64(gu[:, :F], case["act"]) * gu[:, F:]
        w2 = _weights64(s["w2"][e], s["s2"][e], None, case["format"], case["group"])
        y.index_add_(0, t, (h @ w2.t()) * s["weights"][t, j].double()[:, None])
    return y
