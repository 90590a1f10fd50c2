"""Products of 16-bit activations with 16-bit weights and what follows them in a
feed-forward block, as measured calls: listed() names twelve, draw() gives further
ones of the same ranges; prepare() makes what a program holds before the call,
run() is one pass (the framework's entry points where `own`, elementary fp32
tensor operations otherwise), exact() the same result in 64 bits.

Kinds:
  linear  hipgemm_amd.linear: y = act(x W^T + b) + r, x (M x K), W (N x K).
  gated   hipgemm_amd.gated_linear: h = act(x Wg^T + bg) * (x Wu^T + bu), the two
          weights as one (2N x K) matrix, gate rows first.
Where `train`, a pass is the product and its backward pass (linear_backward,
gated_linear_backward): the gradients of x, of the weight and of the bias beside
the result.  (That of the residual is the result's own.)
"""
import math

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16,
          "float32": torch.float32}
#: The largest listed cases bound what a drawn one may cost.
MAX_FLOPS = 3 * 2.0 * 4096 * 2 * 14336 * 4096
MAX_WEIGHTS = 28672 * 8192


def listed():
    return [
        # One token through a square projection, added to the residual stream:
        # what one call costs.
        dict(name="linear one token", kind="linear", M=1, N=4096, K=4096,
             dtype="bfloat16", bias=False, act="none", residual="bfloat16",
             train=False),
        # One token through the largest down projection: a pass over the weights.
        dict(name="linear one token, large", kind="linear", M=1, N=8192, K=28672,
             dtype="float16", bias=False, act="none", residual="float16",
             train=False),
        # Decode of 16 sequences through a down projection with bias.
        dict(name="linear decode 16", kind="linear", M=16, N=4096, K=14336,
             dtype="bfloat16", bias=True, act="none", residual="bfloat16",
             train=False),
        # Odd sizes on every side, bias and activation, residual stream in fp32.
        dict(name="linear ragged", kind="linear", M=333, N=5001, K=3592,
             dtype="float16", bias=True, act="gelu_tanh", residual="float32",
             train=False),
        # A prompt through a down projection.
        dict(name="linear prefill", kind="linear", M=4096, N=4096, K=14336,
             dtype="bfloat16", bias=False, act="none", residual="bfloat16",
             train=False),
        # The up projection of a plain MLP in training.
        dict(name="linear training", kind="linear", M=4096, N=16384, K=4096,
             dtype="bfloat16", bias=True, act="gelu_tanh", residual="none",
             train=True),
        # Odd sizes in training.
        dict(name="linear training, ragged", kind="linear", M=1531, N=2001,
             K=1000, dtype="float16", bias=True, act="relu", residual="float16",
             train=True),
        # One token through gate and up projections: decode latency.
        dict(name="gated one token", kind="gated", M=1, N=14336, K=4096,
             dtype="bfloat16", bias=False, act="silu", residual="none",
             train=False),
        # A decode batch.
        dict(name="gated decode 64", kind="gated", M=64, N=14336, K=4096,
             dtype="bfloat16", bias=False, act="silu", residual="none",
             train=False),
        # A prefill chunk.
        dict(name="gated prefill", kind="gated", M=2048, N=14336, K=4096,
             dtype="bfloat16", bias=False, act="silu", residual="none",
             train=False),
        # A training step's feed-forward input half.
        dict(name="gated training", kind="gated", M=4096, N=14336, K=4096,
             dtype="bfloat16", bias=False, act="silu", residual="none",
             train=True),
        # A small model's, odd sizes, with biases.
        dict(name="gated training, ragged", kind="gated", M=777, N=1400, K=1000,
             dtype="float16", bias=True, act="gelu_tanh", residual="none",
             train=True),
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of step, log-uniform between lo and hi."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(step, int(round(v / step)) * step)


def draw(rng):
    kind = rng.choice(("linear", "gated"))
    train = rng.random() < 0.45
    # One case in three has sizes that are no multiples of tiles.
    odd = rng.random() < 0.34
    while True:
        c = dict(kind=kind, M=_log(rng, 1, 8192),
                 N=_log(rng, 256, 28672, (1 if kind == "linear" else 8) if odd else 128),
                 K=_log(rng, 256, 28672, 8 if odd else 128),
                 dtype=rng.choice(("bfloat16", "bfloat16", "float16")),
                 bias=rng.random() < 0.4,
                 act=rng.choice(("none", "relu", "silu", "gelu_tanh"))
                 if kind == "linear" else rng.choice(("silu", "silu", "gelu_tanh", "relu")),
                 residual="none", train=train)
        if train:
            c["M"] = _log(rng, 64, 8192)
        elif rng.random() < 0.3:
            c["M"] = rng.choice((1, 1, 2, 3, 4, 8))
        if kind == "linear" and rng.random() < 0.5:
            c["residual"] = rng.choice((c["dtype"], c["dtype"], "float32"))
        if (work(c)["flops"] <= MAX_FLOPS
                and c["N"] * c["K"] * (2 if kind == "gated" else 1) <= MAX_WEIGHTS):
            return c


# ---- inputs ---------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)


def _normal(g, *shape, std=1.0, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda").mul_(std).to(dtype)


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case)
    M, N, K, dtype = case["M"], case["N"], case["K"], DTYPES[case["dtype"]]
    rows = 2 * N if case["kind"] == "gated" else N
    # Unit normal rows whose channels differ in scale, as a norm with learned
    # weights leaves them; weights that keep the variance.
    channel = _normal(g, K, std=0.5).exp_()
    s["x"] = (torch.randn((M, K), generator=g, device="cuda") * channel).to(dtype)
    s["w"] = _normal(g, rows, K, std=K ** -0.5, dtype=dtype)
    s["b"] = _normal(g, rows, std=0.2, dtype=dtype) if case["bias"] else None
    s["r"] = None
    if case["residual"] != "none":
        s["r"] = _normal(g, M, N, dtype=DTYPES[case["residual"]])
    # The gradient that comes back, in the result's type.
    s["dy"] = _normal(g, M, N, std=0.5, dtype=dtype) if case["train"] else None
    return s


# ---- one pass -------------------------------------------------------------

def run(s):
    if own:
        return _run_own(s)
    return _plain_gated(s) if s["kind"] == "gated" else _plain_linear(s)


def _run_own(s):
    import hipgemm_amd as hg
    x, w, b, act = s["x"], s["w"], s["b"], s["act"]
    if s["kind"] == "gated":
        if not s["train"]:
            return hg.gated_linear(x, w, bias=b, activation=act)
        h, pre = hg.gated_linear(x, w, bias=b, activation=act, save_pre=True)
        dx, dw, db = hg.gated_linear_backward(s["dy"], x, w, pre, activation=act,
                                              need_bias=b is not None)
        return {"y": h, "dx": dx, "dw": dw, "db": db}
    if not s["train"]:
        return hg.linear(x, w, bias=b, activation=act, residual=s["r"])
    if act == "none":
        pre = None
        y = hg.linear(x, w, bias=b, activation=act, residual=s["r"])
    else:
        y, pre = hg.linear(x, w, bias=b, activation=act, residual=s["r"], save_pre=True)
    dx, dw, db = hg.linear_backward(s["dy"], x, w, pre, activation=act,
                                    need_bias=b is not None)
    return {"y": y, "dx": dx, "dw": dw, "db": db}


C0 = math.sqrt(2 / math.pi)


def _act(v, act):
    if act == "relu":
        return torch.where(v < 0, torch.zeros_like(v), v)
    if act == "silu":
        return v / (1 + torch.exp(-v))
    if act == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(C0 * (v + 0.044715 * v * v * v)))
    return v


def _slope(v, act):
    """The activation's derivative."""
    if act == "relu":
        return (v > 0).to(v.dtype)
    if act == "silu":
        s = 1 / (1 + torch.exp(-v))
        return s * (1 + v * (1 - s))
    if act == "gelu_tanh":
        t = torch.tanh(C0 * (v + 0.044715 * v * v * v))
        return 0.5 * (1 + t) + 0.5 * v * (1 - t * t) * C0 * (1 + 3 * 0.044715 * v * v)
    return torch.ones_like(v)


def _gradients(s, x, w, dz):
    """Of x, the weight and the bias, rounded once."""
    return {"dx": (dz @ w).to(s["x"].dtype), "dw": (dz.t() @ x).to(s["w"].dtype),
            "db": dz.sum(0).to(s["w"].dtype) if s["b"] is not None else None}


def _plain_linear(s):
    x, w = s["x"].float(), s["w"].float()
    z = x @ w.t()
    if s["b"] is not None:
        z += s["b"].float()
    y = _act(z, s["act"])
    if s["r"] is not None:
        y = y + s["r"].float()
    y = y.to(s["x"].dtype)
    if not s["train"]:
        return y
    dz = s["dy"].float() * _slope(z, s["act"])
    return {"y": y, **_gradients(s, x, w, dz)}


def _plain_gated(s):
    x, w, n = s["x"].float(), s["w"].float(), s["N"]
    z = x @ w.t()
    if s["b"] is not None:
        z += s["b"].float()
    gate, up = z[:, :n], z[:, n:]
    a = _act(gate, s["act"])
    h = (a * up).to(s["x"].dtype)
    if not s["train"]:
        return h
    dh = s["dy"].float()
    dz = torch.cat((dh * up * _slope(gate, s["act"]), dh * a), 1)
    return {"y": h, **_gradients(s, x, w, dz)}


# ---- what a pass cannot do without ---------------------------------------

def work(case):
    M, N, K = case["M"], case["N"], case["K"]
    rows = 2 * N if case["kind"] == "gated" else N
    # x, weight, bias, residual in; result out.
    size = 2.0 * M * K + 2.0 * rows * K + 2.0 * M * N
    if case["bias"]:
        size += 2.0 * rows
    if case["residual"] != "none":
        size += (4.0 if case["residual"] == "float32" else 2.0) * M * N
    flops = 2.0 * M * rows * K
    if case["train"]:
        # dy in; gradients of x, weight and bias out; two further products.
        size += 2.0 * M * N + 2.0 * M * K + 2.0 * rows * K
        size += 2.0 * rows if case["bias"] else 0.0
        flops *= 3
    return {"bytes": size, "flops": flops}


# ---- the same in 64 bits --------------------------------------------------

def _act64(v, act):
    if act == "relu":
        return torch.nn.functional.relu(v)
    if act == "silu":
        return torch.nn.functional.silu(v)
    if act == "gelu_tanh":
        return torch.nn.functional.gelu(v, approximate="tanh")
    return v


def exact(case, seed):
    s = prepare(case, seed)
    x, w, train = s["x"].double(), s["w"].double(), case["train"]
    b = s["b"].double() if case["bias"] else torch.zeros(w.shape[0], dtype=torch.float64,
                                                         device="cuda")
    for t in (x, w, b):
        t.requires_grad_(train)
    z = torch.addmm(b, x, w.t())
    if case["kind"] == "gated":
        gate, up = z.chunk(2, 1)
        y = _act64(gate, case["act"]) * up
    else:
        y = _act64(z, case["act"])
        if s["r"] is not None:
            y = y + s["r"].double()
    if not train:
        return y
    dx, dw, db = torch.autograd.grad(y, (x, w, b), s["dy"].double())
    return {"y": y.detach(), "dx": dx, "dw": dw, "db": db if case["bias"] else None}
