"""Plain 64-bit forms of the products with quantised weights, for the tests."""
import torch

FP4 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
#: Unit roundoff by output type.
ROUND = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
#: Half the spacing of the type's subnormals.
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}


def scales64(s):
    if s.dtype != torch.uint8:
        return s.double()
    e = s.double()
    return torch.where(e == 255, torch.full_like(e, float("nan")), torch.exp2(e - 127))


def unpack(w):
    """Codes of packed rows, element 2i in the low nibble."""
    return torch.stack((w & 15, w >> 4), -1).flatten(-2)


def codes64(w, fmt, z, group):
    """Values of the codes, scales excluded, and z along K."""
    q = unpack(w)
    if fmt == "fp4":
        t = torch.tensor([*FP4, *(-v for v in FP4)], dtype=torch.float64, device=w.device)
        return t[q.long()]
    v = q.double()
    if z is None:
        return v - 8
    return v - z.double().repeat_interleave(group, -1)[..., :v.shape[-1]]


def weights64(w, s, fmt, group=0, z=None):
    if fmt == "e4m3":
        return w.double() * s.double()[..., None]
    v = codes64(w, fmt, z, group)
    return v * scales64(s).repeat_interleave(group, -1)[..., :v.shape[-1]]


def act64(v, act):
    if act == "relu":
        return torch.where(v < 0, torch.zeros_like(v), v)
    if act == "silu":
        return v * torch.sigmoid(v)
    if act == "gelu_tanh":
        return torch.nn.functional.gelu(v, approximate="tanh")
    return v


def four_bit(g, shape, K, fmt, group, scale, zeros, pad=0):
    """Random codes (all of them), scales and zero points, on the GPU; rows of
    codes with `pad` bytes between them."""
    w = torch.randint(0, 256, (*shape, K // 2 + pad), generator=g, dtype=torch.uint8,
                      device="cuda")[..., :K // 2]
    groups = -(-K // group)
    s = torch.rand((*shape, groups), generator=g, device="cuda") * 0.02 + 0.002
    if scale == "e8m0":
        s = torch.randint(115, 124, s.shape, generator=g, dtype=torch.uint8, device="cuda")
    else:
        s = s.to(getattr(torch, scale))
    z = (torch.randint(0, 16, s.shape, generator=g, dtype=torch.uint8, device="cuda")
         if zeros else None)
    return w, s, z


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def agree(got, want, slack):
    """got (rounded) is within its type's rounding of want +- slack, infinities
    and NaN in the same places."""
    g = got.double()
    assert torch.equal(torch.isnan(g), torch.isnan(want)), "NaN in other places"
    lim = torch.finfo(got.dtype).max
    inf = torch.isinf(g)
    # beyond the largest number by less than the slack both answers are right
    near = want.abs() * (1 + ROUND[got.dtype]) + slack >= lim
    assert bool((~inf | near | torch.isinf(want)).all()), "infinities"
    winf = torch.isinf(want)
    assert torch.equal(g[winf], want[winf]), "infinities"
    ok = ~(inf | torch.isnan(g) | winf)
    err = (g - want).abs()
    tol = (slack + (want.abs() + slack) * ROUND[got.dtype] + TINY[got.dtype])
    bad = ok & ~(err <= tol)
    if bool(bad.any()):
        at = (err / tol).masked_fill(~ok, 0).argmax().item()
        raise AssertionError(f"{int(bad.sum())} of {bad.numel()} outside: got "
                             f"{g.flatten()[at].item()} want {want.flatten()[at].item()} "
                             f"tol {tol.flatten()[at].item() if tol.dim() else tol}")
