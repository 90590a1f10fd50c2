"""64-bit forms of the products of 16-bit operands, and their error bounds.

Bounds count roundings.  A sum of K products in fp32, in any order: K 2^-24 times the sum
of the absolute products.  An activation multiplies an error of its argument by its slope,
1.13 at most, and adds a few last places of fp32 of its own (8).  A result's rounding is half a
step, finfo.eps / 2 of the value, or half a subnormal's.  dz is rounded to the operands' type
before the two products of the backward pass: half a step of every term."""
import torch

from w4util import TINY, act64

U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
SLOPE = 1.13


def slope64(z, act):
    if act in (None, "none"):
        return torch.ones_like(z)
    if act == "relu":  # 0 at 0
        return torch.where(z.isnan(), z, (z > 0).double())
    z = z.detach().clone().requires_grad_(True)
    g, = torch.autograd.grad(act64(z, act).sum(), z)
    return g


def sums64(x, w, b):
    """z = x w^T + b and the bound of an fp32 sum's error."""
    x, w = x.double(), w.double()
    z, s = x @ w.t(), x.abs() @ w.abs().t()
    if b is not None:
        z, s = z + b.double(), s + b.double().abs()
    return z, (x.shape[1] + 1) * U * s


def rounding(v, dtype):
    return HALF[dtype] * v.abs() + TINY[dtype]


def linear64(x, w, b, act, r, dtype, pre=torch.float32):
    """(z, its bound as held in `pre`, y, its bound)."""
    z, e = sums64(x, w, b)
    y = act64(z, act)
    ey = SLOPE * e + 8 * U * y.abs()
    if r is not None:
        y = y + r.double()
        ey = ey + U * y.abs()
    return z, e + rounding(z.abs() + e, pre), y, ey + rounding(y.abs() + ey, dtype)


def gated64(x, w, b, act, dtype, pre=torch.float32):
    z, e = sums64(x, w, b)
    g, u = z.chunk(2, 1)
    eg, eu = e.chunk(2, 1)
    a = act64(g, act)
    ea = SLOPE * eg + 8 * U * a.abs()
    y = a * u
    ey = ea * u.abs() + a.abs() * eu + ea * eu + U * y.abs()
    return z, e + rounding(z.abs() + e, pre), y, ey + rounding(y.abs() + ey, dtype)


def dz64(dy, pre, act, gated):
    """dz from z as the forward pass left it, and the bound of its fp32 value's error."""
    dy = dy.double()
    if not gated:
        d = dy if pre is None else dy * slope64(pre.double(), act)
        # slope: 16 last places of 1.13 (its terms cancel near its zeros)
        return d, 16 * U * 1.13 * dy.abs()
    g, u = pre.double().chunk(2, 1)
    a = act64(g, act)
    d = torch.cat((dy * u * slope64(g, act), dy * a), 1)
    e = torch.cat((18 * U * 1.13 * (dy * u).abs(), 10 * U * (dy * a).abs()), 1)
    return d, e


def backward64(dy, x, w, pre, act, gated, grad_dtype):
    """{name: (value, bound)} of dx, dw, db."""
    dz, e = dz64(dy, pre, act, gated)
    # as the products read it: rounded to x's type
    er = e + rounding(dz.abs() + e, x.dtype)
    xd, wd = x.double(), w.double()
    M, rows = dz.shape

    def bound(prod, terms, n, dtype):
        e = terms + (n + 1) * U * (prod + terms)
        return lambda v: e + rounding(v.abs() + e, dtype)

    dx = dz @ wd
    dw = dz.t() @ xd
    db = dz.sum(0)
    return {
        "dx": (dx, bound(dz.abs() @ wd.abs(), er @ wd.abs(), rows, x.dtype)(dx)),
        "dw": (dw, bound(dz.abs().t() @ xd.abs(), er.t() @ xd.abs(), M, grad_dtype)(dw)),
        "db": (db, bound(dz.abs().sum(0), e.sum(0), M, grad_dtype)(db)),
    }


def check(name, got, want, bound):
    """got within bound of want, NaN where it is NaN, equal where infinite."""
    got = got.double()
    nan = want.isnan()
    assert bool((got.isnan() == nan).all()), f"{name}: NaN in other places"
    inf = want.isinf()
    assert bool((got[inf] == want[inf]).all()), f"{name}: infinities differ"
    ok = ~(nan | inf)
    err = (got - want).abs()[ok]
    over = err - bound[ok]
    assert err.numel() == 0 or float(over.max()) <= 0, (
        f"{name}: off by {float(err.max()):.3e}, {int((over > 0).sum())} of {err.numel()} past "
        f"their bound, worst ratio {float((err / bound[ok]).max()):.2f}")
