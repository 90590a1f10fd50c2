"""w4_gemm of many rows where sums come out infinite or NaN: by the definition,
and in a time that is of the call's own order.

Tolerance of finite results: as in test_w4_gpu.py."""
import pytest
import torch

import w4util as u
from test_w4_gpu import plain

pytestmark = pytest.mark.gpu


@pytest.fixture()
def hg(gpu):
    import hipgemm_amd
    return hipgemm_amd


# Tiles of 16 rows by four waves along K, of several row tiles, and of 128 x 128.
@pytest.mark.parametrize("M,N", [(9, 70), (60, 4100), (200, 150), (131, 12300), (193, 12300)])
@pytest.mark.parametrize("fmt,group,scale,dtype", [
    ("int4", 128, "bfloat16", "bfloat16"), ("int4", 32, "float32", "float16"),
    ("fp4", 96, "float16", "bfloat16"), ("fp4", 32, "e8m0", "bfloat16")])
def test_by_definition(hg, M, N, fmt, group, scale, dtype):
    g = u.generator(M + group)
    K = 608
    x = torch.randn((M, K), generator=g, device="cuda").to(getattr(torch, dtype))
    w, s, z = u.four_bit(g, (N,), K, fmt, group, scale, fmt == "int4")
    inf, nan = float("inf"), float("nan")
    x[0, 300] = inf
    x[1] = nan
    x[2, [5, 590]] = torch.tensor([inf, -inf], dtype=x.dtype, device="cuda")
    x[3, [0, 607]] = torch.tensor([nan, inf], dtype=x.dtype, device="cuda")
    x[M - 1, 607] = -inf
    x[M // 2, 17], x[M // 2, 18] = torch.finfo(x.dtype).max / 16, torch.finfo(x.dtype).max / 8
    if s.dtype == torch.uint8:
        s[N - 1, 1] = 255  # NaN
    else:
        s[N - 1, 1] = inf
        s[N // 2, 0] = nan
    y = hg.w4_gemm(x, w, s, z, format=fmt, group_size=group, out_dtype=torch.float32)
    # term by term, for what the product makes of infinities and NaN
    wd = u.weights64(w, s, fmt, group, z)
    odd = [0, 1, 2, 3, M - 1]
    rest = [i for i in range(M) if i not in odd]
    for i in odd:
        t = (x[i].double() * wd).sum(1)
        slack = (x[i].double() * wd).abs().nan_to_num(0, 0, 0).sum(1) * 700 * 2.0 ** -24
        u.agree(y[i], t, slack)
    cols = [n for n in range(N) if n not in (N // 2, N - 1)]
    want, slack = plain(x[rest], w[cols], s[cols], None if z is None else z[cols], fmt, group,
                        None, None)
    u.agree(y[rest][:, cols], want, slack)
    for n in (N // 2, N - 1):
        t = (x[rest].double() * wd[n]).sum(1)
        u.agree(y[rest, n], t, (x[rest].double() * wd[n]).abs().nan_to_num(0, 0, 0).sum(1)
                * 700 * 2.0 ** -24)


def seconds(f):
    f()
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    a.record()
    f()
    b.record()
    b.synchronize()
    return a.elapsed_time(b) * 1e-3


def test_nan_takes_no_longer(hg):
    """Rows of NaN (an unset batch) cost one more look at x: a wave's row is read once
    more for each 16 columns, 1 / 16 and less of the products' work, not K steps per
    output of one lane.  10 times the call's time is far from both."""
    g = u.generator(2)
    M, N, K = 200, 1000, 4096
    x = torch.randn((M, K), generator=g, device="cuda").bfloat16()
    w, s, _ = u.four_bit(g, (N,), K, "int4", 128, "bfloat16", False)
    usual = min(seconds(lambda: hg.w4_gemm(x, w, s)) for _ in range(5))
    x.fill_(float("nan"))
    nan = min(seconds(lambda: hg.w4_gemm(x, w, s)) for _ in range(5))
    print(f"usual {usual * 1e6:.0f} us, NaN {nan * 1e6:.0f} us")
    assert bool(torch.isnan(hg.w4_gemm(x, w, s)).all())
    assert nan < 10 * max(usual, 15e-6)
