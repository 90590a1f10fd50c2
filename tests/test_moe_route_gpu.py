"""moe_route against its definition: ids exactly, weights in 64 bits.

Tolerance of the weights: exp of a difference of fp32 numbers (its argument
rounded once: |l - max| 2^-24 relative in the result), exp itself, a sum of up to
1024 terms, a division and a product: |l - max| + 16 roundings for the sums of
tree depth <= 16, and the smallest normal number for what underflows."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def plain(logits, k, scoring, renormalize, scale):
    l = logits.double()
    order = torch.sort(l, dim=1, descending=True, stable=True)
    vals, ids = order.values[:, :k], order.indices[:, :k]
    chosen = vals > float("-inf")
    ref = torch.where(torch.isinf(l.amax(1, keepdim=True)), 0.0, l.amax(1, keepdim=True))
    if scoring == "softmax":
        p, total = torch.exp(vals - ref), torch.exp(l - ref).sum(1, keepdim=True)
    else:
        p, total = torch.sigmoid(vals), torch.ones_like(ref)
    p = torch.where(chosen, p, 0.0)
    if renormalize:
        total = p.sum(1, keepdim=True)
    w = torch.where(chosen, p / total * scale, 0.0)
    dist = torch.where(chosen, (vals - ref).abs() + vals.abs(), 0.0)
    return w, torch.where(chosen, ids, -1).int(), dist


def check(hg, logits, k, scoring="softmax", renormalize=True, scale=1.0):
    w, ids = hg.moe_route(logits, k, scoring=scoring, renormalize=renormalize, scale=scale)
    want, wids, dist = plain(logits, k, scoring, renormalize, scale)
    assert w.dtype == torch.float32 and ids.dtype == torch.int32
    assert torch.equal(ids, wids)
    tol = want.abs() * (dist + 16) * 2.0 ** -24 + 2.0 ** -126
    err = (w.double() - want).abs()
    assert bool((err <= tol).all()), (err / tol).max().item()


@pytest.fixture()
def hg(gpu):
    import hipgemm_amd
    return hipgemm_amd


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 64, 8), (3, 5, 5), (2, 200, 16), (7, 33, 2),
                                   (5, 512, 10), (4, 1024, 64), (65, 100, 1), (130, 256, 8),
                                   (4096, 8, 2), (5000, 60, 6), (4100, 256, 8), (4097, 511, 16),
                                   (4096, 130, 64)])
def test_choice(hg, T, E, k, dtype):
    g = torch.Generator(device="cuda").manual_seed(T + E)
    l = (torch.randn((T, E), generator=g, device="cuda") * 3).to(dtype)
    for scoring in ("softmax", "sigmoid"):
        for renorm in (False, True):
            check(hg, l, k, scoring, renorm, 1.0 if renorm else 2.5)


@pytest.mark.parametrize("T", [9, 4500])
def test_ties_go_to_the_lower_index(hg, T):
    g = torch.Generator(device="cuda").manual_seed(2)
    l = torch.randint(-2, 2, (T, 96), generator=g, device="cuda").float()
    l[1] = 0.0
    l[2, ::2] = -0.0  # equal to 0
    l[2, 1::2] = 0.0
    check(hg, l, 12)
    check(hg, l.bfloat16(), 16)


@pytest.mark.parametrize("T", [6, 4200])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_masked(hg, T, scoring):
    """-inf is never chosen; rows with fewer than k others, and with none."""
    g = torch.Generator(device="cuda").manual_seed(3)
    l = torch.randn((T, 40), generator=g, device="cuda")
    l[:, 7:30] = float("-inf")
    l[1] = float("-inf")
    l[2, 1:] = float("-inf")
    l[3, 4:] = float("-inf")
    for renorm in (True, False):
        check(hg, l, 8, scoring, renorm)
    w, ids = hg.moe_route(l, 8, scoring=scoring)
    assert bool((ids[1] == -1).all()) and bool((w[1] == 0).all())
    assert ids[2].tolist() == [0] + [-1] * 7


def test_extreme_values(hg):
    l = torch.tensor([[3e38, -3e38, 0, 1e30], [-3e38, -2e38, -1e38, -3.4e38],
                      [1e-40, -1e-40, 0, 2e-40]], device="cuda")
    w, ids = hg.moe_route(l, 4)
    assert ids.tolist() == [[0, 3, 2, 1], [2, 1, 0, 3], [3, 0, 2, 1]]
    assert w[0].tolist() == [1, 0, 0, 0] and w[1].tolist() == [1, 0, 0, 0]
    w, ids = hg.moe_route(torch.tensor([[1.0, float("nan"), float("inf"), 2.0]], device="cuda"), 3)
    assert ids.tolist() == [[1, 2, 3]] and bool(torch.isnan(w).all())


def test_strided_rows_and_stream(hg):
    g = torch.Generator(device="cuda").manual_seed(4)
    wide = torch.randn((50, 77), generator=g, device="cuda")
    check(hg, wide[:, 3:70], 5)
    check(hg, wide[::2, 1:65], 5)
    check(hg, wide.bfloat16()[:, 5:40], 5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    a = hg.moe_route(wide, 4, stream=side)
    torch.cuda.synchronize()
    b = hg.moe_route(wide, 4)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_empty(hg):
    w, ids = hg.moe_route(torch.empty((0, 8), device="cuda"), 2)
    assert w.shape == ids.shape == (0, 2)


@pytest.mark.parametrize("make", [
    lambda: (torch.zeros(8), 2), lambda: (torch.zeros((2, 8)), 2),
    lambda: (torch.zeros((2, 8), device="cuda"), 9),
    lambda: (torch.zeros((2, 8), device="cuda"), 0),
    lambda: (torch.zeros((2, 1025), device="cuda"), 2),
    lambda: (torch.zeros((2, 128), device="cuda"), 65),
    lambda: (torch.zeros((2, 8), device="cuda", dtype=torch.float64), 2),
    lambda: (torch.zeros((8, 4), device="cuda").t(), 2),
])
def test_refusals(hg, make):
    with pytest.raises(hg.HipGemmError):
        hg.moe_route(*make())


def test_refuses_scoring(hg):
    with pytest.raises(hg.HipGemmError):
        hg.moe_route(torch.zeros((2, 8), device="cuda"), 2, scoring="max")
