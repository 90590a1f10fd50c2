"""w4_gemm loses no more bits of int4 products in one kernel than in another.

The kernels sum the same exact products of codes (0-15) in fp32 and subtract the zero
point's share, in chains of like length (32 to 128 terms, then groups, lanes and
waves), so the same rows' rms errors are of one size whatever the number of rows; a
factor of 3 is left for the chains' lengths."""
import pytest
import torch

import hipgemm_amd as hg
import w4util as u

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("one_sided", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_errors_of_few_and_of_more_rows(gpu, dtype, one_sided, group, zeros):
    g = u.generator(1)
    N, K = 512, 4096
    w, s, z = u.four_bit(g, (N,), K, "int4", group, "float32", zeros)
    x = torch.randn((8, K), generator=g, device="cuda")
    x = (x.abs() if one_sided else x).to(dtype)
    want = x.double() @ u.weights64(w, s, "int4", group, z).T

    def error(rows):
        y = torch.cat([hg.w4_gemm(p, w, s, z, group_size=group, out_dtype=torch.float32)
                       for p in x.split(rows)])
        return (y - want).pow(2).mean().sqrt().item()

    tiles = error(8)
    for rows in (1, 2, 4):
        assert error(rows) <= 3 * tiles, (rows, error(rows) / want.pow(2).mean().sqrt().item())
