"""dx and dw share a launch where neither alone is slowed much by its tiles there (no GPU): a
gradient asked for alone takes the same kernel as with the other."""
import ctypes

import pytest

import hipgemm_amd as hg


def plans(M, N, K, gated, dx=1, dw=1):
    return hg.linear_backward_select(hg.LinearGradDesc(
        size=ctypes.sizeof(hg.LinearGradDesc), M=M, N=N, K=K, gated=gated, type=1, dx=dx, dw=dw))


TOGETHER = ((128, 128, 1, 0),) * 2


@pytest.mark.parametrize("M,N,K,gated", ((1531, 2001, 1000, 0), (2048, 704, 1024, 1),
                                         (2048, 512, 1024, 0)))
def test_together(M, N, K, gated):
    assert plans(M, N, K, gated) == TOGETHER
    assert plans(M, N, K, gated, dw=0)[0] == plans(M, N, K, gated, dx=0)[1] == TOGETHER[0]


@pytest.mark.parametrize("M,N,K,gated", ((777, 1400, 1000, 1), (1024, 1408, 512, 1),
                                         (512, 4096, 512, 0)))
def test_long_sums_apart(M, N, K, gated):
    """dx's sum over N is long beside its tiles: in slices, with dw and without."""
    of_x, of_w = plans(M, N, K, gated)
    assert of_x[2] > 1 and of_w == TOGETHER[1]
    assert plans(M, N, K, gated, dw=0)[0] == of_x
