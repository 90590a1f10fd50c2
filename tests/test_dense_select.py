"""The choice of kernels of linear and gated_linear, from sizes alone (no GPU)."""
import ctypes

import pytest

import hipgemm_amd as hg


def forward(M, N, K, kind=0):
    return hg.LinearDesc(size=ctypes.sizeof(hg.LinearDesc), M=M, N=N, K=K, gated=int(kind == 2),
                         type=1, residual=int(kind == 1))


def backward(M, N, K, gated=0, dx=1, dw=1):
    return hg.LinearGradDesc(size=ctypes.sizeof(hg.LinearGradDesc), M=M, N=N, K=K, gated=gated,
                             type=1, dx=dx, dw=dw)


def test_known_choices():
    for kind in range(3):
        assert hg.linear_select(forward(1, 4096, 4096, kind))[0] == 0   # a few rows
        assert hg.linear_select(forward(64, 512, 256, kind))[0] == 0
        assert hg.linear_select(forward(65, 512, 256, kind))[:2] == (64, 128)
        assert hg.linear_select(forward(8192, 8192, 8192, kind))[:2] == (256, 256)
    assert hg.linear_select(forward(6000, 3000, 8192))[3] == 2560       # a full round, the rest
    assert hg.linear_backward_select(backward(8192, 8192, 8192)) == ((256, 256, 1, 0),) * 2


def test_workspace_is_for_slices():
    for M in (1, 17, 64, 65, 333, 2051):
        for N in (8, 264, 2056, 8200):
            for K in (8, 520, 4104):
                for kind in range(3):
                    d = forward(M, N, K, kind)
                    slices, first = hg.linear_select(d)[2:]
                    need = 4 * slices * M * (N - first) * (2 if kind == 2 else 1)
                    got = hg.linear_workspace_size(d)
                    assert got == 0 if slices == 1 else need <= got < need + 256, (M, N, K, kind)
                    assert 0 <= first < N and first % 128 == 0


def test_nothing_to_do():
    for M, N in ((0, 8), (8, 0)):
        assert hg.linear_select(forward(M, N, 8)) == (0, 0, 0, 0)
    assert hg.linear_backward_select(backward(8, 8, 8, dx=0))[0] == (0, 0, 0, 0)
    assert hg.linear_backward_select(backward(8, 8, 8, dw=0))[1] == (0, 0, 0, 0)
    assert hg.linear_backward_select(backward(0, 8, 8))[0] == (0, 0, 0, 0)


def test_refusals():
    for field, value in (("size", 8), ("M", -1), ("K", 12), ("type", 0), ("activation", 9),
                         ("gated", 2), ("M", 1 << 30 | 1)):
        for d, f in ((forward(8, 8, 8), hg.linear_select),
                     (backward(8, 8, 8), hg.linear_backward_select)):
            setattr(d, field, value)
            with pytest.raises(hg.HipGemmError):
                f(d)
    d = forward(8, 12, 8, 2)  # gated: N a multiple of 8
    with pytest.raises(hg.HipGemmError):
        hg.linear_select(d)
    assert hg.lib().hipgemm_linear_select(ctypes.byref(forward(8, 8, 8)), None) == 1


def test_packed_descriptor():
    """The calls' packed bytes are the structure's."""
    from hipgemm_amd.dense import _linear_desc
    values = [ctypes.sizeof(hg.LinearDesc)] + [3 + 1000 ** 3 * i for i in range(13)]
    values += list(range(100, 110))
    assert len(values) == len(hg.LinearDesc._fields_)
    assert _linear_desc(*values) == bytes(hg.LinearDesc(*values))
    from hipgemm_amd.dense import _grad_desc
    values = [ctypes.sizeof(hg.LinearGradDesc)] + [3 + 1000 ** 3 * i for i in range(15)]
    values += list(range(100, 111))
    assert len(values) == len(hg.LinearGradDesc._fields_)
    assert _grad_desc(*values) == bytes(hg.LinearGradDesc(*values))


def test_backward_workspace_by_kind():
    """The cached sizes are those of the descriptors themselves."""
    from hipgemm_amd.dense import _backward_bytes
    size = ctypes.sizeof(hg.LinearGradDesc)
    for M, N, K in ((1, 8, 8), (77, 264, 520), (333, 2056, 4104), (2051, 520, 264)):
        for act, gated, dyt in ((0, 0, 1), (2, 0, 1), (0, 0, 0), (2, 1, 1)):
            for dy in (4096, 4098, 4104):
                for lddy in (N, N + 8, N + 1, (1 << 21) + 8):
                    for needs in ((1, 1, 1), (1, 0, 0), (0, 1, 0), (0, 0, 1)):
                        d = hg.LinearGradDesc(size=size, M=M, N=N, K=K, gated=gated, type=1,
                                              activation=act, dy_type=dyt, dy=dy, lddy=lddy,
                                              dx=needs[0], dw=needs[1], db=needs[2])
                        whole = lddy % 8 == 0 and lddy <= 1 << 21
                        got = _backward_bytes(M, N, K, bool(gated), 1, act, dyt, dy % 16 == 0,
                                              whole, *map(bool, needs), 0)
                        assert got == hg.linear_backward_workspace_size(d)
