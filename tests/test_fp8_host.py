"""Refusals of the 8-bit matrices' ops that need no GPU: sizes, types, devices, and the C ABI's own
checks (no kernel is launched)."""

import pytest
import torch

from kernel_optim_amd import _lib
from kernel_optim_amd.kernels import fp8 as P
from kernel_optim_amd.kernels.gemv import EPI_ARGMAX, EPI_BF16, EPI_RESID, EPI_SWIGLU

BF16 = torch.bfloat16


def test_shapes():
    assert P.fp8_shape(17, 136) == (2, 2)
    assert P.fp8_shape(34, 128, pair=True) == (3, 1)
    t = P.fp8_empty(17, 640, "cpu")
    assert t.codes.shape == (2, 5, 2048) and t.scales.shape == (2, 2, 64)
    assert t.nbytes == 2 * 5 * 2048 + 2 * 2 * 64
    for bad in ((0, 8), (1, 0), (1, 12), (2 ** 31, 2 ** 12)):
        with pytest.raises(ValueError):
            P.fp8_shape(*bad)
    with pytest.raises(ValueError):
        P.fp8_shape(3, 8, pair=True)


def test_held_tensors_are_checked():
    t = P.fp8_empty(17, 640, "cpu")
    for codes, scales, rows in ((t.codes[:1], t.scales, 17), (t.codes, t.scales[:, :1], 17),
                                (t.codes.int(), t.scales, 17), (t.codes, t.scales, 33)):
        with pytest.raises(ValueError):
            P.Fp8Tensor(codes, scales, rows, 640)


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 128, dtype=BF16)
    t = P.fp8_empty(4, 128, "cpu")
    for f in (lambda: P.fp8_quantize(x), lambda: P.fp8_read(t, x),
              lambda: P.Fp8Linear(4, 4, 128, EPI_BF16, False)(x, t, y=x)):
        with pytest.raises(ValueError):
            f()


@pytest.mark.parametrize("M,N,K,epi", [(0, 8, 8, EPI_BF16), (1, 0, 8, EPI_BF16),
                                       (1, 8, 12, EPI_BF16), (1, 8, 8, EPI_ARGMAX)])
def test_linear_refuses(M, N, K, epi):
    with pytest.raises(ValueError):
        P.Fp8Linear(M, N, K, epi, False)


def test_c_abi_refuses():
    h, p = _lib.lib(), 1 << 20   # p is never read: the checks come first
    EINVAL, ERANGE, ENOTSUP = -22, -34, -95
    q = lambda x=p, f32=0, stride=8, rows=1, K=8, pair=0, nw=None, codes=p, scales=p: \
        h.ko_fp8_quantize(x, f32, stride, rows, K, pair, nw, 1e-6, codes, scales, None)
    assert q(x=None) == q(codes=None) == q(scales=None) == EINVAL
    assert q(x=p + 2) == q(codes=p + 8) == q(scales=p + 8) == q(nw=p + 2) == EINVAL
    assert q(rows=0) == q(K=12) == q(K=0) == q(stride=4) == q(stride=-8) == EINVAL
    assert q(rows=3, pair=1) == EINVAL
    assert q(nw=p, f32=1) == q(nw=p, pair=1, rows=2) == ENOTSUP
    assert q(rows=2 ** 31 - 1, K=2 ** 20) == ERANGE
    r = lambda codes=p, rows=1, K=8, out=p, stride=8: \
        h.ko_fp8_read(codes, p, rows, K, 0, out, 0, stride, None)
    assert r(codes=None) == r(out=None) == r(out=p + 4) == r(rows=0) == r(K=4) == r(stride=1) == EINVAL
    l = lambda t=p, n=1 << 40, x=None, nw=None, xc=p, y=p, hh=p, M=1, N=8, K=8, epi=EPI_BF16: \
        h.ko_fp8_linear(x, nw, 0.0, xc, p, p, p, y, hh, t, n, M, N, K, epi, None)
    assert l(x=p + 2) == l(nw=p) == l(x=p, nw=p + 2) == EINVAL
    assert l(xc=None) == l(y=None) == l(M=0) == l(N=0) == l(K=12) == EINVAL
    assert l(hh=None, epi=EPI_RESID) == l(hh=p + 2, epi=EPI_RESID) == EINVAL
    assert l(epi=EPI_ARGMAX) == l(epi=-1) == ENOTSUP
    assert l(N=2 ** 30) == ERANGE
    assert l(epi=EPI_SWIGLU, M=0) == EINVAL
    assert l(t=p + 4) == EINVAL
    need = h.ko_fp8_linear_scratch(64, 2560, 9728, EPI_RESID)
    assert need > 0 and l(M=64, N=2560, K=9728, epi=EPI_RESID, n=need - 1) == EINVAL
    assert l(M=64, N=2560, K=9728, epi=EPI_RESID, t=None) == EINVAL
    assert h.ko_fp8_linear_scratch(1, 2560, 9728, EPI_RESID) == 0
    for bad in ((0, 8, 8, 0), (1, 0, 8, 0), (1, 8, 12, 0), (1, 8, 8, 4), (1, 2 ** 30, 8, 0)):
        assert h.ko_fp8_linear_scratch(*bad) == -1


def test_linear_keeps_to_one_device():
    """Another device's call would free the workspace that captured calls use."""
    op = P.Fp8Linear(4, 32, 256, EPI_BF16, False)
    op._dev, op._xq = 0, object()
    made = op._xq
    assert op._workspace(0) is made
    with pytest.raises(ValueError):
        op._workspace(1)
    assert op._xq is made
    with pytest.raises(ValueError):
        P.Fp8Linear(4, 32, 256, EPI_BF16, False, device="cpu")


def test_sizes_past_32_bits_are_refused():
    """Rows and columns that a C int, or a byte's place in a tile as one, does not hold."""
    assert P.fp8_shape(1, 2 ** 27) == (1, 2 ** 20)
    for bad in ((1, 2 ** 27 + 8), (1, 2 ** 31 - 8), (1, 2 ** 32 + 8), (2 ** 31, 8), (2 ** 32 + 5, 8)):
        with pytest.raises(ValueError):
            P.fp8_shape(*bad)
    for M, N, K in ((1, 8, 2 ** 32 + 8), (2 ** 32 + 1, 8, 8), (1, 2 ** 32 + 8, 8), (1, 8, 2 ** 27 + 8)):
        with pytest.raises(ValueError):
            P.Fp8Linear(M, N, K, EPI_BF16, False)
    h, p, ERANGE = _lib.lib(), 1 << 20, -34   # p is never read: the checks come first
    K = 2 ** 27 + 8
    assert h.ko_fp8_quantize(p, 0, K, 1, K, 0, None, 1e-6, p, p, None) == ERANGE
    assert h.ko_fp8_read(p, p, 1, K, 0, p, 0, K, None) == ERANGE
    assert h.ko_fp8_linear(None, None, 0.0, p, p, p, p, p, None, p, 1 << 40, 1, 8, K, EPI_BF16,
                           None) == ERANGE
    assert h.ko_fp8_linear_scratch(1, 8, K, EPI_BF16) == -1
    # more threads than a grid has
    assert h.ko_fp8_quantize(p, 0, 8, 2 ** 30, 8, 0, None, 1e-6, p, p, None) == ERANGE
    assert h.ko_fp8_quantize(p, 1, 8, 2 ** 30, 8, 0, None, 1e-6, p, p, None) == ERANGE
    assert h.ko_fp8_quantize(p, 0, 8, 2 ** 30, 8, 0, p, 1e-6, p, p, None) == ERANGE
    assert h.ko_fp8_read(p, p, 2 ** 30, 8, 0, p, 0, 8, None) == ERANGE


def test_a_norm_of_longer_rows_is_refused():
    """As every bad argument by ValueError, when the object is made."""
    P.Fp8Linear(2, 8, 2 ** 17, EPI_BF16, True)
    P.Fp8Linear(2, 8, 2 ** 17 + 8, EPI_BF16, False)
    with pytest.raises(ValueError):
        P.Fp8Linear(2, 8, 2 ** 17 + 8, EPI_BF16, True)


def test_held_goes_without_a_norm():
    with pytest.raises(ValueError):
        P.Fp8Linear(4, 32, 256, EPI_BF16, True, held=True)
