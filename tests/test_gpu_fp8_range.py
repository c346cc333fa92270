"""8-bit matrices at the ends of the value range, on the GPU: the largest finite values, and factors
below the least normal number."""

import pytest
import torch

from kernel_optim_amd.kernels.fp8 import Fp8Linear, fp8_quantize, fp8_read
from kernel_optim_amd.kernels.gemv import EPI_BF16, EPI_F32
from oracle import fp8 as O

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def tops(n, K, dtype):
    """Rows whose blocks' largest values run over the last binade, both signs, to the type's largest."""
    x = torch.randn(n, K, generator=torch.Generator().manual_seed(n + K)).double()
    for i in range(n):
        for j, k in enumerate(range(0, K, 128)):
            x[i, k + (37 * i + j) % min(128, K - k)] = (-1) ** i * 2.0 ** 127 * (1 + (i + j) % 32 / 32)
    x[0, 0], x[n - 1, K - 1] = torch.finfo(dtype).max, -torch.finfo(dtype).max
    return x.to(dtype)


# 5 rows of a row each, 400 of a wavefront a quad of blocks (more than 3 million values), and fp32
@pytest.mark.parametrize("n,K", [(5, 136), (33, 640), (400, 8192)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_finite_values_stay_finite(dev, n, K, dtype):
    x = tops(n, K, dtype)
    t = fp8_quantize(x.to(dev))
    codes, scales = O.pack(*O.quantise(x))
    assert torch.equal(t.codes.cpu(), codes) and torch.equal(t.scales.cpu(), scales)
    for out in (BF16, F32):
        y = torch.empty(n, K, dtype=out, device=dev)
        fp8_read(t, y)
        assert torch.isfinite(y).all()
        assert torch.equal(y.cpu(), O.held(x).to(out))


@pytest.mark.parametrize("n", [3, 300])
def test_behind_a_norm(dev, n):
    """A gain of the largest bf16: rows of +-1 (eps 0, a norm of exactly 1) become it throughout."""
    K = 256
    x = torch.where(torch.rand(n, K, generator=torch.Generator().manual_seed(n)) < 0.5, -1.0, 1.0)
    top = torch.finfo(BF16).max
    nw = torch.full((K,), top, dtype=BF16)
    t = fp8_quantize(x.to(BF16).to(dev), nw=nw.to(dev), eps=0.0)
    y = torch.empty(n, K, device=dev)
    fp8_read(t, y)
    assert torch.equal(y.cpu(), x * 240 * 2.0 ** 120)


@pytest.mark.parametrize("M", [1, 4, 16, 20, 33, 64, 100])
@pytest.mark.parametrize("epi", [EPI_F32, EPI_BF16])
def test_products_of_the_largest_values(dev, M, epi):
    """x at the top times a weight of 2^-120: finite, the same from 1 row to many, in each kernel's
    own quantiser and with x held."""
    K, N = 256, 32
    x = tops(M, K, BF16)
    w = torch.zeros(N, K)
    w[torch.arange(N), 8 * torch.arange(N)] = 2.0 ** -120
    wd = fp8_quantize(w.to(dev))
    want = (O.held(x) @ O.held(w).t()).to(F32 if epi == EPI_F32 else BF16)   # one product each: exact
    for given in (x.to(dev), fp8_quantize(x.to(dev))):
        y = torch.empty(M, N, dtype=want.dtype, device=dev)
        Fp8Linear(M, N, K, epi, False)(given, wd, y=y)
        assert torch.equal(y.cpu(), want)


@pytest.mark.parametrize("M", [1, 4, 16, 20, 33, 64, 100])
@pytest.mark.parametrize("epi", [EPI_F32, EPI_BF16])
def test_products_of_subnormal_values(dev, M, epi):
    """Factors of 2^-130, below the least normal fp32, times 2^126: 256 products of 2^-4 each."""
    K, N = 256, 32
    x = torch.full((M, K), 2.0 ** -130)
    w = torch.full((N, K), 2.0 ** 126)
    xd, wd = fp8_quantize(x.to(dev)), fp8_quantize(w.to(dev))
    for given in (xd, x.to(BF16).to(dev)):
        y = torch.empty(M, N, dtype=F32 if epi == EPI_F32 else BF16, device=dev)
        Fp8Linear(M, N, K, epi, False)(given, wd, y=y)
        assert (y == K * 2.0 ** -4).all()
