"""GPU: 8-bit matrices whose offsets pass 32 bits, and the longest rows. Small whole numbers: every code,
product and sum is exact (no sum passes 2^24, no product has bits 2^-13 below another), so results must
be equal whatever the order."""

import pytest
import torch

from kernel_optim_amd.kernels.fp8 import Fp8Linear, fp8_empty, fp8_quantize, fp8_read, fp8_slice
from kernel_optim_amd.kernels.gemv import EPI_BF16, EPI_F32

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def free():
    yield
    torch.cuda.empty_cache()


def whole(dev, seed, *shape, dtype=BF16):
    g = torch.Generator(device=dev).manual_seed(seed)
    return torch.randint(-8, 9, shape, generator=g, device=dev, dtype=torch.int8).to(dtype)


def test_a_weight_of_more_than_4_gib(dev):
    N, K = 540_000, 8200   # 4.5 GB of codes
    w = whole(dev, 1, N, K)
    t = fp8_quantize(w)
    assert t.codes.numel() > 2 ** 32
    back = torch.empty_like(w)
    fp8_read(t, back)
    assert torch.equal(back, w)
    last = torch.cat((w[:32], w[-64:])).cpu().double()
    del back
    for M, epi, dtype in ((1, EPI_F32, F32), (16, EPI_F32, F32), (20, EPI_F32, F32), (40, EPI_BF16, BF16),
                          (70, EPI_F32, F32), (70, EPI_BF16, BF16)):
        x = whole(dev, 2 + M, M, K)
        y = torch.empty(M, N, dtype=dtype, device=dev)
        Fp8Linear(M, N, K, epi, False)(x, t, y=y)
        want = (x.cpu().double() @ last.t()).to(dtype)
        assert torch.equal(torch.cat((y[:, :32], y[:, -64:]), 1).cpu(), want)


@pytest.mark.parametrize("epi,dtype", [(EPI_F32, F32), (EPI_BF16, BF16)])
def test_results_of_more_than_2_31_elements(dev, epi, dtype):
    M, N, K = 16_411, 131_003, 136
    x, w = whole(dev, 3, M, K), whole(dev, 4, N, K)
    y = torch.empty(M, N, dtype=dtype, device=dev)
    Fp8Linear(M, N, K, epi, False)(x, fp8_quantize(w), y=y)
    for a, b in ((slice(0, 64), slice(0, 64)), (slice(-64, None), slice(-64, None)),
                 (slice(-64, None), slice(0, 64))):
        want = (x[a].cpu().double() @ w[b].cpu().double().t()).to(dtype)
        assert torch.equal(y[a, b].cpu(), want)


@pytest.mark.parametrize("K", [2 ** 23 + 136, 2 ** 27])
def test_the_longest_rows(dev, K):
    """Rows of zeros but for their ends and a middle: 2^27 values are 2^20 blocks."""
    at = torch.tensor([0, 1, K // 2 - 1, K // 2, K - 9, K - 1], device=dev)
    for M, epi, dtype in ((1, EPI_F32, F32), (20, EPI_F32, F32), (20, EPI_BF16, BF16)):
        M = M if K < 2 ** 27 else min(M, 17)
        x, w = (torch.zeros(n, K, dtype=BF16, device=dev) for n in (M, 3))
        xs, ws = whole(dev, M, M, len(at)), whole(dev, M + 1, 3, len(at))
        x[:, at], w[:, at] = xs, ws
        t = fp8_quantize(w)
        back = torch.empty_like(w)
        fp8_read(t, back)
        assert torch.equal(back, w)
        y = torch.empty(M, 3, dtype=dtype, device=dev)
        Fp8Linear(M, 3, K, epi, False)(x, t, y=y)
        assert torch.equal(y.cpu(), (xs.cpu().double() @ ws.cpu().double().t()).to(dtype))


def test_many_long_rows(dev):
    """The tiled product over rows of 2^20 blocks: a byte's place in a tile ends just below 2^31."""
    M, N, K = 65, 3, 2 ** 27
    x = torch.zeros(1, K, dtype=BF16, device=dev)
    x[0, 5], x[0, -1] = 3, -7
    held = fp8_empty(M, K, dev)
    for i in range(0, M, 16):   # rows 16 at a time: 65 of them would be 17 GB in bf16
        n = min(16, M - i)
        fp8_quantize(x.expand(n, K), out=fp8_slice(held, i, i + n))
    w = torch.zeros(N, K, dtype=BF16, device=dev)
    w[:, 5], w[:, -1] = 2, torch.tensor([1.0, 2.0, 3.0], dtype=BF16, device=dev)
    t = fp8_quantize(w)
    for epi, dtype in ((EPI_F32, F32), (EPI_BF16, BF16)):
        y = torch.empty(M, N, dtype=dtype, device=dev)
        Fp8Linear(M, N, K, epi, False, device=dev)(held, t, y=y)
        assert torch.equal(y.cpu(), torch.tensor([[-1.0, -8.0, -15.0]], dtype=dtype).expand(M, N))
