"""GPU: rows quantised behind a norm against the oracle's norm (statistics in 64 bits), code by code,
at sizes and eps that change the codes.

How many codes may differ. A block's sum of squares is fp32's, 12 roundings of at most 2^-24 each on the
way of any of its terms, and blocks add up in 64 bits: the inverse root is off by at most half of
that, 6 * 2^-24, and its own rounding, 2^-24; the product with x rounds once more: t = x * rstd is
within 8 * 2^-24 = 2^-21 of itself. A border between two bf16 values, which lie 2^-8 of themselves apart
or more, falls in between with probability 2^-13 at most. One bf16 step of t is at most two of the
value behind the gain (2^-6 of it), and codes lie 2^-4 of themselves apart or more: a code differs, by one,
with probability 2^-13 * 2^-6 / 2^-4 = 2^-15. Below a code's least normal value they lie further apart.
Of n codes at most n 2^-15 differ on average, and six deviations more in any one test. A block's scale
differs only where its largest value crosses a border, one in 2^7 bf16 values, and steps: 2^-20 of blocks.

An inverse root off by 2^-18 would change 2^-12 of the codes, eight times as many, eps left out
nearly all."""

import pytest
import torch

from kernel_optim_amd.kernels.fp8 import Fp8Linear, fp8_quantize, fp8_read
from kernel_optim_amd.kernels.gemv import EPI_F32
from oracle import fp8 as O

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def inputs(n, K, size, seed):
    g = torch.Generator().manual_seed(seed)
    x = size * torch.randn(n, K, generator=g) * (0.5 + torch.rand(n, 1, generator=g))
    x[:, ::41] *= 9
    return x.to(BF16), (1 + 0.3 * torch.randn(K, generator=g)).to(BF16)


def read_codes(t):
    """codes [rows, blocks * 128] and scale bytes [rows, blocks] of t, by the layout."""
    tiles, blocks = t.codes.shape[:2]
    # [tile, block, j, g, row, byte]: value 64 j + 16 g + byte
    c = t.codes.cpu().view(tiles, blocks, 2, 4, 16, 16).permute(0, 4, 1, 2, 3, 5)
    s = t.scales.cpu().view(tiles, -1, 16, 4).permute(0, 2, 1, 3)
    return (c.reshape(16 * tiles, -1)[:t.rows],
            s.reshape(16 * tiles, -1)[:t.rows, :blocks])


def compare(t, want):
    codes, scales = read_codes(t)
    wc, ws = O.quantise(want)
    same = (scales == ws).repeat_interleave(128, 1)
    assert (scales != ws).sum() <= 1 + scales.numel() * 2.0 ** -20
    off = same & (codes != wc)
    assert ((codes.int() - wc.int()).abs() <= 1)[same].all()
    mean = want.numel() * 2.0 ** -15
    assert off.sum() <= mean + 6 * mean ** 0.5 + 1, (int(off.sum()), mean)


# a workgroup for each row up to 3 * 2^20 values; beyond, one for each 16 rows, with 2 or 4 blocks a
# wavefront in registers or (the last) the rows read twice
SHAPES = [(1, 128), (7, 1000), (64, 2560), (33, 9736), (3, 65536), (1300, 2560), (400, 8192), (370, 8712)]


@pytest.mark.parametrize("n,K", SHAPES)
@pytest.mark.parametrize("size,eps", [(1e-3, 1e-6), (1.0, 0.5), (1e3, 1e-6), (1e-20, 1e-12)])
def test_codes_behind_a_norm(dev, n, K, size, eps):
    x, nw = inputs(n, K, size, n + K)
    compare(fp8_quantize(x.to(dev), nw=nw.to(dev), eps=eps), O.norm(x, nw, eps))


@pytest.mark.parametrize("M", [1, 3, 4, 5, 16, 40])
@pytest.mark.parametrize("K", [128, 2560, 4096, 4104])
@pytest.mark.parametrize("size,eps", [(1e-3, 1e-6), (1.0, 0.5)])
def test_rows_in_a_projection(dev, M, K, size, eps):
    """A projection on the identity gives the values that its rows are held as: up to 4 rows it
    quantises them itself, and must hold what fp8_quantize holds."""
    x, nw = inputs(M, K, size, M + K)
    xd, nd = x.to(dev), nw.to(dev)
    y, want = (torch.empty(M, K, device=dev) for _ in range(2))
    Fp8Linear(M, K, K, EPI_F32, True, eps=eps)(xd, fp8_quantize(torch.eye(K, device=dev)), y=y, nw=nd)
    t = fp8_quantize(xd, nw=nd, eps=eps)
    fp8_read(t, want)
    assert torch.equal(y, want)
    compare(t, O.norm(x, nw, eps))


@pytest.mark.parametrize("n", [1, 33])
def test_the_longest_rows(dev, n):
    """2^17 values; longer ones are refused."""
    x, nw = inputs(n, 2 ** 17, 1e-3, n)
    compare(fp8_quantize(x.to(dev), nw=nw.to(dev), eps=1e-6), O.norm(x, nw, 1e-6))
    x, nw = (torch.zeros(*s, dtype=BF16, device=dev) for s in ((n, 2 ** 17 + 8), (2 ** 17 + 8,)))
    with pytest.raises(ValueError):
        fp8_quantize(x, nw=nw)
