"""The oracle of matrices held in 8-bit floating point, against the format's own statements."""

import pytest
import torch

from oracle import fp8 as O

F64 = torch.float64


def test_codes_are_e4m3():
    t = O.e4m3_values()
    assert t[0] == 0 and t[1] == 2.0 ** -9 and t[8] == 2.0 ** -6 and t[126] == 448
    assert torch.equal(t.float(), torch.arange(127, dtype=torch.uint8).view(
        torch.float8_e4m3fn).float())


@pytest.mark.parametrize("K", [8, 128, 136, 640])
def test_rule(K):
    g = torch.Generator().manual_seed(K)
    x = torch.randn(33, K, generator=g, dtype=F64) * torch.logspace(-40, 37, 33, dtype=F64)[:, None]
    x[3] = 0
    x[4, ::3] = 0
    x = x.float()
    codes, b = O.quantise(x)
    v = O.values(codes, b)[:, :K]
    s = torch.ldexp(torch.ones((), dtype=F64), b.int() - 127).repeat_interleave(128, 1)[:, :K]
    top = torch.nn.functional.pad(x.double(), (0, -K % 128)).unflatten(1, (-1, 128)).abs().amax(-1)
    s1 = torch.ldexp(torch.ones((), dtype=F64), b.int() - 127)
    assert (top <= 448 * s1).all() and ((top > 224 * s1) | (b == 0)).all()
    assert ((v - x).abs() <= torch.maximum(2.0 ** -4 * x.abs().double(), 2.0 ** -10 * s)).all()


def test_rounding_is_torchs():
    """Codes in range round as torch's own conversion on the CPU does."""
    x = torch.linspace(-448, 448, 128 * 4001).view(-1, 128)
    x[:, 0] = 448
    codes, b = O.quantise(x)
    assert (b == 127).all()
    assert torch.equal(codes, x.to(torch.float8_e4m3fn).view(torch.uint8))


def test_no_numbers():
    x = torch.ones(4, 256)
    x[0, 3] = float("nan")
    x[1, 200] = float("inf")
    x[2, 0] = -float("inf")
    v = O.held(x)
    bad = torch.zeros(4, 256, dtype=torch.bool)
    bad[0, :128] = bad[1, 128:] = bad[2, :128] = True
    assert torch.equal(torch.isnan(v), bad) and (v[~bad] == 1).all()


@pytest.mark.parametrize("rows,K,pair", [(1, 8, False), (17, 520, False), (34, 136, True)])
def test_layout_holds_every_value_once(rows, K, pair):
    blocks = -(-K // 128)
    codes = (torch.arange(rows * blocks * 128) % 251 + 1).to(torch.uint8).view(rows, -1)
    scales = (torch.arange(rows * blocks) % 250 + 1).to(torch.uint8).view(rows, -1)
    c, s = O.pack(codes, scales, pair)
    assert torch.equal(c[c > 0].sort().values, codes.flatten().sort().values)
    assert torch.equal(s[s > 0].sort().values, scales.flatten().sort().values)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_finite_values_stay_finite(dtype):
    """Up to the type's largest, within 2^-4: no code stands for 2^128."""
    top = torch.finfo(dtype).max
    x = torch.tensor([top, -top, 248 * 2.0 ** 120, 247 * 2.0 ** 120, -255 * 2.0 ** 120, 1.0]).to(dtype)
    v = O.held(torch.cat((x, torch.zeros(2, dtype=dtype)))[None])[0, :6]
    assert torch.isfinite(v.to(dtype)).all()
    assert ((v - x.double()).abs() <= 2.0 ** -4 * x.double().abs())[:5].all() and v[5] == 0
    assert v[0] == 240 * 2.0 ** 120 == -v[1] == v[2] == v[3] == -v[4]
    below = torch.tensor([[224 * 2.0 ** 120, 2.0 ** 119, 256 * 2.0 ** 119]])
    assert (O.held(torch.nn.functional.pad(below, (0, 5)))[0, :3] == below.double()).all()
