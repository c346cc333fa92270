"""The 4-bit cache's quantiser and block format (CPU)."""

import math

import pytest
import torch

from kernel_optim_amd.kernels.kv4 import kv4_block_bytes
from oracle import kv4 as O

FORMATS = [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)]


@pytest.mark.parametrize("d,group", FORMATS)
def test_every_bit_of_a_block_belongs_to_one_value(d, group):
    at = O.places(d).flatten()
    nibbles = sorted((at // 4).tolist())
    assert (at % 4 == 0).all() and nibbles == list(range(2 * 32 * d))
    assert kv4_block_bytes(d, group) == 32 * d + 2 * 32 * (d // group) * 4


@pytest.mark.parametrize("d,group", FORMATS)
def test_pack_and_unpack(d, group):
    g = torch.Generator().manual_seed(d + group)
    cache = torch.randint(0, 256, (2, 3, 2, kv4_block_bytes(d, group)), generator=g,
                          dtype=torch.uint8)
    cache[..., 32 * d:] &= 0x3f   # scales that are numbers: bits survive the way through fp32
    assert torch.equal(O.pack(*O.unpack(cache, d, group)), cache)


@pytest.mark.parametrize("scale", [1e-30, 1e-3, 1.0, 300.0, 1e30])
@pytest.mark.parametrize("shift", [0.0, 0.7, -40.0])
def test_values_are_within_half_a_step(scale, shift):
    g = torch.Generator().manual_seed(1)
    x = ((torch.randn(200, 128, generator=g) + shift) * scale).to(O.BF16)
    n, s, c = O.quantise(x, 32)
    err = (O.values(n, s, c, 32) - x.double()).abs()
    # half a step, and up to 8 s 2^-8 where the rounded s falls short of the group's ends
    # (fp32's own roundings are below 2^-10 s for |x| < 2^13 s)
    step = s.double().repeat_interleave(32, -1)
    assert (err <= step * (0.5 + 2.0 ** -5 + 2.0 ** -10)).all()


def test_groups_that_hold_one_value_and_none():
    x = torch.tensor([0.0, -3.0, 1e-38, 3e38, 2.0 ** -133]).to(O.BF16)[:, None].expand(-1, 32)
    n, s, c = O.quantise(x, 32)
    # 7/15 x + 8/15 x is x up to fp32's rounding, which the rounding to bf16 takes back; the
    # subnormals are exact sums too
    assert torch.equal(O.values(n, s, c, 32), x.double())
    for bad in (math.nan, math.inf, -math.inf):
        y = torch.ones(2, 64)
        y[0, 40] = bad
        n, s, c = O.quantise(y, 32)
        v = O.values(n, s, c, 32)
        assert v[0, 32:].isnan().all() and not v[0, :32].isnan().any() and not v[1].isnan().any()


def test_attention_of_an_empty_row_is_zero():
    cache = torch.zeros(1, 1, 1, kv4_block_bytes(64, 64), dtype=torch.uint8)
    cache[..., 32 * 64:] = 0xff   # NaN everywhere: nothing may read it
    out, _, _ = O.attention(torch.ones(2, 64), cache, [0], 2, 1, 64, 64)
    assert (out == 0).all()
