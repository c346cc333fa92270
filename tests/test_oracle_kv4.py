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


BF16_MAX = torch.finfo(O.BF16).max


def top_groups():
    """Groups whose span passes fp32's range by up to twice, and groups of one sign near the largest
    value: [N, 32] bf16, both ends among them."""
    t = torch.cat((torch.linspace(2.9e38, BF16_MAX, 40), torch.tensor([1e38, 2.0 ** 120])))
    t = t.to(O.BF16).double()
    lo = torch.cat((-t, -t, -t, t[:20]))
    hi = torch.cat((t, t.flip(0), -t.flip(0) / 8, torch.full((20,), BF16_MAX, dtype=torch.float64)))
    lo, hi = torch.minimum(lo, hi), torch.maximum(lo, hi)
    # one whose code 0 lies past the largest value, where code 1 is more than half a step off
    lo = torch.cat((lo, torch.tensor([-3.3895313892515355e38])))
    hi = torch.cat((hi, torch.tensor([-3.083808950221005e38])))
    at = torch.linspace(0, 1, 32, dtype=torch.float64)
    return (lo[:, None] + (hi - lo)[:, None] * at).to(O.BF16)


def test_groups_at_the_top_of_the_range():
    """Any finite group is held within the bound of the others, and reads back finite."""
    x = top_groups()
    n, s, c = O.quantise(x, 32)
    assert s.isfinite().all() and c.isfinite().all()
    err = (O.values(n, s, c, 32) - x.double()).abs()
    assert (err <= s.double() * (0.5 + 2.0 ** -5 + 2.0 ** -10)).all()
    back = O.read_back(n, s, c, 32)
    assert back.isfinite().all()
    # clamping brings a value nearer; then bf16's rounding
    err = (back.double() - x.double()).abs()
    assert (err <= s.double() * (0.5 + 2.0 ** -5 + 2.0 ** -10) + x.double().abs() * 2.0 ** -8).all()
    for bad in (math.nan, math.inf, -math.inf):
        y = x.clone()
        y[:, 5] = bad
        assert O.read_back(*O.quantise(y, 32), 32).isnan().all()
