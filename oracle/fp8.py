"""Oracle of matrices held in 8-bit floating point: the quantiser in plain arithmetic on the CPU
in 64 bits, the block layout by index, and the projections over the held values.

kernel_optim_amd/kernels/fp8.py states the rule: a block of 128 values of a row has the least power
of two s >= 2^-127 with max |x| <= 448 s, and holds x / s rounded to e4m3, but 240 where that
gives 256 and s is 2^120 (256 s is past fp32's largest)."""

import torch

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
BLOCK = 128


def e4m3_values():
    """The 127 finite values of a code's lower 7 bits (0x7f is NaN), by the format's definition."""
    c = torch.arange(127)
    e, m = c >> 3, (c & 7).to(F64)
    return torch.where(e == 0, m * 2.0 ** -9, (8 + m) * torch.ldexp(torch.ones(127, dtype=F64), e - 10))


def quantise(x):
    """x [rows, K] -> codes [rows, blocks * 128] uint8, scale bytes [rows, blocks] uint8."""
    rows, K = x.shape
    g = torch.nn.functional.pad(x.to(F64), (0, -K % BLOCK)).unflatten(1, (-1, BLOCK))
    top = g.abs().amax(-1)
    bad = ~torch.isfinite(g).all(-1)
    s = torch.ldexp(torch.ones((), dtype=F64), torch.arange(-127, 121))   # every scale there is
    b = torch.searchsorted(448 * s, torch.where(bad, 0.0, top))            # the first >= top
    v = torch.where(bad[..., None], 0.0, g / s[b][..., None])
    table = e4m3_values()
    mid = (table[1:] + table[:-1]) / 2
    c = torch.searchsorted(mid, v.abs())             # ties: the lower code,
    tie = (c < 126) & (v.abs() == mid[c.clamp_max(125)])
    c = torch.where(tie & (c % 2 == 1), c + 1, c)    # unless the upper one is even
    c = torch.where((b[..., None] == 247) & (c == 0x78), 0x77, c)   # 256 -> 240
    c = torch.where(torch.signbit(v), c + 128, c)
    c = torch.where(bad[..., None], 0x7f, c)
    return c.to(torch.uint8).flatten(1), torch.where(bad, 255, b).to(torch.uint8)


def values(codes, scales):
    """What codes and scales stand for, fp64 [rows, blocks * 128]."""
    table = torch.cat((e4m3_values(), torch.full((1,), float("nan"), dtype=F64)))
    v = table[(codes & 127).long()]
    v = torch.where(codes >= 128, -v, v)
    s = torch.where(scales == 255, float("nan"),
                    torch.ldexp(torch.ones((), dtype=F64), scales.int() - 127))
    return v * s.repeat_interleave(BLOCK, 1)


def binades(codes, scales):
    """Each value's 2^exponent (of the code, -6 for codes below 2^-6; 0 for a zero) times its scale."""
    e = torch.ldexp(torch.ones((), dtype=F64), (((codes & 127) >> 3).int() - 7).clamp_min(-6))
    s = torch.ldexp(torch.ones((), dtype=F64), scales.int() - 127).repeat_interleave(BLOCK, 1)
    return torch.where(codes & 127 == 0, 0.0, e * s)


def held(x):
    """The values that 8 bits hold of x [rows, K], fp64."""
    return values(*quantise(x))[:, :x.shape[1]]


def norm(x, w, eps):
    """The bf16 chain's RMSNorm with fp64 statistics."""
    t = (x.to(F64) * torch.rsqrt(x.to(F64).square().mean(-1, keepdim=True) + eps)).to(BF16)
    return (w.to(F64) * t.to(F64)).to(BF16)


def pack(codes, scales, pair=False):
    """The bytes of a matrix: codes [tiles, blocks, 2048] and scales [tiles, quads, 64], byte by byte
    as kernel_optim_amd/csrc/fp8_core.h places them."""
    halves = 2 if pair else 1
    n = codes.shape[0] // halves
    blocks = scales.shape[1]
    T = -(-n // (16 // halves))
    out = torch.zeros(T, blocks, 2048, dtype=torch.uint8)
    sc = torch.zeros(T, -(-blocks // 4), 64, dtype=torch.uint8)
    k = torch.arange(blocks * 128)
    kb, j, g, i = k // 128, k % 128 // 64, k % 64 // 16, k % 16
    b = torch.arange(blocks)
    for row in range(codes.shape[0]):
        h, m = divmod(row, n)
        t, r = (m // 8, 8 * h + m % 8) if pair else (m // 16, m % 16)
        out[t, kb, 1024 * j + 16 * (16 * g + r) + i] = codes[row]
        sc[t, b // 4, 4 * r + b % 4] = scales[row]
    return out, sc


def linear(x, w, epi, h=None):
    """x [M, K] W [N, K]^T in fp64 over held values (fp64), with the epilogue "f32" | "bf16" (none),
    "resid" or "swiglu" without the bf16 chain's roundings; and the sums' terms' magnitudes."""
    y, size = x @ w.t(), x.abs() @ w.abs().t()
    if epi == "resid":
        return h.to(F64) + y, size, y
    if epi == "swiglu":
        n = w.shape[0] // 2
        g, u = y[:, :n], y[:, n:]
        return g / (1 + torch.exp(-g)) * u, (size[:, :n], size[:, n:]), (g, u)
    return y, size, y
