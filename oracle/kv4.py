"""Oracle of the 4-bit KV cache: its quantiser and block format in plain torch on the CPU, and the
attention over what a cache holds in 64 bits.

A group of `group` values of a head vector is held as x = c + s (n - 8), n = 0..15, s and c bf16
(kernel_optim_amd/kernels/kv4.py states the rule). `quantise` runs the rule in float32, one torch
operation per rounding, so the kernels' codes can be compared bit for bit where their
inputs are bf16."""

import math

import torch

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def quantise(x, group):
    """x [.., d] -> codes [.., d] (uint8), s and c [.., d / group] (float32 holding bf16)."""
    x = x.to(F32).unflatten(-1, (-1, group))
    lo, hi = x.amin(-1), x.amax(-1)
    c = (lo * (7 / 15) + hi * (8 / 15)).to(BF16).to(F32)
    # (c - lo) / 8 of the parts: the difference itself may pass fp32's range
    s = torch.maximum((hi - c) * (1 / 7), c * 0.125 - lo * 0.125).to(BF16).to(F32)
    bad = ~(torch.isfinite(lo) & torch.isfinite(hi))
    c, s = (t.masked_fill(bad, math.nan) for t in (c, s))
    s = s.masked_fill(s < 2.0 ** -126, 0.0)
    inv = torch.where(s == 0, torch.zeros_like(s), 1.0 / s)
    n = torch.round(((x - c[..., None]) * inv[..., None] + 8).clamp(0, 15)).nan_to_num(0)
    return n.to(torch.uint8).flatten(-2), s, c


def values(n, s, c, group, dtype=F64):
    """What codes, s and c stand for."""
    n = n.to(dtype).unflatten(-1, (-1, group)) - 8
    return (c.to(dtype)[..., None] + s.to(dtype)[..., None] * n).flatten(-2)


def read_back(n, s, c, group):
    """The bf16 that a read returns: a value that the step's rounding puts past bf16's largest
    comes back as that."""
    top = torch.finfo(BF16).max
    return values(n, s, c, group).clamp(-top, top).to(F32).to(BF16)


def places(d):
    """[2, 32, d]: the bit of a block at which the code of (K or V, key, column) begins."""
    key = torch.arange(32)[:, None]
    col = torch.arange(d)[None]
    k = 8 * (key * (d // 2) + col % 32 // 8 * (d // 8) + 4 * (col // 32)) + 4 * (col % 8 // 2) + 16 * (col % 2)
    j, n = 2 * (col // 32) + col % 2, col % 32 // 2
    v = 8 * (16 * d + ((key // 8 * (d // 64) + j // 4) * 16 + n) * 16 + key % 8 // 2 * 4)
    return torch.stack((k, v + 16 * (key % 2) + 4 * (j % 4)))


def unpack(cache, d, group):
    """cache [B, nkv, blocks, bytes] -> codes [2, B, nkv, keys, d], s and c [2, B, nkv, keys, NG]
    of K and V."""
    cache = cache.cpu()
    B, H, nb, _ = cache.shape
    at = places(d).flatten()
    n = (cache[..., at // 8] >> (at % 8).to(torch.uint8)) & 15
    n = n.view(B, H, nb, 2, 32, d).permute(3, 0, 1, 2, 4, 5).reshape(2, B, H, nb * 32, d)
    sc = cache[..., 32 * d:].contiguous().view(BF16).to(F32).view(B, H, nb, 2, d // group, 32, 2)
    sc = sc.permute(6, 3, 0, 1, 2, 5, 4).reshape(2, 2, B, H, nb * 32, d // group)
    return n, sc[0], sc[1]


def pack(n, s, c):
    """unpack's inverse."""
    _, B, H, rows, d = n.shape
    nb, ng = rows // 32, s.shape[-1]
    at = places(d).flatten()
    n = n.view(2, B, H, nb, 32, d).permute(1, 2, 3, 0, 4, 5).reshape(B, H, nb, -1)
    codes = torch.zeros(B, H, nb, 32 * d, dtype=torch.int32)
    codes.scatter_add_(-1, (at // 8).expand(B, H, nb, -1), n.to(torch.int32) << (at % 8).to(torch.int32))
    sc = torch.stack((s, c)).view(2, 2, B, H, nb, 32, ng).permute(2, 3, 4, 1, 6, 5, 0)
    sc = sc.to(BF16).contiguous().view(torch.uint8).reshape(B, H, nb, -1)
    return torch.cat((codes.to(torch.uint8), sc), -1)


def write(cache, k, v, start, lengths, group):
    """cache (CPU) with rows 0 .. lengths[b] - 1 of k, v [B, nkv, S, d] in the slots from start[b]."""
    d = k.shape[-1]
    n, s, c = (t.clone() for t in unpack(cache, d, group))
    for b in range(k.shape[0]):
        for i in range(min(lengths[b], k.shape[2])):
            slot = start[b] + i
            if 0 <= slot < n.shape[3]:
                for which, x in enumerate((k, v)):
                    n[which, b, :, slot], s[which, b, :, slot], c[which, b, :, slot] = quantise(
                        x[b, :, i].cpu(), group)
    return pack(n, s, c)


def norm_rope(x, w, cos, sin, eps):
    """RMSNorm with gain w and RoPE with rows cos, sin in 64 bits; x [.., d]."""
    x, d = x.to(F64), x.shape[-1]
    y = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.to(F64)
    half = torch.cat((-y[..., d // 2:], y[..., :d // 2]), -1)
    return y * cos.to(F64) + half * sin.to(F64)


def attention(q, cache, lens, T, nq, d, group):
    """q [B*T, nq*d]; query t of sequence b sees its keys below lens[b] - T + t + 1. Returns out
    [B*T, nq*d] in 64 bits and, per element, the sums over p of |s (n - 8)| and of |x| (what
    roundings of p are relative to)."""
    n, s, c = unpack(cache, d, group)
    B, H = cache.shape[:2]
    G = nq // H
    q = q.cpu().to(F64).view(B, T, H, G, d)
    out, step, size = (torch.zeros(B, T, H, G, d, dtype=F64) for _ in range(3))
    for b in range(B):
        for t in range(T):
            m = min(lens[b], n.shape[3]) - T + t + 1
            if m <= 0:
                continue
            k = values(n[0, b, :, :m], s[0, b, :, :m], c[0, b, :, :m], group)
            v = values(n[1, b, :, :m], s[1, b, :, :m], c[1, b, :, :m], group)
            p = torch.softmax(q[b, t] @ k.transpose(1, 2).contiguous() * d ** -0.5, -1)
            out[b, t] = p @ v
            dev = v - c[1, b, :, :m].to(F64).repeat_interleave(group, -1)
            step[b, t], size[b, t] = p @ dev.abs(), p @ v.abs()
    return tuple(x.reshape(B * T, nq * d) for x in (out, step, size))
