"""Refusals of the 4-bit cache's ops that need no GPU: sizes, types, devices, and the C ABI's own
checks (no kernel is launched)."""

import pytest
import torch

from kernel_optim_amd import _lib
from kernel_optim_amd.kernels import kv4 as K


def test_formats():
    assert K.kv4_block_bytes(128, 32) == 5120 and K.kv4_block_bytes(64, 64) == 2304
    for d, group in ((96, 32), (128, 16), (64, 128), (256, 64)):
        with pytest.raises(ValueError):
            K.kv4_block_bytes(d, group)
    assert len(K._FORMATS) == 5   # every block size names one format


def test_caches():
    c = K.kv4_cache(2, 3, 33, 128, "cpu", group=64, layers=4)
    assert c.shape == (4, 2, 3, 2, 4608) and c.dtype == torch.uint8
    assert K.kv4_cache(1, 1, 1, 64, "cpu").shape == (1, 1, 1, 2560)
    for bad in ((0, 1, 1), (1, 0, 1), (1, 1, 0)):
        with pytest.raises(ValueError):
            K.kv4_cache(*bad, 128, "cpu")


@pytest.mark.parametrize("kw", [dict(T=0), dict(T=9), dict(nq=7, nkv=2), dict(B=0), dict(cap=0),
                                dict(d=96), dict(group=16), dict(T=8, nq=18, nkv=2),
                                dict(nq=65, nkv=1), dict(device="cpu")])
def test_attention_refuses(kw):
    args = dict(B=1, T=1, cap=32, nq=8, nkv=2, d=128, device="cuda:0", group=32) | kw
    with pytest.raises(ValueError):
        K.Kv4Attention(**args)


def test_cpu_tensors_are_refused():
    c = K.kv4_cache(1, 1, 32, 128, "cpu")
    x = torch.zeros(1, 1, 4, 128, dtype=torch.bfloat16)
    for f, args in ((K.kv4_write, (x, x, c)), (K.kv4_read, (c, x, x))):
        with pytest.raises(ValueError):
            f(*args)
    with pytest.raises(ValueError):
        K.kv4_append(x, x, x, x, x, x, x, c, 1, 1e-6, 1, 1, 128)


def test_elements_that_share_memory():
    K._no_overlap(torch.zeros(2, 3, 4, 8).transpose(0, 2), "t")
    K._no_overlap(torch.zeros(4, 8)[:, ::2], "t")
    K._no_overlap(torch.zeros(1, 8).expand(1, 8), "t")
    for t in (torch.zeros(1, 8).expand(2, 8), torch.zeros(20).as_strided((4, 8), (4, 1)),
              torch.zeros(20).as_strided((3, 2, 2), (1, 2, 8))):
        with pytest.raises(ValueError):
            K._no_overlap(t, "t")


# A pointer that the host never follows: the calls below are refused before a launch.
P = 1 << 20
ROWS = dict(k=P, kb=128, kh=128, ks=128, v=P, vb=128, vh=128, vs=128, cache=P, cb=5120, ch=5120,
            start=None, lengths=None, B=1, S=1, nkv=1, cap=32, d=128, group=32)


@pytest.mark.parametrize("kw,status", [
    (dict(k=None), -22), (dict(v=None), -22), (dict(cache=None), -22), (dict(B=0), -22),
    (dict(S=0), -22), (dict(nkv=0), -22), (dict(cap=0), -22), (dict(d=96), -95),
    (dict(group=16), -95), (dict(d=64, group=128), -95), (dict(k=P + 8), -22),
    (dict(cache=P + 8), -22), (dict(cb=5121), -22), (dict(ks=4), -22),
    (dict(B=1 << 16, nkv=1 << 16), -34), (dict(S=2 ** 31 - 1, B=2), -34)])
def test_c_rows_refused(kw, status):
    a = ROWS | kw
    h = _lib.lib()
    kv = [a[x] for x in ("k", "kb", "kh", "ks", "v", "vb", "vh", "vs")]
    c = [a[x] for x in ("cache", "cb", "ch")]
    rest = [a[x] for x in ("start", "lengths", "B", "S", "nkv", "cap", "d", "group")]
    assert h.ko_kv4_write(*kv, *c, *rest, None) == status
    assert h.ko_kv4_read(*c, *kv, *rest, None) == status


@pytest.mark.parametrize("kw,status", [
    (dict(qkv=None), -22), (dict(cache=None), -22), (dict(M=0), -22), (dict(T=0), -22),
    (dict(M=3, T=2), -22), (dict(nq=0), -22), (dict(nkv=0), -22), (dict(max_pos=0), -22),
    (dict(M=2, T=2, rope=P), -22), (dict(rope=P + 8), -22), (dict(d=80), -95), (dict(cache=P + 4), -22), (dict(cb=8), -22), (dict(M=1 << 30), -34)])
def test_c_append_refused(kw, status):
    a = dict(qkv=P, q_w=P, k_w=P, cos=P, sin=P, pos=P, q_out=P, cache=P, M=1, T=1, cb=5120, ch=5120,
             eps=1e-6, nq=4, nkv=1, d=128, group=32, max_pos=32, rope=None) | kw
    assert _lib.lib().ko_kv4_append(*a.values(), None) == status


def test_c_attention_refused():
    h = _lib.lib()
    base = dict(q=P, cache=P, cb=5120, ch=5120, lens=P, off=0, cap=32, B=1, T=1, nq=4, nkv=1, d=128,
                group=32, scale=0.1, part=P, part_len=1 << 30, counters=P, grid=512, min_run=8,
                out=P)
    for kw, status in ((dict(q=None), -22), (dict(lens=None), -22), (dict(counters=None), -22),
                       (dict(T=0), -22), (dict(grid=0), -22), (dict(min_run=0), -22),
                       (dict(cap=0), -22), (dict(nq=5, nkv=2), -95), (dict(T=8, nq=9), -95),
                       (dict(d=100), -95), (dict(q=P + 2), -22), (dict(ch=4), -22),
                       (dict(part_len=100), -34), (dict(grid=1 << 21), -34),
                       (dict(B=1 << 20, cap=1 << 20), -34)):
        assert h.ko_kv4_attn(*(base | kw).values(), None) == status, kw
    assert h.ko_kv4_attn_scratch(4, 128, 32, 512) == 2 * 512 * 4 * 130
    assert h.ko_kv4_attn_scratch(33, 64, 32, 10) == 2 * 10 * 64 * 66
    for bad in ((0, 128, 32, 1), (65, 128, 32, 1), (4, 96, 32, 1), (4, 128, 32, 0)):
        assert h.ko_kv4_attn_scratch(*bad) == -1


def test_more_steps_than_the_kernel_counts_are_refused():
    # 64 x 8 pairs of 32768 blocks: 2^24 steps
    with pytest.raises(ValueError, match="24"):
        K.Kv4Attention(64, 1, 1 << 20, 32, 8, 128, "cuda:0")
    kw = dict(q=P, cache=P, cb=5120, ch=5120, lens=P, off=0, T=1, nq=32, nkv=8, d=128, group=32,
              scale=0.1, part=P, part_len=1 << 40, counters=P, grid=512, min_run=8, out=P)
    a = {k: kw.get(k) for k in ("q", "cache", "cb", "ch", "lens", "off", "cap", "B", "T", "nq", "nkv",
                                "d", "group", "scale", "part", "part_len", "counters", "grid",
                                "min_run", "out")} | dict(cap=1 << 20, B=64)
    assert _lib.lib().ko_kv4_attn(*a.values(), None) == -34


def test_tensors_that_meet():
    """_meet against the elements' addresses, over offsets and layouts."""
    hold = torch.arange(500)
    layouts = [((2, 3, 2, 4), s) for s in ((24, 8, 4, 1), (48, 8, 4, 1), (48, 4, 12, 1), (24, 4, 12, 1),
                                           (12, 24, 4, 1))]
    layouts += [((1, 3, 1, 4), (7, 12, 5, 1)), ((1, 1, 1, 4), (1, 1, 1, 1))]
    for shape, strides in layouts:
        a = hold.as_strided(shape, strides, 100)
        for offset in range(250):
            b = hold.as_strided(shape, strides, offset)
            meet = bool(set(a.flatten().tolist()) & set(b.flatten().tolist()))
            assert K._meet(a, b) == K._meet(b, a) == meet, (strides, offset)
