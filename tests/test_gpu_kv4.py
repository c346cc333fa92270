"""The 4-bit KV cache on the GPU against the oracle: writes bit for bit, values read back, and
attention over what the cache holds in 64 bits."""

import math

import pytest
import torch

from kernel_optim_amd.kernels.kv4 import (KV4_KEYS, Kv4Attention, kv4_append, kv4_block_bytes,
                                          kv4_cache, kv4_read, kv4_write)
from kernel_optim_amd.kernels.fused import rope_rows
from oracle import kv4 as O
from tests.test_oracle_kv4 import top_groups

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
FORMATS = [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def junk(shape, seed):
    """Bytes of a used cache: any codes, scales that are no numbers."""
    t = torch.randint(0, 256, shape, generator=gen(seed), dtype=torch.uint8)
    d = {kv4_block_bytes(d, g): d for d, g in FORMATS}[shape[-1]]
    t[..., 32 * d:] = 0xff
    return t


def randn(seed, *shape):
    return torch.randn(*shape, generator=gen(seed))


def rows(seed, B, H, S, d):
    """K or V rows with strong channels and small tokens among them."""
    x = randn(seed, B, H, S, d)
    x[..., ::17] *= 9
    x[:, :, ::5] *= 1e-4
    return x.to(BF16)


def filled(B, H, cap, d, group, lens, seed):
    """A cache with lens[b] keys of sequence b, and no numbers behind them."""
    k, v = (rows(seed + i, B, H, cap, d) for i in range(2))
    (nk, sk, ck), (nv, sv, cv) = O.quantise(k, group), O.quantise(v, group)
    pad = -cap % 32
    stack = lambda a, b: torch.nn.functional.pad(torch.stack((a, b)), (0, 0, 0, pad))
    n, s, c = stack(nk, nv), stack(sk, sv), stack(ck, cv)
    for b, m in enumerate(lens):
        s[:, b, :, m:] = c[:, b, :, m:] = math.nan
    return O.pack(n, s, c)


# ---------------------------------------------------------------------------
# Writing and reading.
# ---------------------------------------------------------------------------
CASES = [  # B, nkv, S, blocks, start, lengths
    (1, 1, 1, 1, [0], None),
    (2, 3, 32, 2, [0, 32], None),
    (3, 2, 45, 4, [7, 0, 64], [45, 3, 0]),
    (2, 1, 100, 3, [-5, 61], [100, 99]),       # rows in front of the cache and behind it
    (2, 2, 17, 2, [63, 64], None),             # the last slot; none
    (1, 2, 200, 9, [31], [1000]),
]


@pytest.mark.parametrize("d,group", FORMATS)
@pytest.mark.parametrize("case", range(len(CASES)))
def test_write_and_read(dev, d, group, case):
    B, H, S, nb, start, lengths = CASES[case]
    k, v = rows(1, B, H, S, d), rows(2, B, H, S, d)
    old = junk((B, H, nb, kv4_block_bytes(d, group)), 3)
    want = O.write(old, k, v, start, lengths or [S] * B, group)
    cache = old.to(dev)
    st = torch.tensor(start, dtype=torch.int32, device=dev)
    ln = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=dev)
    kv4_write(k.to(dev), v.to(dev), cache, start=st, lengths=ln)
    assert torch.equal(cache.cpu(), want)
    ko, vo = (torch.full((B, H, S, d), 7.0, dtype=BF16, device=dev) for _ in range(2))
    kv4_read(cache, ko, vo, start=st, lengths=ln)
    n, s, c = O.unpack(want, d, group)
    held = O.values(n, s, c, group).to(torch.float32).to(BF16)
    for i, got in enumerate((ko.cpu(), vo.cpu())):
        expect = torch.full_like(got, 7.0)
        for b in range(B):
            for r in range(min(S, lengths[b] if lengths else S)):
                if 0 <= start[b] + r < nb * KV4_KEYS:
                    expect[b, :, r] = held[i, b, :, start[b] + r]
        assert torch.equal(got, expect)


@pytest.mark.parametrize("d,group", [(128, 32), (64, 64)])
def test_strided_rows_and_caches(dev, d, group):
    B, H, S = 2, 3, 50
    k, v = rows(4, B, S, H, d).transpose(1, 2), rows(5, B, H, S + 6, d)[:, :, 3:-3]
    size = kv4_block_bytes(d, group)
    big = junk((B, 2, H, 3, size), 6)
    want = big.clone()
    want[:, 1] = O.write(big[:, 1].contiguous(), k, v, [0] * B, [S] * B, group)
    got = big.to(dev)
    wide = torch.zeros(B, H, S + 6, d, dtype=BF16, device=dev)
    wide[:, :, 3:-3] = v.to(dev)
    kd = k.transpose(1, 2).contiguous().to(dev).transpose(1, 2)
    kv4_write(kd, wide[:, :, 3:-3], got[:, 1])
    assert torch.equal(got.cpu(), want)
    ko = torch.zeros(B, S, H, d, dtype=BF16, device=dev).transpose(1, 2)
    wide.zero_()
    kv4_read(got[:, 1], ko, wide[:, :, 3:-3])
    n, s, c = O.unpack(want[:, 1], d, group)
    held = O.values(n, s, c, group)[:, :, :, :S].to(torch.float32).to(BF16)
    assert torch.equal(ko.cpu(), held[0]) and torch.equal(wide[:, :, 3:-3].cpu(), held[1])
    assert (wide[:, :, :3] == 0).all() and (wide[:, :, -3:] == 0).all()


def test_values_at_the_ends(dev):
    """Groups of one value, zeros, subnormals, NaN and infinities."""
    d, group = 128, 32
    k = rows(7, 1, 1, 32, d)
    k[0, 0, 0] = 0
    k[0, 0, 1] = -3.0
    k[0, 0, 2] = 2.0 ** -133
    k[0, 0, 3] = torch.linspace(-1, 1, d).to(BF16) * 2.0 ** -127
    k[0, 0, 4, 40] = math.nan
    k[0, 0, 5, 70] = math.inf
    k[0, 0, 6, 100] = -math.inf
    k[0, 0, 7] = torch.linspace(-1, 1, d).to(BF16) * 2.0 ** 120
    v = k.flip(2).contiguous()
    cache = kv4_cache(1, 1, 32, d, dev, group)
    kv4_write(k.to(dev), v.to(dev), cache)
    got = O.unpack(cache, d, group)
    want = O.unpack(O.write(torch.zeros_like(cache, device="cpu"), k, v, [0], [32], group), d, group)
    for a, b in zip(got[1:], want[1:]):
        assert torch.equal(a.isnan(), b.isnan())
        assert torch.equal(a.nan_to_num(5.0), b.nan_to_num(5.0))
    fine = ~want[1].isnan().repeat_interleave(group, -1)
    assert torch.equal(got[0][fine], want[0][fine])
    ko, vo = (torch.empty(1, 1, 32, d, dtype=BF16, device=dev) for _ in range(2))
    kv4_read(cache, ko, vo)
    assert torch.equal(ko.cpu()[0, 0, :3], k[0, 0, :3])
    assert ko[0, 0, 4, 32:64].isnan().all() and not ko[0, 0, 4, :32].isnan().any()
    assert ko[0, 0, 5, 64:96].isnan().all() and ko[0, 0, 6, 96:].isnan().all()


# ---------------------------------------------------------------------------
# The append.
# ---------------------------------------------------------------------------
def step_inputs(seed, B, T, nq, nkv, d, n_rows, dev):
    qkv = (randn(seed, B * T, (nq + 2 * nkv) * d) * 3).to(BF16)
    q_w, k_w = ((1 + 0.2 * randn(seed + i, d)).to(BF16) for i in (1, 2))
    ang = torch.arange(n_rows)[:, None] * 10000.0 ** (-torch.arange(0, d, 2) / d)
    ang = torch.cat((ang, ang), -1)
    return [t.to(dev) for t in (qkv, q_w, k_w, ang.cos().to(BF16), ang.sin().to(BF16))]


def check_appended(cache, old, qkv, k_w, cos, sin, pos, T, eps, nq, nkv, d, group):
    """The appended slots are the format's of the 64-bit k and of v; every other byte stayed."""
    B = cache.shape[0]
    n, s, c = O.unpack(cache, d, group)
    n0, s0, c0 = (t.clone() for t in O.unpack(old, d, group))
    cap = min(n.shape[3], cos.shape[0])
    x = qkv.cpu().view(B, T, nq + 2 * nkv, d)
    for b in range(B):
        for t in range(T):
            p = pos[b] + t
            if not 0 <= p < cap:
                continue
            k = O.norm_rope(x[b, t, nq:nq + nkv], k_w.cpu(), cos[p].cpu(), sin[p].cpu(), eps)
            _, sk, _ = O.quantise(k, group)
            got = O.values(n[0, b, :, p], s[0, b, :, p], c[0, b, :, p], group)
            step = sk.double().repeat_interleave(group, -1)
            # half a step of an s one bf16 step off (2^-7), 8 s 2^-8 at the ends, and fp32's norm
            # and rotation (2^-20 of values below 2^4 s)
            assert ((got - k).abs() <= step * (0.5 + 2.0 ** -7 + 2.0 ** -5 + 2.0 ** -10)).all()
            assert ((s[0, b, :, p] - sk).abs() <= sk * 2.0 ** -7).all()
            nv, sv, cv = O.quantise(x[b, t, nq + nkv:], group)
            assert torch.equal(n[1, b, :, p], nv)
            assert torch.equal(s[1, b, :, p], sv) and torch.equal(c[1, b, :, p], cv)
            for a, a0 in ((n, n0), (s, s0), (c, c0)):
                a0[:, b, :, p] = a[:, b, :, p]
    assert torch.equal(O.pack(n0, s0, c0), cache.cpu())


@pytest.mark.parametrize("d,group", FORMATS)
@pytest.mark.parametrize("B,T,nq,nkv", [(1, 1, 4, 1), (3, 7, 6, 2), (2, 8, 3, 3)])
def test_append(dev, d, group, B, T, nq, nkv):
    nb, eps, n_rows = 3, 1e-6, 90     # the RoPE tables end inside the cache
    pos = [0, 29, 85][:B] if B > 1 else [63]
    old = junk((B, nkv, nb, kv4_block_bytes(d, group)), 8)
    qkv, q_w, k_w, cos, sin = step_inputs(9, B, T, nq, nkv, d, n_rows, dev)
    cache, q = old.to(dev), torch.full((B * T, nq * d), 7.0, dtype=BF16, device=dev)
    kv4_append(qkv, q_w, k_w, cos, sin, torch.tensor(pos, dtype=torch.int32, device=dev), q, cache,
               T, eps, nq, nkv, d)
    check_appended(cache, old, qkv, k_w, cos, sin, pos, T, eps, nq, nkv, d, group)
    x, got = qkv.cpu().view(B, T, -1, d)[:, :, :nq], q.cpu().view(B, T, nq, d)
    for b in range(B):
        for t in range(T):
            if pos[b] + t >= n_rows:
                assert (got[b, t] == 7.0).all()
                continue
            want = O.norm_rope(x[b, t], q_w.cpu(), cos[pos[b] + t].cpu(), sin[pos[b] + t].cpu(), eps)
            # one rounding to bf16, over fp32 sums of terms below 8
            assert ((got[b, t].double() - want).abs() <= want.abs() * 2.0 ** -8 + 2.0 ** -18).all()


# ---------------------------------------------------------------------------
# Attention.
# ---------------------------------------------------------------------------
def check_attention(got, q, cache, lens, T, nq, d, group):
    want, step, size = O.attention(q, cache, lens, T, nq, d, group)
    # out's rounding to bf16 (2^-8 of it); p s rounded to bf16 for the matrix product (2^-8 of
    # the terms p |s (n - 8)|); fp32 scores below 2^6 through exp2 (2^-13 of the terms p |x|)
    tol = want.abs() * 2.0 ** -8 + step * 2.0 ** -8 + size * 2.0 ** -13 + 1e-30
    err = (got.cpu().double() - want).abs()
    assert not got.isnan().any()
    assert (err <= tol).all(), f"worst {(err / tol).max():.3f} of the bound"


def attend(dev, B, T, nq, nkv, d, group, cap, lens, seed=11):
    cache = filled(B, nkv, cap, d, group, lens, seed).to(dev)
    q = randn(seed + 5, B * T, nq * d).to(BF16).to(dev)
    out = torch.full_like(q, math.nan)
    plan = Kv4Attention(B, T, cap, nq, nkv, d, dev, group=group)
    ln = torch.tensor(lens, dtype=torch.int32, device=dev)
    plan.with_lengths(q, cache, ln, out)
    check_attention(out, q, cache, lens, T, nq, d, group)
    if min(lens) >= T:   # the same call by position
        again = torch.full_like(q, math.nan)
        plan(q, cache, ln - T, again)
        assert torch.equal(again, out)


@pytest.mark.parametrize("d,group", FORMATS)
@pytest.mark.parametrize("n", [0, 1, 2, 7, 31, 32, 33, 64, 100, 257, 1000])
def test_one_sequence(dev, d, group, n):
    attend(dev, 1, 1, 8, 2, d, group, max(n, 1), [n])


@pytest.mark.parametrize("G", [1, 2, 3, 4, 5, 8, 16, 33, 64])
@pytest.mark.parametrize("d,group", [(128, 32), (128, 128), (64, 32)])
def test_head_layouts(dev, G, d, group):
    attend(dev, 2, 1, 3 * G, 3, d, group, 200, [200, 77])


@pytest.mark.parametrize("d,group", FORMATS)
@pytest.mark.parametrize("T", [2, 3, 4, 5, 7, 8])
def test_query_tokens(dev, d, group, T):
    attend(dev, 4, T, 8, 2, d, group, 150, [T, 150, 33, 1])   # a block of rows that see nothing


@pytest.mark.parametrize("T,G", [(8, 8), (3, 8), (5, 5), (8, 1), (4, 16), (2, 32)])
def test_tokens_and_heads(dev, T, G):
    attend(dev, 2, T, 2 * G, 2, 128, 32, 70, [70, 40])
    attend(dev, 2, T, 2 * G, 2, 64, 64, 70, [0, 69])


@pytest.mark.parametrize("B", [2, 63, 64, 65, 130])
def test_ragged_batches(dev, B):
    lens = [(37 * i * i + 11 * i) % 300 for i in range(B)]
    attend(dev, B, 1, 4, 1, 128, 64, 300, lens)


def test_long_sequences(dev):
    attend(dev, 1, 1, 4, 1, 128, 32, 20000, [19987])
    attend(dev, 3, 1, 8, 2, 64, 64, 9000, [9000, 1, 4321])


def test_lengths_past_the_cache_are_cut(dev):
    cache = filled(1, 1, 64, 128, 32, [64], 3).to(dev)
    q = randn(4, 1, 4 * 128).to(BF16).to(dev)
    plan = Kv4Attention(1, 1, 64, 4, 1, 128, dev)
    outs = []
    for n in (64, 1000, 2 ** 31 - 1, -3, -2 ** 31):
        out = torch.empty_like(q)
        plan.with_lengths(q, cache, torch.tensor([n], dtype=torch.int32, device=dev), out)
        outs.append(out)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
    assert (outs[3] == 0).all() and (outs[4] == 0).all()
    out = torch.empty_like(q)   # a position whose sum with T passes 32 bits
    plan(q, cache, torch.tensor([2 ** 31 - 1], dtype=torch.int32, device=dev), out)
    assert torch.equal(out, outs[0])


def test_a_cache_of_other_strides_and_shared_sequences(dev):
    B, H, d, group, cap = 3, 2, 128, 32, 100
    one = filled(1, H, cap, d, group, [cap], 5).to(dev)
    q = randn(6, B, 8 * d).to(BF16).to(dev)
    lens = torch.tensor([100, 50, 3], dtype=torch.int32, device=dev)
    plan = Kv4Attention(B, 1, cap, 8, H, d, dev, group=group)
    want, got = torch.empty_like(q), torch.empty_like(q)
    plan.with_lengths(q, one.expand(B, -1, -1, -1).contiguous(), lens, want)
    plan.with_lengths(q, one.expand(B, -1, -1, -1), lens, got)       # one prefix, three sequences
    assert torch.equal(want, got)
    turned = one.expand(B, -1, -1, -1).transpose(0, 1).contiguous().transpose(0, 1)
    plan.with_lengths(q, turned, lens, got)
    assert torch.equal(want, got)


def test_a_cached_nan_reaches_the_rows_that_see_it(dev):
    cache = filled(2, 1, 40, 128, 32, [40, 40], 7)
    n, s, c = O.unpack(cache, 128, 32)
    s[0, 0, 0, 39, 2] = math.nan       # a key
    c[1, 1, 0, 38, 1] = math.nan       # a value
    cache = O.pack(n, s, c).to(dev)
    q = randn(8, 2 * 2, 4 * 128).to(BF16).to(dev)
    out = torch.empty_like(q)
    Kv4Attention(2, 2, 40, 4, 1, 128, dev)(q, cache, torch.tensor([38, 38], dtype=torch.int32,
                                                                  device=dev), out)
    assert not out[0].isnan().any() and out[1].isnan().all()
    bad = out[2:].view(2, 4, 128)
    assert bad[..., 32:64].isnan().all()
    assert not bad[..., :32].isnan().any() and not bad[..., 64:].isnan().any()


# ---------------------------------------------------------------------------
# A run of them, as a step uses them.
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("d,group", FORMATS)
@pytest.mark.parametrize("B,T", [(1, 1), (5, 1), (3, 4)])
def test_prompt_then_steps(dev, d, group, B, T):
    nq, nkv, cap, eps, S = 8, 2, 96, 1e-6, 30
    lens = [30, 1, 17, 0, 29][:B]
    cache = junk((B, nkv, cap // 32, kv4_block_bytes(d, group)), 20).to(dev)
    k, v = rows(21, B, nkv, S, d).to(dev), rows(22, B, nkv, S, d).to(dev)
    pos = torch.tensor(lens, dtype=torch.int32, device=dev)
    kv4_write(k, v, cache, lengths=pos)
    plan = Kv4Attention(B, T, cap, nq, nkv, d, dev, group=group)
    for step in range(6):
        qkv, q_w, k_w, cos, sin = step_inputs(30 + step, B, T, nq, nkv, d, cap, dev)
        old = cache.cpu()
        q = torch.empty(B * T, nq * d, dtype=BF16, device=dev)
        out = torch.empty_like(q)
        args = (qkv, q_w, k_w, cos, sin, pos)
        other = cache.clone()
        kv4_append(*args, q, other, T, eps, nq, nkv, d)
        if T == 1:
            plan.decode_qkv(*args, cache, out, eps)
        else:
            cache.copy_(other)
            plan(q, cache, pos, out)
        at = [n + T * step for n in lens]
        check_appended(cache, old, qkv, k_w, cos, sin, at, T, eps, nq, nkv, d, group)
        total = [n + T for n in at]
        want, mid, size = O.attention(q, cache, total, T, nq, d, group)
        # check_attention's bound, and for decode_qkv a q that may lie a bf16 step from kv4_append's
        tol = want.abs() * 2.0 ** -8 + mid * 2.0 ** -8 + size * 2.0 ** -13
        err = (out.cpu().double() - want).abs()
        assert (err <= tol + (size * 2.0 ** -7 if T == 1 else 0)).all()
        pos += T


@pytest.mark.parametrize("d,group", FORMATS)
@pytest.mark.parametrize("nq,nkv", [(3, 3), (8, 1), (40, 2)])
def test_decode_qkv_head_layouts_and_positions(dev, d, group, nq, nkv):
    """1, 8 and 20 query heads a KV head; positions at a block's and the cache's ends, and outside
    the cache and the tables; the RoPE rows from the tables and as rows."""
    pos = [0, 31, 32, 63, 95, 96, -1, 2 ** 31 - 1, 70, 64]
    B, cap, n_rows, eps = len(pos), 96, 70, 1e-6
    plan = Kv4Attention(B, 1, cap, nq, nkv, d, dev, group=group)
    lens = [min(max(p, 0), cap) for p in pos]
    old = filled(B, nkv, cap, d, group, lens, 70)
    qkv, q_w, k_w, cos, sin = step_inputs(71, B, 1, nq, nkv, d, n_rows, dev)
    at = torch.tensor(pos, dtype=torch.int32, device=dev)
    cache, out = old.to(dev), torch.full((B, nq * d), math.nan, dtype=BF16, device=dev)
    plan.decode_qkv(qkv, q_w, k_w, cos, sin, at, cache, out, eps)
    check_appended(cache, old, qkv, k_w, cos, sin, pos, 1, eps, nq, nkv, d, group)
    fine = [0 <= p < n_rows for p in pos]
    x = qkv.cpu().view(B, -1, d)[:, :nq]
    for b, ok in enumerate(fine):
        if not ok:
            assert (out[b] == 0).all()
            continue
        q = O.norm_rope(x[b], q_w.cpu(), cos[pos[b]].cpu(), sin[pos[b]].cpu(), eps)
        want, mid, size = O.attention(q.to(BF16).view(1, -1), cache[b:b + 1], [pos[b] + 1], 1, nq, d,
                                      group)
        # check_attention's bound; a few of q's values may lie a bf16 step off
        tol = want.abs() * 2.0 ** -8 + mid * 2.0 ** -8 + size * (2.0 ** -13 + 2.0 ** -7)
        assert ((out[b].cpu().double() - want).abs() <= tol).all()
    rope = torch.zeros(B, 2, d, dtype=BF16, device=dev)
    rope_rows(at, cos, sin, rope)
    cache2, out2 = old.to(dev), torch.empty_like(out)
    plan.decode_qkv(qkv, q_w, k_w, cos, sin, at, cache2, out2, eps, rope=rope)
    assert torch.equal(out2, out) and torch.equal(cache2, cache)


def test_captured_steps_replay(dev):
    """decode_qkv in a graph: three steps a replay, eager work between the replays, every
    replay against the same steps made eagerly."""
    B, nq, nkv, d, group, cap, eps = 2, 8, 2, 128, 32, 128, 1e-6
    plan, other = (Kv4Attention(B, 1, cap, nq, nkv, d, dev, group=group) for _ in range(2))
    qkv, q_w, k_w, cos, sin = step_inputs(40, B, 1, nq, nkv, d, cap, dev)
    start = torch.tensor([5, 40], dtype=torch.int32, device=dev)
    pos, out, cache = start.clone(), torch.empty(3, B, nq * d, dtype=BF16, device=dev), None
    cache = filled(B, nkv, cap, d, group, [5, 40], 41).to(dev)
    first = cache.clone()

    def steps(plan, cache, pos, out):
        for i in range(3):
            plan.decode_qkv(qkv, q_w, k_w, cos, sin, pos, cache, out[i], eps)
            pos.add_(1)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        steps(plan, cache, pos, out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    cache.copy_(first)
    pos.copy_(start)
    with torch.cuda.graph(graph):
        steps(plan, cache, pos, out)
    cache.copy_(first)
    pos.copy_(start)
    e_cache, e_pos, e_out = first.clone(), start.clone(), torch.empty_like(out)
    for rep in range(4):
        qkv.copy_(step_inputs(50 + rep, B, 1, nq, nkv, d, cap, dev)[0])
        steps(other, e_cache, e_pos, e_out)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, e_out) and torch.equal(cache, e_cache) and torch.equal(pos, e_pos)


def test_runs_repeat_bit_for_bit(dev):
    lens = [3000, 17, 801]
    cache = filled(3, 2, 3000, 128, 32, lens, 60).to(dev)
    q = randn(61, 3, 8 * 128).to(BF16).to(dev)
    plan = Kv4Attention(3, 1, 3000, 8, 2, 128, dev)
    ln = torch.tensor(lens, dtype=torch.int32, device=dev)
    outs = [torch.empty_like(q) for _ in range(20)]
    for o in outs:
        plan.with_lengths(q, cache, ln, o)
    assert all(torch.equal(o, outs[0]) for o in outs)


@pytest.mark.parametrize("d,group", FORMATS)
def test_a_workgroup_of_8_wavefronts_a_pair(dev, d, group):
    """129 to 256 pairs, and blocks of 16 query rows: lengths that keep to one part, that are cut,
    and that share a run."""
    attend(dev, 40, 1, 16, 4, d, group, 200, [200] * 40)
    attend(dev, 43, 1, 15, 5, d, group, 700, [(97 * i) % 700 for i in range(43)])
    attend(dev, 3, 5, 8, 2, d, group, 2100, [2100, 1, 300])


def test_decode_qkv_of_many_pairs(dev):
    B, nq, nkv, d, group, cap, eps = 40, 16, 4, 128, 32, 128, 1e-6
    pos = [(5 * i) % cap for i in range(B)]
    old = filled(B, nkv, cap, d, group, pos, 80)
    qkv, q_w, k_w, cos, sin = step_inputs(81, B, 1, nq, nkv, d, cap, dev)
    at = torch.tensor(pos, dtype=torch.int32, device=dev)
    cache, out = old.to(dev), torch.empty(B, nq * d, dtype=BF16, device=dev)
    plan = Kv4Attention(B, 1, cap, nq, nkv, d, dev, group=group)
    plan.decode_qkv(qkv, q_w, k_w, cos, sin, at, cache, out, eps)
    check_appended(cache, old, qkv, k_w, cos, sin, pos, 1, eps, nq, nkv, d, group)
    q = torch.empty_like(out)
    kv4_append(qkv, q_w, k_w, cos, sin, at, q, old.to(dev), 1, eps, nq, nkv, d)
    want, mid, size = O.attention(q, cache, [p + 1 for p in pos], 1, nq, d, group)
    tol = want.abs() * 2.0 ** -8 + mid * 2.0 ** -8 + size * (2.0 ** -13 + 2.0 ** -7)
    assert ((out.cpu().double() - want).abs() <= tol).all()


@pytest.mark.parametrize("nq,nkv,d,group", [(4, 1, 128, 32), (16, 2, 64, 64)])
@pytest.mark.parametrize("T", [2, 7])
def test_tokens_behind_the_cache_do_not_move_the_others(dev, nq, nkv, d, group, T):
    """Queries at pos .. pos + T - 1 of which the last lie behind the cache: each sees the keys up to
    its own position that there are."""
    cap = 64
    pos = [60, 63, 64, 100, 2 ** 31 - 1, cap - T]
    cache = filled(len(pos), nkv, cap, d, group, [cap] * len(pos), 90).to(dev)
    q = randn(91, len(pos) * T, nq * d).to(BF16).to(dev)
    out = torch.full_like(q, math.nan)
    Kv4Attention(len(pos), T, cap, nq, nkv, d, dev, group=group)(
        q, cache, torch.tensor(pos, dtype=torch.int32, device=dev), out)
    for b, p in enumerate(pos):
        for t in range(T):
            row = slice(b * T + t, b * T + t + 1)
            check_attention(out[row], q[row], cache[b:b + 1], [min(p + t + 1, cap)], 1, nq, d, group)


def test_a_capacity_is_whole_blocks(dev):
    """kv4_cache, kv4_append and the attention agree on the slots of a cap between two blocks."""
    nq, nkv, d, cap, eps, pos = 4, 1, 128, 33, 1e-6, [40, 63, 64]
    B = len(pos)
    cache = kv4_cache(B, nkv, cap, d, dev)
    assert cache.shape[2] == 2
    cache.copy_(filled(B, nkv, 64, d, 32, [40, 63, 64], 92))
    qkv, q_w, k_w, cos, sin = step_inputs(93, B, 1, nq, nkv, d, 100, dev)
    at = torch.tensor(pos, dtype=torch.int32, device=dev)
    out = torch.full((B, nq * d), math.nan, dtype=BF16, device=dev)
    plan = Kv4Attention(B, 1, cap, nq, nkv, d, dev)
    plan.decode_qkv(qkv, q_w, k_w, cos, sin, at, cache, out, eps)
    assert (out[2] == 0).all()
    want = torch.empty_like(out)
    Kv4Attention(B, 1, 64, nq, nkv, d, dev).with_lengths(plan._q, cache, at + 1, want)
    assert torch.equal(out[:2], want[:2])


@pytest.mark.parametrize("grid,min_run", [(1, 1), (2, 8), (5, 3), (64, 1), (512, 40)])
@pytest.mark.parametrize("T,nq,nkv,d,group", [(1, 8, 2, 128, 32), (5, 8, 2, 64, 64)])
def test_any_number_of_workgroups(dev, grid, min_run, T, nq, nkv, d, group):
    """Few workgroups, whose runs cross from pair to pair, and short or long runs."""
    lens = [700, 3, 0, 1500, 33, 64, 901]
    B, cap = len(lens), 1500
    cache = filled(B, nkv, cap, d, group, lens, 94).to(dev)
    q = randn(95, B * T, nq * d).to(BF16).to(dev)
    plan = Kv4Attention(B, T, cap, nq, nkv, d, dev, group=group)
    plan.grid, plan.MIN_RUN = grid, min_run
    for _ in range(2):   # the second finds the counters as the first left them
        out = torch.full_like(q, math.nan)
        plan.with_lengths(q, cache, torch.tensor(lens, dtype=torch.int32, device=dev), out)
        check_attention(out, q, cache, lens, T, nq, d, group)
    assert not plan._counters.any()


@pytest.mark.parametrize("T,d,group", [(17, 128, 32), (33, 128, 128), (64, 64, 32), (64, 128, 64)])
def test_more_query_tokens_than_the_op_offers(dev, monkeypatch, T, d, group):
    """The C entry serves T * nq / nkv up to 64, whatever T: the last tokens' limits then lie in three
    blocks."""
    monkeypatch.setattr(Kv4Attention, "MAX_T", 64)
    attend(dev, 3, T, 2, 2, d, group, 400, [385, T, 70])
    attend(dev, 1, T, 1, 1, d, group, 1500, [1473])


def test_offsets_past_32_bits(dev):
    """Sequences 5 GiB apart in the cache, and 6 GiB in the rows that are written and read."""
    d, group, nb, S, eps = 128, 32, 3, 70, 1e-6
    far, row = 5 << 30, 3 << 30
    size = kv4_block_bytes(d, group)
    hold = torch.empty(far + nb * size, dtype=torch.uint8, device=dev)
    cache = hold.as_strided((2, 1, nb, size), (far, nb * size, size, 1))
    rows_k = torch.empty(row + S * d, dtype=BF16, device=dev).as_strided((2, 1, S, d), (row, S * d, d, 1))
    k, v = rows(100, 2, 1, S, d).to(dev), rows(101, 2, 1, S, d).to(dev)
    near = kv4_cache(2, 1, nb * KV4_KEYS, d, dev, group)
    cache.copy_(near)
    rows_k.copy_(k)
    kv4_write(k, v, near)
    kv4_write(rows_k, v, cache)
    assert torch.equal(cache, near)
    rows_k.zero_()
    k1, v1, v2 = (torch.zeros_like(k) for _ in range(3))
    kv4_read(near, k1, v1)
    kv4_read(cache, rows_k, v2)
    assert torch.equal(rows_k, k1) and torch.equal(v2, v1)
    pos = torch.tensor([S, S - 3], dtype=torch.int32, device=dev)
    qkv, q_w, k_w, cos, sin = step_inputs(102, 2, 1, 4, 1, d, 96, dev)
    plan = Kv4Attention(2, 1, nb * KV4_KEYS, 4, 1, d, dev, group=group)
    out = torch.empty(2, 2, 4 * d, dtype=BF16, device=dev)
    plan.decode_qkv(qkv, q_w, k_w, cos, sin, pos, near, out[0], eps)
    plan.decode_qkv(qkv, q_w, k_w, cos, sin, pos, cache, out[1], eps)
    assert torch.equal(cache, near) and torch.equal(out[0], out[1])


def test_two_objects_on_two_streams(dev):
    """Calls of two objects at once, each with its own workspace, against the same calls in turn."""
    lens = [[2500, 31, 900], [1200, 2000, 5]]
    caches = [filled(3, 2, 2500, 128, 32, n, 110 + i).to(dev) for i, n in enumerate(lens)]
    q = [randn(112 + i, 3, 8 * 128).to(BF16).to(dev) for i in range(2)]
    ln = [torch.tensor(n, dtype=torch.int32, device=dev) for n in lens]
    plans = [Kv4Attention(3, 1, 2500, 8, 2, 128, dev) for _ in range(2)]
    want = [torch.empty_like(x) for x in q]
    for i in range(2):
        plans[i].with_lengths(q[i], caches[i], ln[i], want[i])
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[torch.empty_like(x) for _ in range(20)] for x in q]
    torch.cuda.synchronize()
    for j in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                plans[i].with_lengths(q[i], caches[i], ln[i], outs[i][j])
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in outs[i])


def test_refusals(dev):
    """What each op names, of tensors on the GPU."""
    B, nq, nkv, d, S = 2, 4, 2, 128, 5
    cache = kv4_cache(B, nkv, 64, d, dev)
    k = torch.zeros(B, nkv, S, d, dtype=BF16, device=dev)
    ints = torch.zeros(B, dtype=torch.int32, device=dev)
    for args, kw in (((k.float(), k, cache), {}), ((k, k[:, :1], cache), {}),
                     ((k[..., ::2], k, cache), {}), ((k, k, cache[0]), {}), ((k, k, cache[..., 1:]), {}),
                     ((k, k, cache.float()), {}), ((k, k, cache), dict(start=ints.long())),
                     ((k, k, cache), dict(lengths=ints[:1])), ((k, k.cpu(), cache), {}),
                     ((k, k, cache), dict(lengths=ints.cpu())), ((k, None, cache), {}),
                     ((k, k, cache[:1].expand(B, -1, -1, -1)), {}),
                     ((k.flatten()[1:-7].view(-1), k, cache), {})):
        with pytest.raises(ValueError):
            kv4_write(*args, **kw)
    for a, b in ((k, k), (k, k[:1].expand(B, -1, -1, -1)), (k, k.float())):
        with pytest.raises(ValueError):
            kv4_read(cache, a, b)
    qkv, w = torch.zeros(B, (nq + 2 * nkv) * d, dtype=BF16, device=dev), torch.zeros(d, dtype=BF16, device=dev)
    tab, q = torch.zeros(64, d, dtype=BF16, device=dev), torch.zeros(B, nq * d, dtype=BF16, device=dev)
    plan, out = Kv4Attention(B, 1, 64, nq, nkv, d, dev), torch.zeros_like(q)
    good = [qkv, w, w, tab, tab, ints]
    for i, bad in ((0, qkv[:1]), (0, qkv.float()), (1, w[:64]), (2, w.cpu()), (3, tab[:0]), (4, tab[0]),
                   (3, tab.t()), (5, ints.long()), (5, None)):
        args = good[:i] + [bad] + good[i + 1:]
        with pytest.raises(ValueError):
            kv4_append(*args, q, cache, 1, 1e-6, nq, nkv, d)
        with pytest.raises(ValueError):
            plan.decode_qkv(*args, cache, out, 1e-6)
    for bad in (dict(T=0), dict(T=2), dict(nkv=1), dict(d=64), dict(q=q[:1]), dict(q=None),
                dict(cache=cache.cpu()), dict(cache=cache[:1].expand(B, -1, -1, -1))):
        a = dict(q=q, cache=cache, T=1, nkv=nkv, d=d) | bad
        with pytest.raises(ValueError):
            kv4_append(*good, a["q"], a["cache"], a["T"], 1e-6, nq, a["nkv"], a["d"])
    for a in ((q, cache, ints, q), (q[:1], cache, ints, out), (q, cache[:1], ints, out),
              (q, cache, ints.long(), out), (q, cache, ints, out.float()), (None, cache, ints, out),
              (q, cache.cpu(), ints, out), (q, cache, ints, None)):
        with pytest.raises(ValueError):
            plan(*a)
    with pytest.raises(ValueError):
        Kv4Attention(B, 2, 64, nq, nkv, d, dev).decode_qkv(*good, cache, out, 1e-6)
    with pytest.raises(ValueError):
        plan.decode_qkv(*good, cache[:1].expand(B, -1, -1, -1), out, 1e-6)
    with pytest.raises(ValueError):
        plan.decode_qkv(*good, cache, out, 1e-6, rope=tab)
    torch.cuda.synchronize()
    assert not cache.any() and not out.any() and not q.any()


@pytest.mark.parametrize("d,group", FORMATS)
def test_the_top_of_the_range(dev, d, group):
    """Finite groups whose ends lie further apart than fp32's largest number, or next to bf16's: held
    as any other group is, by both writers, and read back finite."""
    g = top_groups()
    per, reps = d // group, group // 32
    S = -(-len(g) // per)
    x = torch.cat((g, g[:S * per - len(g)])).repeat_interleave(reps, 1)
    x = x.reshape(1, 1, S, d)
    k, v = torch.cat((x, x.flip(2)), 1), torch.cat((-x, x), 1)
    nb = -(-S // KV4_KEYS)
    old = junk((1, 2, nb, kv4_block_bytes(d, group)), 120)
    want = O.write(old, k, v, [0], [S], group)
    cache = old.to(dev)
    kv4_write(k.to(dev), v.to(dev), cache)
    assert torch.equal(cache.cpu(), want)
    ko, vo = (torch.empty(1, 2, S, d, dtype=BF16, device=dev) for _ in range(2))
    kv4_read(cache, ko, vo)
    held = O.read_back(*O.unpack(want, d, group), group)[:, :, :, :S]
    assert held.isfinite().all()
    assert torch.equal(ko.cpu(), held[0]) and torch.equal(vo.cpu(), held[1])
    # the append: the same rows as V of one sequence's tokens
    qkv = torch.zeros(S, 1 + 2 * 2, d, dtype=BF16)
    qkv[:, 3:] = v[0].transpose(0, 1)
    w, tab = torch.ones(d, dtype=BF16, device=dev), torch.ones(S, d, dtype=BF16, device=dev)
    q, cache = torch.empty(S, d, dtype=BF16, device=dev), old.to(dev)
    kv4_append(qkv.flatten(1).to(dev), w, w, tab, tab, torch.zeros(1, dtype=torch.int32, device=dev),
               q, cache, S, 1e-6, 1, 2, d)
    for got, ref in zip(O.unpack(cache, d, group), O.unpack(want, d, group)):
        assert torch.equal(got[1, :, :, :S], ref[1, :, :, :S])


def test_every_scale_and_the_borders_of_its_codes(dev):
    """Groups whose scale takes every normal bf16 below 2^125 (from there on only the widest
    spans, test_the_top_of_the_range), with the values on both sides of each border between two
    codes: a reciprocal of s that is off by its last bit moves codes of 3,800 of them."""
    s = (torch.arange(0x0080, 0x7e00, dtype=torch.int32) << 16).view(torch.float32).double()
    lo, hi = -8 * s, (7 * s).to(BF16).double()
    border = (torch.arange(15, dtype=torch.float64) - 7.5) * s[:, None]
    near = border.to(BF16)
    # the neighbour on the border's other side, where the border is no bf16 itself: one bit pattern
    # further from zero or nearer to it
    bits = near.view(torch.int16)
    further = near.double().abs() < border.abs()
    other = (bits + torch.where(further, 1, -1).to(torch.int16)).view(BF16)
    x = torch.cat((lo[:, None], hi[:, None], near.double(), other.double()), 1)
    x = torch.minimum(torch.maximum(x, lo[:, None]), hi[:, None]).to(BF16)
    d, group = 128, 32
    S = len(s) // 4
    k = x.reshape(1, 1, S, d)
    v = k.flip(2).contiguous()
    cache = kv4_cache(1, 1, S, d, dev, group)
    kv4_write(k.to(dev), v.to(dev), cache)
    n, sc, c = O.unpack(cache, d, group)
    for i, rows_ in enumerate((k, v)):
        want = O.quantise(rows_, group)
        for got, w in zip((n[i], sc[i], c[i]), want):
            assert torch.equal(got[:, :, :S], w)
    assert torch.equal(sc[0, 0, 0, :S].flatten().double(), s)   # every scale occurs


def exact_step(dev, B, nq, nkv, d, group, cap, pos, seed):
    """decode_qkv against kv4_append and with_lengths, bit for bit, and the result within the
    attention's own bound of the 64-bit one over the same q."""
    old = filled(B, nkv, cap, d, group, pos, seed)
    qkv, q_w, k_w, cos, sin = step_inputs(seed + 1, B, 1, nq, nkv, d, cap, dev)
    at = torch.tensor(pos, dtype=torch.int32, device=dev)
    cache, out = old.to(dev), torch.full((B, nq * d), math.nan, dtype=BF16, device=dev)
    plan = Kv4Attention(B, 1, cap, nq, nkv, d, dev, group=group)
    plan.decode_qkv(qkv, q_w, k_w, cos, sin, at, cache, out, 1e-6)
    apart, q, again = old.to(dev), torch.empty_like(out), torch.full_like(out, math.nan)
    kv4_append(qkv, q_w, k_w, cos, sin, at, q, apart, 1, 1e-6, nq, nkv, d)
    plan.with_lengths(q, apart, at + 1, again)
    assert torch.equal(cache, apart) and torch.equal(out, again)
    check_attention(out, q, cache, [p + 1 for p in pos], 1, nq, d, group)


@pytest.mark.parametrize("d,group", FORMATS)
def test_a_decode_step_is_its_two_ops(dev, d, group):
    exact_step(dev, 1, 8, 2, d, group, 96, [64], 130)
    exact_step(dev, 5, 8, 2, d, group, 96, [30, 1, 17, 0, 95], 132)
    exact_step(dev, 40, 16, 4, d, group, 128, [(5 * i) % 128 for i in range(40)], 134)
    exact_step(dev, 2, 8, 1, d, group, 3000, [2900, 77], 136)


@pytest.mark.parametrize("T,nq,nkv,d,group", [
    (1, 8, 1, 128, 32),    # 8 held rows: 2 a wavefront in the merge
    (1, 4, 1, 64, 64),     # one group a head: 16 held rows, 4 a wavefront
    (5, 4, 1, 128, 32),    # 20 query rows in two blocks of 16, 8 wavefronts
    (8, 8, 1, 128, 32),    # 64 in four
    (8, 4, 1, 64, 32)])
def test_more_than_64_parts_of_a_pair(dev, T, nq, nkv, d, group):
    """The merge takes 64 parts at a time and rescales what it has; 79 parts here."""
    attend(dev, 1, T, nq, nkv, d, group, 20000, [19987])


def scaled(cache, d, group, by_k, by_v):
    """The cache with its K and V values times powers of two."""
    n, s, c = O.unpack(cache, d, group)
    by = torch.tensor([by_k, by_v]).view(2, 1, 1, 1, 1)
    return O.pack(n, s * by, c * by)


@pytest.mark.parametrize("T,nq,nkv,d,group", [(1, 8, 2, 128, 32), (1, 8, 1, 64, 64), (5, 8, 2, 128, 64),
                                              (1, 4, 4, 128, 128)])
@pytest.mark.parametrize("power", [4, 10, 15, 20, 38])
def test_large_scores(dev, T, nq, nkv, d, group, power):
    """q and K of 2^power: the scores' differences decide, whatever the scores are. One wavefront's
    steps, several wavefronts and several parts."""
    for lens in ([40, 7], [300, 257], [2900, 1031]):
        B, cap = 2, max(lens)
        cache = scaled(filled(B, nkv, cap, d, group, lens, 140 + power), d, group, 2.0 ** power, 1.0)
        cache = cache.to(dev)
        q = (randn(141, B * T, nq * d) * 2.0 ** power).to(BF16)
        # fp32 scores are off by up to 2^-14 of sum |q k| (codes as 128 + n: 136 / 8 of 2^-23 a term
        # and the sum's roundings); far below the distance of a row's two largest
        n, s, c = O.unpack(cache, d, group)
        clear = torch.zeros(B, T, nq, dtype=torch.bool)
        for b in range(B):
            for t in range(T):
                m = lens[b] - T + t + 1
                k = O.values(n[0, b, :, :m], s[0, b, :, :m], c[0, b, :, :m], group)
                x = q.double().view(B, T, nkv, -1, d)[b, t] @ k.transpose(1, 2).contiguous()
                size = q.double().view(B, T, nkv, -1, d)[b, t].abs() @ k.abs().transpose(1, 2).contiguous()
                top = x.topk(2, -1).values
                clear[b, t] = (top[..., 0] - top[..., 1] > 2.0 ** -12 * size.amax(-1)).flatten()
        q, ln = q.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev)
        out = torch.full_like(q, math.nan)
        Kv4Attention(B, T, cap, nq, nkv, d, dev, group=group).with_lengths(q, cache, ln, out)
        want, step, size = O.attention(q, cache, lens, T, nq, d, group)
        assert not out.isnan().any()
        if power >= 10:   # one key takes all of a row's weight
            tol = want.abs() * 2.0 ** -8 + step * 2.0 ** -8 + size * 2.0 ** -13 + 1e-30
            fine = (out.cpu().double() - want).abs() <= tol
            assert clear.float().mean() > 0.9
            assert fine.view(B, T, nq, d)[clear].all()


@pytest.mark.parametrize("T,nq,nkv,d,group", [(1, 8, 2, 128, 32), (5, 8, 2, 64, 64)])
def test_large_values(dev, T, nq, nkv, d, group):
    """V of the largest magnitude that the attention's sums are promised for: 2^115 over the keys."""
    lens = [1000, 333]
    cache = filled(2, nkv, 1000, d, group, lens, 150)
    n, s, c = O.unpack(cache, d, group)
    top = O.values(n[1], s[1], c[1], group).nan_to_num(0).abs().max().item()
    by = 2.0 ** math.floor(math.log2(2.0 ** 115 / 1000 / top))
    cache = scaled(cache, d, group, 1.0, by).to(dev)
    q = randn(151, 2 * T, nq * d).to(BF16).to(dev)
    out = torch.full_like(q, math.nan)
    Kv4Attention(2, T, 1000, nq, nkv, d, dev, group=group).with_lengths(
        q, cache, torch.tensor(lens, dtype=torch.int32, device=dev), out)
    check_attention(out, q, cache, lens, T, nq, d, group)


def test_outputs_that_overlap_are_refused(dev):
    """Two outputs of a read, or an output and the rows that other workgroups still read, in one piece
    of memory: by any distance, in any layout. Neighbours in one buffer are served."""
    B, nq, nkv, d, S = 2, 4, 2, 128, 8
    cache = filled(B, nkv, 64, d, 32, [64, 64], 160).to(dev)
    hold = torch.zeros(1 << 16, dtype=BF16, device=dev)
    n = B * nkv * S * d

    def at(offset, *strides):
        return hold.as_strided((B, nkv, S, d), strides or (nkv * S * d, S * d, d, 1), offset)

    both = (2 * nkv * S * d, S * d, d, 1)     # [B, 2, nkv, S, d]
    turned = (S * 2 * nkv * d, d, 2 * nkv * d, 1)   # [B, S, 2, nkv, d]
    for a, b in ((at(0), at(8)), (at(n - 8), at(0)), (at(0), at(n - d)),
                 (at(0, *both), at(S * d, *both)), (at(0, *turned), at(d, *turned)),
                 (at(2 * nkv * d, *turned), at(0, *turned)), (at(0, *both), at(0, *turned))):
        for k, v in ((a, b), (b, a)):
            with pytest.raises(ValueError, match="overlap"):
                kv4_read(cache, k, v)
    want = [torch.empty(B, nkv, S, d, dtype=BF16, device=dev) for _ in range(2)]
    kv4_read(cache, *want)
    for a, b in ((at(0), at(n)), (at(n + 64), at(0)), (at(0, *both), at(nkv * S * d, *both)),
                 (at(nkv * d, *turned), at(0, *turned)), (at(0, *turned), at(2 * n))):
        kv4_read(cache, a, b)
        assert torch.equal(a, want[0]) and torch.equal(b, want[1])
    plan = Kv4Attention(B, 1, 64, nq, nkv, d, dev)
    ints = torch.full((B,), 3, dtype=torch.int32, device=dev)
    row = lambda offset, cols: hold[offset:offset + B * cols].view(B, cols)
    for offset in (0, 8, B * nq * d - 8):
        for q, out in ((0, offset), (offset, 0)):
            with pytest.raises(ValueError, match="overlap"):
                plan(row(q, nq * d), cache, ints, row(out, nq * d))
    plan(row(0, nq * d), cache, ints, row(B * nq * d, nq * d))
    w, tab, wide = torch.ones(d, dtype=BF16, device=dev), torch.ones(64, d, dtype=BF16, device=dev), nq + 2 * nkv
    for x, q in ((0, 0), (0, 8), (0, B * wide * d - 8), (B * nq * d - 8, 0)):
        with pytest.raises(ValueError, match="overlap"):
            kv4_append(row(x, wide * d), w, w, tab, tab, ints, row(q, nq * d), cache, 1, 1e-6, nq, nkv, d)
    # one row in place: every head reads and writes its own values
    hold.copy_(randn(161, 1 << 16))
    x, one = hold[:wide * d].view(1, -1), cache[:1].clone()
    q, again = torch.empty(1, nq * d, dtype=BF16, device=dev), cache[:1].clone()
    kv4_append(x, w, w, tab, tab, ints[:1], q, one, 1, 1e-6, nq, nkv, d)
    kv4_append(x, w, w, tab, tab, ints[:1], x[:, :nq * d], again, 1, 1e-6, nq, nkv, d)
    assert torch.equal(x[:, :nq * d], q) and torch.equal(again, one)


def test_captured_prompts_and_verify_steps_replay(dev):
    """kv4_write, kv4_append, the attention and kv4_read in one graph, with other rows, starts,
    lengths and positions in every replay, each against the same calls made eagerly between them."""
    B, T, nq, nkv, d, group, cap, S = 3, 4, 8, 2, 128, 32, 256, 70
    plans = [Kv4Attention(B, T, cap, nq, nkv, d, dev, group=group) for _ in range(2)]
    qkv, q_w, k_w, cos, sin = step_inputs(170, B, T, nq, nkv, d, cap, dev)
    k, v = (torch.empty(B, nkv, S, d, dtype=BF16, device=dev) for _ in range(2))
    start, lengths, pos = (torch.zeros(B, dtype=torch.int32, device=dev) for _ in range(3))
    ints = lambda *x: torch.tensor(x, dtype=torch.int32)

    def state():
        return dict(cache=junk((B, nkv, cap // 32, kv4_block_bytes(d, group)), 171).to(dev),
                    q=torch.zeros(B * T, nq * d, dtype=BF16, device=dev),
                    out=torch.zeros(B * T, nq * d, dtype=BF16, device=dev),
                    back=torch.zeros(2, B, nkv, S + T, d, dtype=BF16, device=dev))

    def calls(plan, st):
        kv4_write(k, v, st["cache"], start=start, lengths=lengths)
        kv4_append(qkv, q_w, k_w, cos, sin, pos, st["q"], st["cache"], T, 1e-6, nq, nkv, d)
        plan(st["q"], st["cache"], pos, st["out"])
        kv4_read(st["cache"], *st["back"], start=start, lengths=lengths)

    def inputs(rep):
        k.copy_(rows(172 + rep, B, nkv, S, d))
        v.copy_(rows(182 + rep, B, nkv, S, d))
        qkv.copy_(step_inputs(192 + rep, B, T, nq, nkv, d, cap, dev)[0])
        n = [(S, 1 + 9 * rep, S - rep), (7, S, 33), (S, S, S)][rep % 3]
        at = [ints(0, 0, 0), ints(5, 31, 32), ints(100, 64, 186)][rep % 3]
        start.copy_(at)
        lengths.copy_(ints(*n))
        pos.copy_(at + ints(*n))

    graphed, eager = state(), state()
    inputs(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        calls(plans[0], graphed)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls(plans[0], graphed)
    graphed["cache"].copy_(eager["cache"])
    for rep in range(6):
        inputs(rep)
        calls(plans[1], eager)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for name in eager:
            same = torch.equal(eager[name].view(torch.uint8), graphed[name].view(torch.uint8))
            assert same, (rep, name)
