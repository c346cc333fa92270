"""A KV cache held in 4 bits: writing it, reading it back, and decode attention over it.

The ops stand beside ``kernels.fused``'s for the bf16 cache and follow their manner: tensors
are the caller's, every call launches on the current stream of the current device, allocates
nothing and never synchronises (so calls can be captured), and a bad argument raises
ValueError before anything is launched (RuntimeError where a call is too large for one launch: 2^26
heads of rows to append, 2^25 blocks to write or read).

- ``kv4_cache`` allocates a cache; ``kv4_write`` quantises bf16 K/V rows into it, ``kv4_read``
  reads cached keys back as bf16;
- ``kv4_append``: ``qk_norm_rope`` (engine/kernels/fused.py:99-106) with the quantised append;
- ``Kv4Attention``: ``DecodeAttention`` (fused.py:204-234) over the 4-bit cache, and its
  ``decode_qkv`` for the whole of a decode step's attention.

A head vector's values are held in groups of 32, 64 or 128 that share a bf16 scale s and a bf16
value c: x = c + s (n - 8), n = 0..15, within s / 2 of what was written (up to the rounding of
s itself, 2^-8 of up to 8 s); a group of equal bf16 values reads back as it was, a group with a NaN or
an infinity as NaN throughout, a finite group finite. 5, 4.5 or 4.25 bits a value, scales included.

A cache is a uint8 tensor [B, nkv, blocks, bytes]: 32 keys of a (sequence, KV head) pair are one
block (csrc/kv4_core.h has its layout). Blocks must be contiguous; the two outer strides are
free, in multiples of 16 bytes. Slots that were never written may hold anything: nothing reads
past a sequence's length.
"""

import torch

from .. import _lib
from .fused import BF16, _need

KV4_KEYS = 32  # keys of a block


def kv4_block_bytes(d, group):
    """Bytes of a block of 32 keys (K and V): 32 d of codes and 256 a group of scales."""
    _need(d in (64, 128), f"head_dim must be 64 or 128, got {d}")
    _need(group in (32, 64, 128) and group <= d,
          f"group must be 32, 64 or 128 and at most head_dim, got {group}")
    return 32 * d + 256 * (d // group)


_FORMATS = {kv4_block_bytes(d, g): (d, g) for d in (64, 128) for g in (32, 64, 128) if g <= d}


def kv4_cache(B, nkv, cap, d, device, group=32, layers=None):
    """An empty cache for cap keys (rounded up to whole blocks) of B sequences and nkv KV heads:
    uint8 [B, nkv, blocks, bytes], or [layers, ...]."""
    _need(B >= 1 and nkv >= 1 and cap >= 1, "B, nkv and cap must be positive")
    shape = (B, nkv, -(-cap // KV4_KEYS), kv4_block_bytes(d, group))
    return torch.zeros(shape if layers is None else (layers, *shape), dtype=torch.uint8,
                       device=device)


# The current device and its stream's handle, for devices that are known to be initialised: a third
# of the time of torch.cuda.current_device() and of _lib.stream_ptr().
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _lib.stream_ptr)


def _here(dev):
    _need(dev == torch.cuda.current_device(), f"tensors are on cuda:{dev}, the current device is "
          f"cuda:{torch.cuda.current_device()}")


def _tensor(t, name, dtype, shape, dev, contiguous=True):
    _need(isinstance(t, torch.Tensor), f"{name} must be a tensor")
    _need(t.dtype == dtype, f"{name} must be {dtype}, got {t.dtype}")
    _need(tuple(t.shape) == tuple(shape),
          f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    _need(t.is_cuda and t.get_device() == dev, f"{name} must be on cuda:{dev}")
    _need(not contiguous or t.is_contiguous(), f"{name} must be contiguous")
    _need(not t.is_cuda or t.data_ptr() % (4 if dtype == torch.int32 else 16) == 0,
          f"{name} must be aligned to 16 bytes (int32: 4)")


def _no_overlap(t, name):
    """A tensor that is written holds each element once."""
    reach = 0
    for stride, size in sorted((t.stride(i), t.shape[i]) for i in range(t.dim()) if t.shape[i] > 1):
        _need(stride > reach, f"{name}: elements share memory (strides {tuple(t.stride())})")
        reach += stride * (size - 1)


def _meet(a, b):
    """Whether two tensors of one shape, each without elements that share memory, have an element
    in common. Layouts of different strides are taken to, where one lies within the other's reach."""
    size, strides = a.element_size(), sorted(
        ((s, n) for s, n in zip(a.stride(), a.shape) if n > 1), reverse=True)
    span = 1 + sum(s * (n - 1) for s, n in strides)
    other = 1 + sum(s * (n - 1) for s, n in zip(b.stride(), b.shape) if n > 1)
    off = abs(b.data_ptr() - a.data_ptr())
    if off >= size * (span if b.data_ptr() > a.data_ptr() else other):
        return False
    if off % size or strides != sorted(
            ((s, n) for s, n in zip(b.stride(), b.shape) if n > 1), reverse=True):
        return True

    # off = sum of stride * i with |i| < n: the largest stride first, by at most its two neighbours
    def reached(off, i):
        if i == len(strides):
            return off == 0
        stride, n = strides[i]
        return any(abs(k) < n and reached(off - k * stride, i + 1)
                   for k in (off // stride, off // stride + 1))

    return reached(off // size, 0)


def _check_cache(cache, written):
    """The cache's (B, nkv, blocks, d, group, device)."""
    _need(isinstance(cache, torch.Tensor) and cache.dtype == torch.uint8 and cache.dim() == 4,
          "cache must be a uint8 tensor [B, nkv, blocks, bytes]")
    B, nkv, nb, size = cache.shape
    _need(size in _FORMATS, f"cache: {size} bytes are no block's size ({sorted(_FORMATS)})")
    _need(min(B, nkv, nb) >= 1, "cache must not be empty")
    _need(cache.is_cuda, "cache must be on the GPU")
    sb, sh, sk, s1 = cache.stride()
    _need(s1 == 1 and (sk == size or nb == 1) and (sb % 16 == 0 or B == 1)
          and (sh % 16 == 0 or nkv == 1) and cache.data_ptr() % 16 == 0,
          "cache: blocks must be contiguous, outer strides and the address multiples of 16")
    if written:
        _no_overlap(cache, "cache")
    return B, nkv, nb, *_FORMATS[size], cache.get_device()


def _outer(t):
    """The outer strides of a 4-d tensor; those of single rows do not matter."""
    return [t.stride(i) if t.shape[i] > 1 else 0 for i in range(t.dim() - 1)]


def _check_rows(cache, k, v, start, lengths, written, names):
    """What kv4_write and kv4_read check alike, naming what is wrong."""
    B, nkv, nb, d, group, dev = _check_cache(cache, written)
    _here(dev)
    for t, name in ((k, names[0]), (v, names[1])):
        _need(isinstance(t, torch.Tensor) and t.dim() == 4, f"{name} must be [B, nkv, S, d]")
        _tensor(t, name, BF16, (B, nkv, k.shape[2], d), dev, contiguous=False)
        _need(t.stride(3) == 1, f"{name}: the inner stride must be 1")
        _need(all(s % 8 == 0 for s in _outer(t)), f"{name}: strides must be multiples of 8")
        if not written:
            _no_overlap(t, name)
    for t, name in ((start, "start"), (lengths, "lengths")):
        if t is not None:
            _tensor(t, name, torch.int32, (B,), dev)


def _ints(t, B, dev):
    return t is None or (t.dtype is torch.int32 and t.get_device() == dev and t.shape == (B,)
                         and t.is_contiguous())


def _usual(cache, k, v, start, lengths, written):
    """The C arguments of a call that needs no closer look: contiguous outputs, and inputs whose
    strides suit as they are; else None. Tests that could name each fault take 25 us, more
    than a prompt of 500 tokens on the GPU; these take 2."""
    try:
        B, nkv, nb, size = cache.shape
        d, group = _FORMATS[size]
        shape, dev = k.shape, cache.get_device()
        S = shape[2]
        kb, kh, ks, k1 = k.stride()
        vb, vh, vs, v1 = v.stride()
        cp, kp, vp = cache.data_ptr(), k.data_ptr(), v.data_ptr()
        if (shape == v.shape == (B, nkv, S, d) and cache.dtype is torch.uint8
                and k.dtype is v.dtype is BF16 and k1 == v1 == 1
                and (kb | kh | ks | vb | vh | vs) % 8 == 0 and cache.is_contiguous()
                and (written or (k.is_contiguous() and v.is_contiguous()))
                and (cp | kp | vp) % 16 == 0 and B > 0 and nkv > 0 and nb > 0
                and dev == k.get_device() == v.get_device() == _current_device()
                and _ints(start, B, dev) and _ints(lengths, B, dev)):
            return (S, (cp, nkv * nb * size, nb * size), (kp, kb, kh, ks, vp, vb, vh, vs),
                    (None if start is None else start.data_ptr(),
                     None if lengths is None else lengths.data_ptr(),
                     B, S, nkv, nb * KV4_KEYS, d, group), dev)
    except (AttributeError, KeyError, ValueError, IndexError, TypeError, RuntimeError):
        pass   # no tensors of these dimensions: _check_rows says which
    return None


def _rows(cache, k, v, start, lengths, written, names):
    """The checked C arguments of kv4_write and kv4_read."""
    usual = _usual(cache, k, v, start, lengths, written)
    if usual is not None:
        return usual
    _check_rows(cache, k, v, start, lengths, written, names)
    B, nkv, nb, size = cache.shape
    S = k.shape[2]   # single rows' strides may be odd: _outer's are passed
    return (S, (cache.data_ptr(), *_outer(cache)[:2]),
            (k.data_ptr(), *_outer(k), v.data_ptr(), *_outer(v)),
            (_lib.ptr(start), _lib.ptr(lengths), B, S, nkv, nb * KV4_KEYS, *_FORMATS[size]),
            cache.get_device())


def kv4_write(k, v, cache, start=None, lengths=None):
    """Quantise rows of K and V into the cache: row i of sequence b goes to slot start[b] + i.

    k, v: [B, nkv, S, d] bf16, inner stride 1, other strides multiples of 8 (a projection's
    [B, S, nkv, d] transposed serves); start: [B] int32 on the GPU (None: 0); lengths: [B] int32,
    the valid rows of a padded batch (None: S). Rows whose slot lies outside the cache are
    dropped; other slots keep what they hold."""
    S, c, kv, rest, dev = _rows(cache, k, v, start, lengths, True, ("k", "v"))
    if S:
        _lib.call("ko_kv4_write", *kv, *c, *rest, _stream(dev))


def kv4_read(cache, k_out, v_out, start=None, lengths=None):
    """Read cached keys back: row i of k_out and v_out [B, nkv, S, d] bf16 receives the values
    of slot start[b] + i, i < lengths[b] (None: S); other rows are left as they are, as are rows
    whose slot lies outside the cache. The two must not overlap. Strides and the other
    arguments as for kv4_write."""
    S, c, kv, rest, dev = _rows(cache, k_out, v_out, start, lengths, False, ("k_out", "v_out"))
    if S:
        if abs(kv[0] - kv[4]) < 2 * k_out.numel() or not (k_out.is_contiguous()
                                                          and v_out.is_contiguous()):
            _need(not _meet(k_out, v_out), "k_out and v_out must not overlap")
        _lib.call("ko_kv4_read", *c, *kv, *rest, _stream(dev))


def _check_qkv(qkv, q_w, k_w, cos, sin, pos, rows, B, nq, nkv, d, dev):
    """The addresses of the first five, and the rows that both tables have."""
    try:   # the usual call, 1.5 us; the tests below name what is wrong
        (rc, dc), (rs, ds) = cos.shape, sin.shape
        ptrs = (qkv.data_ptr(), q_w.data_ptr(), k_w.data_ptr(), cos.data_ptr(), sin.data_ptr())
        if (qkv.shape == (rows, (nq + 2 * nkv) * d) and q_w.shape == k_w.shape == (d,)
                and pos.shape == (B,) and dc == ds == d and rc > 0 and rs > 0
                and qkv.dtype is q_w.dtype is k_w.dtype is cos.dtype is sin.dtype is BF16
                and pos.dtype is torch.int32 and qkv.is_contiguous() and q_w.is_contiguous()
                and k_w.is_contiguous() and cos.is_contiguous() and sin.is_contiguous()
                and pos.is_contiguous() and dev == qkv.get_device() == q_w.get_device()
                == k_w.get_device() == cos.get_device() == sin.get_device() == pos.get_device()
                and (ptrs[0] | ptrs[1] | ptrs[2] | ptrs[3] | ptrs[4]) % 16 == 0):
            return ptrs, rc if rc < rs else rs
    except (AttributeError, ValueError, TypeError, RuntimeError):
        pass
    _tensor(qkv, "qkv", BF16, (rows, (nq + 2 * nkv) * d), dev)
    _tensor(q_w, "q_w", BF16, (d,), dev)
    _tensor(k_w, "k_w", BF16, (d,), dev)
    for t, name in ((cos, "cos"), (sin, "sin")):
        _need(isinstance(t, torch.Tensor) and t.dim() == 2 and t.shape[0] >= 1,
              f"{name} must be [rows, d]")
        _tensor(t, name, BF16, (t.shape[0], d), dev)
    _tensor(pos, "pos", torch.int32, (B,), dev)
    return tuple(t.data_ptr() for t in (qkv, q_w, k_w, cos, sin)), min(cos.shape[0], sin.shape[0])


def kv4_append(qkv, q_w, k_w, cos, sin, pos, q_out, cache, T, eps, nq, nkv, d):
    """qk_norm_rope over the 4-bit cache: qkv [B*T, (nq+2nkv)*d] bf16, row m is sequence m // T at
    position pos[b] + m % T. Per-head RMSNorm and RoPE of q into q_out [B*T, nq*d], of k into
    the cache's slot at that position with v, both quantised. Everything is fp32 up to the one
    rounding of q and the quantisation of k. Positions outside the cache or the RoPE tables
    [rows, d] are skipped (their q_out rows too). q_out must not overlap qkv; of a single row it
    may be the first nq*d values."""
    try:   # the usual call; the tests below name what is wrong
        B, ck, nb, size = cache.shape
        cd, group = _FORMATS[size]
        dev, qp, cp = cache.get_device(), q_out.data_ptr(), cache.data_ptr()
        cb, ch = ck * nb * size, nb * size
        usual = (cache.dtype is torch.uint8 and cache.is_contiguous() and ck == nkv and cd == d
                 and T >= 1 and nq >= 1 and B > 0 and nkv > 0 and nb > 0
                 and q_out.shape == (B * T, nq * d) and q_out.dtype is BF16
                 and q_out.is_contiguous() and (qp | cp) % 16 == 0
                 and dev == q_out.get_device() == _current_device())
    except (AttributeError, KeyError, ValueError, TypeError, RuntimeError):
        usual = False
    if not usual:
        B, ck, nb, cd, group, dev = _check_cache(cache, True)
        _here(dev)
        _need(T >= 1 and nq >= 1, "T and nq must be positive")
        _need((ck, cd) == (nkv, d), f"cache has {ck} heads of {cd}, not {nkv} of {d}")
        _tensor(q_out, "q_out", BF16, (B * T, nq * d), dev)
        qp, cp, (cb, ch, _) = q_out.data_ptr(), cache.data_ptr(), _outer(cache)
    ptrs, n_rows = _check_qkv(qkv, q_w, k_w, cos, sin, pos, B * T, B, nq, nkv, d, dev)
    off, row = qp - ptrs[0], 2 * B * T * d   # bytes
    _need(off >= row * (nq + 2 * nkv) or -off >= row * nq or (off == 0 and B * T == 1),
          "q_out must not overlap qkv")
    _lib.call("ko_kv4_append", *ptrs, pos.data_ptr(), qp, cp, B * T, T, cb, ch, eps, nq, nkv, d,
              group, min(nb * KV4_KEYS, n_rows), None, _stream(dev))


class Kv4Attention:
    """Decode attention over a 4-bit cache for T query tokens per sequence, fixed (B, T, cap); cap is
    rounded up to whole blocks, as kv4_cache does.

    Any number of query heads per KV head and tokens with T * nq / nkv <= 64, T <= 8; head_dim 64
    or 128. A query row that sees no key is zero. Sums run unnormalised in fp32: |v|
    times the number of keys may reach 2^115, and |q . k| 1e30. Calls of one object share its workspace:
    they must not overlap on two streams, nor may graphs captured from them.
    """

    MAX_T = 8
    GRID = 512     # workgroups of 4 wavefronts: two on each of the 256 CUs
    MIN_RUN = 8    # least steps of 32 keys in a workgroup's run
    PAIR_STEPS, MAX_STEPS = 24, (1 << 24) - GRID - MIN_RUN   # the C entry's limit

    def __init__(self, B, T, cap, nq, nkv, d, device, group=32):
        self.block_bytes = kv4_block_bytes(d, group)
        _need(B >= 1 and cap >= 1 and nkv >= 1 and nq >= 1 and nq % nkv == 0,
              "B, cap and nkv must be positive, nq a multiple of nkv")
        _need(1 <= T <= self.MAX_T, f"T must be in 1..{self.MAX_T}")
        _need(T * (nq // nkv) <= 64, "at most 64 query rows (T * nq / nkv) a KV head")
        self.B, self.T, self.nq, self.nkv, self.d, self.group = B, T, nq, nkv, d, group
        dev = torch.device(device)
        _need(dev.type == "cuda", "device must be a GPU")
        self.blocks = -(-cap // KV4_KEYS)
        self.cap = self.blocks * KV4_KEYS
        _need(B * nkv * (self.blocks + self.PAIR_STEPS) <= self.MAX_STEPS,
              f"B * nkv * blocks of {KV4_KEYS} keys must stay below 2^24")
        self.device = torch.cuda.current_device() if dev.index is None else dev.index
        self.scale = d ** -0.5
        # Workspace: the runs' partial sums, and arrival counters that are zero before the first
        # call and left zero by every call. Whatever stream that call is on, their fill must be
        # done: the constructor waits for it, which a capture does not allow.
        _need(not torch.cuda.is_current_stream_capturing(), "make the object before the capture")
        self.grid = self.GRID
        self._part = torch.empty(_lib.lib().ko_kv4_attn_scratch(T * nq // nkv, d, group, self.grid),
                                 dtype=torch.float32, device=dev)
        self._counters = torch.zeros(self.grid, dtype=torch.int32, device=dev)
        torch.cuda.current_stream(dev).synchronize()
        self._work = self._part.data_ptr(), self._part.numel(), self._counters.data_ptr()
        self._q = torch.empty(B, nq * d, dtype=BF16, device=dev) if T == 1 else None
        self._q_shape = torch.Size((B * T, nq * d))
        self._q_bytes = 2 * B * T * nq * d
        self._cache_shape = torch.Size((B, nkv, self.blocks, self.block_bytes))
        self._len_shape = torch.Size((B,))

    def _check_cache(self, cache, written=False):
        _need(isinstance(cache, torch.Tensor) and cache.shape == self._cache_shape,
              f"cache must be a uint8 tensor {list(self._cache_shape)}")
        _need(_check_cache(cache, written)[5] == self.device, f"cache must be on cuda:{self.device}")

    def _run(self, q, cache, lens, len_offset, out):
        dev = self.device
        try:   # the usual call; the tests below name what is wrong
            qp, cp, op = q.data_ptr(), cache.data_ptr(), out.data_ptr()
            usual = (q.shape == out.shape == self._q_shape and q.dtype is out.dtype is BF16
                     and q.is_contiguous() and out.is_contiguous() and lens.shape == self._len_shape
                     and lens.dtype is torch.int32 and lens.is_contiguous()
                     and cache.shape == self._cache_shape and cache.dtype is torch.uint8
                     and cache.is_contiguous() and dev == q.get_device() == out.get_device()
                     == lens.get_device() == cache.get_device() and (qp | cp | op) % 16 == 0)
        except (AttributeError, ValueError, TypeError, RuntimeError):
            usual = False
        if not usual:
            _tensor(q, "q", BF16, self._q_shape, dev)
            _tensor(out, "out", BF16, self._q_shape, dev)
            _tensor(lens, "pos/lengths", torch.int32, self._len_shape, dev)
            self._check_cache(cache)
        if dev != _current_device():
            _here(dev)
        _need(abs(qp - op) >= self._q_bytes, "out must not overlap q")
        cb, ch, _, _ = cache.stride()
        if cb % 16 or ch % 16:   # strides of single rows
            cb, ch, _ = _outer(cache)
        _lib.call("ko_kv4_attn", qp, cp, cb, ch, lens.data_ptr(), len_offset, self.cap, self.B,
                  self.T, self.nq, self.nkv, self.d, self.group, self.scale, *self._work, self.grid,
                  self.MIN_RUN, op, _stream(dev))

    def __call__(self, q, cache, pos, out):
        """q: [B*T, nq*d] bf16; cache: [B, nkv, blocks, bytes]; pos: [B] int32, the position of a
        sequence's first query (keys 0 .. pos + T - 1 are cached, query t sees those up to pos +
        t, none behind the cache's end); out: [B*T, nq*d] bf16."""
        self._run(q, cache, pos, self.T, out)

    def with_lengths(self, q, cache, lengths, out):
        """lengths[b] = number of cached keys of sequence b (int32); its T queries sit at the last
        T positions. Rows in front of the first key (lengths[b] < T) are zero. A length that passes
        the cache's end places the queries; the keys are those up to the end."""
        self._run(q, cache, lengths, 0, out)

    def decode_qkv(self, qkv, q_w, k_w, cos, sin, pos, cache, out, eps, rope=None):
        """A decode step's attention (T = 1) straight from the bf16 QKV projection [B, (nq+2nkv)*d]:
        kv4_append at pos[b], then attention over keys 0..pos[b]. A sequence whose
        position lies outside the cache or the RoPE tables appends nothing and its row of
        out is zero. rope ([B, 2, d] bf16, optional): the cos and sin rows at pos[b], as
        fused.rope_rows writes them."""
        _need(self.T == 1, "decode_qkv serves one decode token per sequence")
        B, nq, nkv, d, dev = self.B, self.nq, self.nkv, self.d, self.device
        try:   # the usual call; the tests below name what is wrong
            cp, op = cache.data_ptr(), out.data_ptr()
            usual = (cache.shape == self._cache_shape and cache.dtype is torch.uint8
                     and cache.is_contiguous() and out.shape == self._q_shape and out.dtype is BF16
                     and out.is_contiguous() and (cp | op) % 16 == 0
                     and dev == cache.get_device() == out.get_device() == _current_device())
        except (AttributeError, ValueError, TypeError, RuntimeError):
            usual = False
        if not usual:
            self._check_cache(cache, True)
            _tensor(out, "out", BF16, self._q_shape, dev)
            _here(dev)
        ptrs, n_rows = _check_qkv(qkv, q_w, k_w, cos, sin, pos, B, B, nq, nkv, d, dev)
        if rope is not None:
            _tensor(rope, "rope", BF16, (B, 2, d), dev)
        cb, ch, _, _ = cache.stride()
        if cb % 16 or ch % 16:   # strides of single rows
            cb, ch, _ = _outer(cache)
        _lib.call("ko_kv4_attn_qkv", *ptrs, n_rows, pos.data_ptr(), cp, cb, ch, self.cap, B,
                  nq, nkv, d, self.group, eps, self.scale, self._q.data_ptr(), *self._work,
                  self.grid, self.MIN_RUN, op, _lib.ptr(rope), _stream(dev))
