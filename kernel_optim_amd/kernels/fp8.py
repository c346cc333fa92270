"""Matrices held in 8-bit floating point, and the projections of a decode step or a prompt on them.

The ops stand beside ``kernels.gemv``'s for bf16 weights and follow their manner: tensors are the
caller's, every call launches on the current stream of the current device and never synchronises
(so calls can be captured), and a bad argument raises ValueError before anything is launched
(RuntimeError where a call is too large for one launch: 2^26 blocks to read, 2^26 runs of 4 to write).

- ``fp8_quantize``: rows [rows, K] in bf16 or fp32, behind an RMSNorm if asked, to 8 bits (a
  weight once at load, a projection's input in every call); ``fp8_read`` gives the values back,
  ``fp8_slice`` a part of the rows;
- ``Fp8Linear``: ``Gemv`` (engine/kernels/gemv.py:109-150) with both factors in 8 bits, for any
  number of rows: y = x W^T with a norm in front and the F32, BF16, RESID or SWIGLU epilogue.

A value is held as an OCP e4m3 code times its block's scale, a power of two: a block is 128
neighbouring values of a row, and the scale the least 2^e >= 2^-127 with max |x| <= 448 * 2^e. A code
is x / 2^e rounded to nearest (ties to even; at e = 120 256 becomes 240, as 2^128 is no number of
either type): within 2^-4 of x, or within 2^(e - 10) where |x| is below 2^(e - 6). A block with a
NaN or an infinity reads back as NaN throughout. 8.06 bits a value. K is a multiple of 8, up to 2^27;
the last block may be short.
"""

import torch

from .. import _lib
from .fused import BF16, _cdiv, _need
from .gemv import EPI_BF16, EPI_F32, EPI_RESID, EPI_SWIGLU
from .kv4 import _current_device, _here, _no_overlap, _stream, _tensor

F32 = torch.float32
FP8_BLOCK = 128   # values that share a scale
NORM_K = 2 ** 17   # the longest rows that a norm in front takes


class Fp8Tensor:
    """A matrix [rows, K] in 8 bits: ``codes`` uint8 [tiles, blocks, 2048] (16 rows x 128 values a
    block) and ``scales`` uint8 [tiles, quads, 64] (16 rows x 4 blocks), as csrc/fp8_core.h lays
    them out. ``pair``: a tile has 8 rows of each half of the rows (gate | up)."""

    __slots__ = ("codes", "scales", "rows", "K", "pair")

    def __init__(self, codes, scales, rows, K, pair=False):
        tiles, blocks = fp8_shape(rows, K, pair)
        for t, name, shape in ((codes, "codes", (tiles, blocks, 2048)),
                               (scales, "scales", (tiles, _cdiv(blocks, 4), 64))):
            _need(isinstance(t, torch.Tensor) and t.dtype == torch.uint8 and t.shape == shape
                  and t.is_contiguous(), f"{name} must be a contiguous uint8 tensor {shape}")
        _need(codes.device == scales.device, "codes and scales must be on one device")
        self.codes, self.scales, self.rows, self.K, self.pair = codes, scales, rows, K, bool(pair)

    @property
    def nbytes(self):
        return self.codes.numel() + self.scales.numel()

    def __repr__(self):
        return (f"Fp8Tensor([{self.rows}, {self.K}]{', pair' if self.pair else ''}, "
                f"{self.codes.device})")


def fp8_shape(rows, K, pair=False):
    """(tiles of 16 rows, blocks of 128 values) of a matrix [rows, K]."""
    _need(rows >= 1 and K >= 8 and K % 8 == 0, "rows must be positive, K a positive multiple of 8")
    _need(not pair or rows % 2 == 0, "a pair has an even number of rows")
    tiles = _cdiv(rows // 2, 8) if pair else _cdiv(rows, 16)
    blocks = _cdiv(K, FP8_BLOCK)
    _need(tiles * blocks < 2 ** 31, "the matrix has 2^31 blocks or more")
    _need(rows < 2 ** 31 and K <= 2 ** 27, f"2^31 rows or more, or more than 2^27 columns: [{rows}, {K}]")
    return tiles, blocks


def fp8_empty(rows, K, device, pair=False):
    """An Fp8Tensor [rows, K] to be written by fp8_quantize."""
    tiles, blocks = fp8_shape(rows, K, pair)
    return Fp8Tensor(torch.empty(tiles, blocks, 2048, dtype=torch.uint8, device=device),
                     torch.empty(tiles, _cdiv(blocks, 4), 64, dtype=torch.uint8, device=device),
                     rows, K, pair)


def fp8_slice(t, begin, end):
    """Rows begin .. end - 1 of t, which share its memory: begin a multiple of 16, end too unless it is
    the last row. Not of a pair."""
    _need(isinstance(t, Fp8Tensor) and not t.pair, "t must be an Fp8Tensor that is no pair")
    _need(0 <= begin < end <= t.rows and begin % 16 == 0 and (end % 16 == 0 or end == t.rows),
          f"rows {begin} to {end} of {t.rows} are not whole tiles")
    at = slice(begin // 16, _cdiv(end, 16))
    return Fp8Tensor(t.codes[at], t.scales[at], end - begin, t.K)


def _check_held(t, name, rows, K, pair, dev):
    # without a fault no message is made: it would take longer than the test
    if (isinstance(t, Fp8Tensor) and t.rows == rows and t.K == K and t.pair == pair
            and t.codes.get_device() == dev >= 0
            and not (t.codes.data_ptr() | t.scales.data_ptr()) & 15):
        return
    _need(isinstance(t, Fp8Tensor), f"{name} must be an Fp8Tensor (fp8_quantize)")
    _need((t.rows, t.K, t.pair) == (rows, K, pair),
          f"{name} must hold [{rows}, {K}]{' as a pair' if pair else ''}, got {t!r}")
    _need(t.codes.is_cuda and t.codes.get_device() == dev, f"{name} must be on cuda:{dev}")
    _need((t.codes.data_ptr() | t.scales.data_ptr()) % 16 == 0, f"{name} must be aligned to 16 bytes")


def _check_rows(x, name, dtypes):
    """A matrix of rows: its device and row stride."""
    if (isinstance(x, torch.Tensor) and x.dim() == 2 and x.dtype in dtypes and x.is_cuda
            and x.is_contiguous() and x.numel() and not x.shape[1] & 7 and not x.data_ptr() & 15):
        return x.get_device(), x.shape[1] if x.shape[0] > 1 else 0
    _need(isinstance(x, torch.Tensor) and x.dim() == 2, f"{name} must be [rows, K]")
    _need(x.dtype in dtypes, f"{name} must be {' or '.join(map(str, dtypes))}, got {x.dtype}")
    _need(x.is_cuda, f"{name} must be on the GPU")
    rows, K = x.shape
    _need(rows >= 1 and K >= 8 and K % 8 == 0,
          f"{name} must have rows, and columns in a multiple of 8, got {tuple(x.shape)}")
    stride = x.stride(0) if rows > 1 else 0
    _need(x.stride(1) == 1 and stride % 8 == 0 and stride >= 0 and x.data_ptr() % 16 == 0,
          f"{name}: the inner stride must be 1, the row stride a multiple of 8, the address of 16")
    return x.get_device(), stride


def _bytes(t):
    """A tensor's first byte and the one behind its last (strides >= 0)."""
    reach = t.numel() if t.is_contiguous() else sum(
        (n - 1) * s for n, s in zip(t.shape, t.stride())) + 1
    return t.data_ptr(), t.data_ptr() + reach * t.element_size()


def _need_apart(a, b, what):
    (a0, a1), (b0, b1) = _bytes(a), _bytes(b)
    _need(a1 <= b0 or b1 <= a0, f"{what} must not overlap")


def fp8_quantize(x, out=None, nw=None, eps=1e-6, pair=False):
    """Quantise rows x [rows, K] (bf16 or fp32, inner stride 1, row stride a multiple of 8 or 0) into
    ``out`` (None: a new Fp8Tensor), which is returned. ``nw`` [K] bf16, K <= 2^17: bf16 rows go through an
    RMSNorm with this gain first, rounded as the bf16 chain is (bf16(nw * bf16(x * rstd)), a block's
    squares summed in fp32, the blocks in 64 bits).
    ``pair``: x is gate | up, [2 N, K], for an Fp8Linear with SWIGLU; ``out`` says so itself."""
    dev, stride = _check_rows(x, "x", (BF16, F32))
    _here(dev)
    rows, K = x.shape
    if nw is not None:
        _need(x.dtype == BF16 and not pair and not (isinstance(out, Fp8Tensor) and out.pair),
              "a norm goes with bf16 rows that are no pair")
        _need(K <= NORM_K, f"a norm goes with rows of up to {NORM_K} values, got {K}")
        _tensor(nw, "nw", BF16, (K,), dev)
    if out is None:
        out = fp8_empty(rows, K, x.device, pair)
    else:
        _check_held(out, "out", rows, K, out.pair if isinstance(out, Fp8Tensor) else pair, dev)
        _need(out.pair or not pair, "out holds no pair")
        for t in (x,) if nw is None else (x, nw):
            _need_apart(t, out.codes, "out and what it is made of")
            _need_apart(t, out.scales, "out and what it is made of")
    _lib.call("ko_fp8_quantize", x.data_ptr(), x.dtype == F32, stride, rows, K, out.pair,
              _lib.ptr(nw), eps, out.codes.data_ptr(), out.scales.data_ptr(), _stream(dev))
    return out


def fp8_read(t, out):
    """The values that t holds, into out [rows, K] bf16 or fp32 (strides as x's of fp8_quantize;
    elements must not share memory); exact in either but for values below the type's
    least subnormal."""
    dev, stride = _check_rows(out, "out", (BF16, F32))
    _here(dev)
    _need(isinstance(t, Fp8Tensor), "t must be an Fp8Tensor (fp8_quantize)")
    _check_held(t, "t", out.shape[0], out.shape[1], t.pair, dev)
    if not out.is_contiguous():
        _no_overlap(out, "out")
    _need_apart(out, t.codes, "t and out")
    _need_apart(out, t.scales, "t and out")
    _lib.call("ko_fp8_read", t.codes.data_ptr(), t.scales.data_ptr(), t.rows, t.K, t.pair,
              out.data_ptr(), out.dtype == F32, stride, _stream(dev))


class Fp8Linear:
    """One projection y[M, N] = x[M, K] W[N, K]^T, x and W in 8 bits, sums in fp32, with a norm in
    front (``norm``, gain ``nw``, K <= 2^17) and an epilogue: EPI_F32 (y fp32), EPI_BF16, EPI_RESID
    (y = bf16(h + bf16(x W^T)); y None: h itself) or EPI_SWIGLU (W is gate | up held as a pair;
    y = bf16(bf16(silu(g)) * u) of the bf16 products g and u).

    Up to 32 rows, and for fp32 results, every product of codes enters the sum whole; beyond, the 8-bit
    matrix instruction cuts 8 neighbouring products off 2^-13 below the largest one's binade: sums come
    out 2^-14 off as a rule, and some bf16 results (step 2^-8) are another in their last bit.

    ``x`` is [M, K] bf16 and is quantised in the call (with the norm) into a workspace of the object's,
    or an Fp8Tensor where there is no norm; with ``held`` always the latter, and the workspace, M K bytes
    otherwise, is small. The workspace is made for ``device``, or in the first call, which must not be
    under graph capture, on the stream that is current then. The object stays on that device, and has
    to outlive the graphs that captured its calls. Calls of one object share the workspace: they
    must be ordered behind its making and each other, on one stream or by events, captured calls'
    replays included. y (and h where it is y) must not overlap x, nw or w."""

    def __init__(self, M, N, K, epi, norm, eps=1e-6, device=None, held=False):
        _need(epi in (EPI_F32, EPI_BF16, EPI_RESID, EPI_SWIGLU), f"bad epilogue {epi}")
        _need(M >= 1 and N >= 1, "M and N must be positive")
        fp8_shape((2 if epi == EPI_SWIGLU else 1) * N, K, epi == EPI_SWIGLU)
        fp8_shape(M, K)
        _need(not norm or K <= NORM_K, f"a norm goes with rows of up to {NORM_K} values, got {K}")
        _need(not (norm and held), "a norm goes with x in bf16")
        self.M, self.N, self.K, self.epi, self.norm, self.eps = M, N, K, epi, bool(norm), eps
        self.held = bool(held)
        self._dev = self._xq = self._scratch = None
        wide = (2 if epi == EPI_SWIGLU else 1) * N
        tiles, blocks = fp8_shape(wide, K, epi == EPI_SWIGLU)
        # what _usual compares with: shapes, W's rows, and bytes of x, y, h, nw and W
        self._x, self._y, self._nw = torch.Size((M, K)), torch.Size((M, N)), torch.Size((K,))
        self._rows, self._dtype = wide, F32 if epi == EPI_F32 else BF16
        self._bytes = (2 * M * K, M * N * (4 if epi == EPI_F32 else 2), 2 * M * N, 2 * K,
                       tiles * blocks * 2048, tiles * _cdiv(blocks, 4) * 64)
        if device is not None:
            device = torch.device(device)
            _need(device.type == "cuda", "device must be a GPU")
            self._workspace(torch.cuda.current_device() if device.index is None else device.index)

    def _workspace(self, dev):
        if self._dev is None:
            _need(not torch.cuda.is_current_stream_capturing(), "the workspace is made in the first "
                  "call: make it before the capture, or give the object its device")
            at = torch.device("cuda", dev)
            n = _lib.lib().ko_fp8_linear_scratch(self.M, self.N, self.K, self.epi)
            # the counters among it start at zero, and every call leaves them there
            self._scratch = torch.zeros(max(n, 16), dtype=torch.uint8, device=at)
            self._xq = None if self.held else fp8_empty(self.M, self.K, at)
            self._dev = dev
        # a new one would free what captured calls use
        _need(self._dev == dev, f"the object's workspace is on cuda:{self._dev}: make another object "
              f"for cuda:{dev}")
        return self._xq

    def _usual(self, x, w, y, nw, h):
        """The C arguments of a call that needs no closer look, else None: tests that name each
        fault take longer than a short call on the GPU."""
        try:
            q = self._xq
            dev, epi = q.codes.get_device(), self.epi
            nx, ny, nh, nn, nc, ns = self._bytes
            hp = np = 0
            if epi == EPI_RESID:
                hp = h.data_ptr()
                if y is None:
                    y = h
                if not (h.dtype is BF16 and h.shape == self._y and h.is_contiguous()
                        and h.get_device() == dev and (y is h or abs(y.data_ptr() - hp) >= nh)):
                    return None
            elif h is not None:
                return None
            if self.norm:
                if not (nw.dtype is BF16 and nw.shape == self._nw and nw.is_contiguous()
                        and nw.get_device() == dev):
                    return None
                np = nw.data_ptr()
            elif nw is not None:
                return None
            wc, ws, xp, yp = w.codes, w.scales, x.data_ptr(), y.data_ptr()
            cp, sp = wc.data_ptr(), ws.data_ptr()
            # y apart from what other workgroups still read
            if (-ny < yp - xp < nx or -ny < yp - cp < nc or -ny < yp - sp < ns
                    or np and -ny < yp - np < nn):
                return None
            if (type(w) is Fp8Tensor and w.rows == self._rows and w.K == self.K
                    and w.pair is (epi == EPI_SWIGLU) and x.shape == self._x and y.shape == self._y
                    and x.dtype is BF16 and y.dtype is self._dtype and x.is_contiguous()
                    and y.is_contiguous() and dev == wc.get_device() == x.get_device()
                    == y.get_device() == _current_device()
                    and not (xp | yp | cp | sp | np | hp) & 15):
                t = self._scratch
                return (xp, np or None, self.eps, q.codes.data_ptr(), q.scales.data_ptr(), cp, sp, yp,
                        hp or None, t.data_ptr(), t.numel(), self.M, self.N, self.K, epi,
                        _stream(dev))
        except (AttributeError, TypeError, RuntimeError):
            pass   # no tensors: the tests below say which
        return None

    def __call__(self, x, w, y=None, nw=None, h=None):
        usual = self._usual(x, w, y, nw, h)
        if usual is not None:
            _lib.call("ko_fp8_linear", *usual)
            return
        M, N, K, epi = self.M, self.N, self.K, self.epi
        _need(isinstance(w, Fp8Tensor), "w must be an Fp8Tensor (fp8_quantize)")
        _need(w.codes.is_cuda, "w must be on the GPU")
        dev = w.codes.get_device()
        _here(dev)
        pair = epi == EPI_SWIGLU
        _check_held(w, "w", 2 * N if pair else N, K, pair, dev)
        _need((nw is not None) == self.norm, "nw goes with a norm")
        if epi == EPI_RESID:
            _tensor(h, "h", BF16, (M, N), dev)
            y = h if y is None else y
        else:
            _need(h is None, "h goes with EPI_RESID")
        _tensor(y, "y", F32 if epi == EPI_F32 else BF16, (M, N), dev)
        if y is not h and epi == EPI_RESID and y.data_ptr() != h.data_ptr():
            _need_apart(y, h, "y and h, unless they are the same,")
        if isinstance(x, Fp8Tensor):
            _need(not self.norm, "a norm goes with x in bf16")
            _check_held(x, "x", M, K, False, dev)
            self._workspace(dev)
            q, x = x, None
        else:
            _need(not self.held, "x must be an Fp8Tensor, as the object was made with held")
            _tensor(x, "x", BF16, (M, K), dev)
            if self.norm:
                _tensor(nw, "nw", BF16, (K,), dev)
            q = self._workspace(dev)
        for t in (x, nw, w.codes, w.scales, q.codes, q.scales):   # other workgroups still read these
            if t is not None:
                _need_apart(y, t, "y and what the call reads (but h)")
        _lib.call("ko_fp8_linear", _lib.ptr(x), _lib.ptr(nw), self.eps, q.codes.data_ptr(),
                  q.scales.data_ptr(), w.codes.data_ptr(), w.scales.data_ptr(), y.data_ptr(),
                  _lib.ptr(h), self._scratch.data_ptr(), self._scratch.numel(), M, N, K, epi,
                  _stream(dev))
