"""Drawing the next tokens from logits, by temperature, top-k, top-p and min-p.

``Sampler`` stands where the engine's greedy steps have ``argmax_rows`` (the reference's
torch.argmax, engine/engine.py:299, 397), with random numbers that the caller gives: the same numbers
draw the same tokens, on any machine and however the rows are batched. Tensors are the caller's,
every call launches on the current stream of the current device, allocates nothing and never
synchronises (so calls can be captured), and a bad argument raises ValueError before anything is
launched.
"""

import torch

from .. import _lib
from .fused import BF16, _cdiv, _need
from .kv4 import _current_device, _here, _stream

F32 = torch.float32
MAX_VOCAB = 1 << 20
MAX_ROWS = 65535


def _chunks(B, V):
    """Workgroups that a row is cut into: enough rows fill the GPU by themselves."""
    return max(1, min(_cdiv(V, 4096), 512 // B))


class Sampler:
    """Draws one token for each of B rows of V logits.

    A row's tokens in order of falling logit (ties: the lowest index first), with probabilities
    softmax(logits / temperature), pass three filters, each of which keeps a beginning of the order:
    ``top_k`` the first k tokens (0: all), ``top_p`` those with less than p of the mass that top_k left
    before them (1: all), ``min_p`` those of at least min_p times the largest probability (0: all);
    the first token is always kept. The token is drawn in which u times the kept mass falls, in the same
    order. Temperature 0 takes the first token. Masses are held to 2^-43 of the largest
    probability, below which a token is never drawn. NaN counts as -infinity; a row with nothing above -infinity gets the id -1.

    The object holds the scratch of its calls: they must be ordered, on one stream or by events,
    captured calls' replays included, and it has to outlive the graphs that captured them."""

    def __init__(self, B, V, device):
        _need(1 <= B <= MAX_ROWS, f"B must be 1 to {MAX_ROWS}")
        _need(1 <= V <= MAX_VOCAB, f"V must be 1 to {MAX_VOCAB}")
        device = torch.device(device)
        _need(device.type == "cuda", "device must be a GPU")
        self.B, self.V, self.chunks = B, V, _chunks(B, V)
        n = _lib.lib().ko_sample_scratch(B, self.chunks)
        self._scratch = torch.empty(max(n, 16), dtype=torch.uint8, device=device)
        self._dev = self._scratch.get_device()

    def __call__(self, logits, u, ids, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
                 logprobs=None):
        """ids [B] int64 receives the tokens drawn from logits [B, V] (bf16 or fp32, inner stride 1)
        with u [B] fp32 of [0, 1) (below 0 or NaN: 0; from 1 on: the last kept token).

        temperature, top_k, top_p and min_p are numbers for all rows (temperature >= 0, top_k >= 0,
        top_p and min_p of [0, 1]) or tensors [B] on the GPU (fp32, top_k int32), whose values are read
        as the call runs: a temperature that is not above 0 is 0, a top_k below 1 is 0, a top_p that
        is not below 1 is 1, a min_p that is not above 0 is 0. logprobs [B] fp32 (optional)
        receives the log of the token's share of the kept mass (0 where the first token is
        taken, -infinity beside the id -1). ids and logprobs must not overlap the other tensors."""
        B, V, dev = self.B, self.V, self._dev
        usual = self._usual(logits, u, ids, logprobs)
        if usual is None:
            _here(dev)
            _need(isinstance(logits, torch.Tensor) and logits.dtype in (BF16, F32)
                  and tuple(logits.shape) == (B, V), f"logits must be [{B}, {V}] in bf16 or fp32")
            _need(logits.is_cuda and logits.get_device() == dev, f"logits must be on cuda:{dev}")
            _need(logits.stride(1) == 1 or V == 1, "logits: the inner stride must be 1")
            _vector(u, "u", F32, B, dev)
            _vector(ids, "ids", torch.int64, B, dev)
            if logprobs is not None:
                _vector(logprobs, "logprobs", F32, B, dev)
            usual = (logits.data_ptr(), u.data_ptr(), ids.data_ptr(), _lib.ptr(logprobs))
        t = _setting(temperature, "temperature", F32, B, dev, _at_least_0)
        k = _setting(top_k, "top_k", torch.int32, B, dev, _whole)
        p = _setting(top_p, "top_p", F32, B, dev, _share)
        m = _setting(min_p, "min_p", F32, B, dev, _share)
        # outputs apart from what a row's other workgroups still read
        ins = [(usual[0], logits.element_size() * ((B - 1) * logits.stride(0) + V)), (usual[1], 4 * B)]
        ins += [(a, 4 * B) for a, _ in (t, k, p, m) if a]
        outs = [(usual[2], 8 * B)] + ([(usual[3], 4 * B)] if usual[3] else [])
        for a, n in outs:
            for c, size in ins + [o for o in outs if o[0] != a]:
                if a < c + size and c < a + n:
                    raise ValueError("ids and logprobs must not overlap what the call reads, or each other")
        if len(outs) == 2 and outs[0][0] == outs[1][0]:
            raise ValueError("ids and logprobs must not overlap")
        _lib.call("ko_sample", usual[0], logits.dtype is F32, logits.stride(0) if B > 1 else 0, B, V,
                  usual[1], *t, k[0], min(int(k[1]), V), *p, *m, usual[2], usual[3],
                  self._scratch.data_ptr(), self._scratch.numel(), self.chunks, _stream(dev))

    def _usual(self, logits, u, ids, logprobs):
        """The addresses of a call that needs no closer look, else None."""
        try:
            B, dev = self.B, self._dev
            if (logits.shape == (B, self.V) and logits.dtype in (BF16, F32) and logits.is_contiguous()
                    and u.dtype is F32 and ids.dtype is torch.int64 and u.shape == ids.shape == (B,)
                    and u.is_contiguous() and ids.is_contiguous()
                    and dev == logits.get_device() == u.get_device() == ids.get_device()
                    == _current_device()):
                if logprobs is None:
                    return logits.data_ptr(), u.data_ptr(), ids.data_ptr(), None
                if (logprobs.dtype is F32 and logprobs.shape == (B,) and logprobs.is_contiguous()
                        and logprobs.get_device() == dev):
                    return logits.data_ptr(), u.data_ptr(), ids.data_ptr(), logprobs.data_ptr()
        except (AttributeError, TypeError, RuntimeError):
            pass   # no tensors: the tests above say which
        return None


def _at_least_0(v):
    return v >= 0


def _whole(v):
    return v >= 0 and (isinstance(v, int) or v.is_integer())


def _share(v):
    return 0 <= v <= 1


def _vector(t, name, dtype, B, dev):
    _need(isinstance(t, torch.Tensor) and t.dtype == dtype and tuple(t.shape) == (B,)
          and t.is_contiguous(), f"{name} must be a contiguous {dtype} tensor [{B}]")
    _need(t.is_cuda and t.get_device() == dev, f"{name} must be on cuda:{dev}")


def _setting(v, name, dtype, B, dev, valid):
    """(address, value) of a setting, one of them unused."""
    if isinstance(v, torch.Tensor):
        if not (v.dtype is dtype and v.shape == (B,) and v.is_contiguous() and v.get_device() == dev):
            _vector(v, name, dtype, B, dev)   # says what is wrong
        return v.data_ptr(), 0
    if not (isinstance(v, (int, float)) and valid(v)):
        raise ValueError(f"{name} is out of range: {v!r}")
    return None, v
