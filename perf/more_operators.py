"""The operators of 8-bit projections and of sampling, as cases that can be timed and checked.

Three kinds, each through public entry points:

- ``quant`` (``kernel_optim_amd.kernels.fp8``): rows quantised to 8-bit floating point (e4m3)
  with a scale for each block of 128 values of a row, behind an RMSNorm or not, and read back;
- ``linear`` (same module): a projection of a decode step or a prompt, y = x W^T, with x
  (bf16, behind an RMSNorm or not) quantised in the call, W held quantised, and the
  projection's epilogue (``out``): "f32", "bf16", "resid" (h + y) or "swiglu" (W is gate | up);
- ``sample`` (``kernel_optim_amd.kernels.sampling``): one token for each row of logits by
  temperature, top-k, top-p and min-p from given random numbers, with its log-probability.

A block's scale is the least power of two s >= 2^-127 with max |x| <= 448 s; its codes are x / s
rounded to e4m3 (to nearest, ties to even). Sampling orders a row's tokens by falling logit
(ties: the lowest index first). Each filter keeps a beginning of that order: top-k the first k
tokens; top-p those with less than p of the (top-k) mass before them; min-p those of at least
min_p times the largest probability. The first token is always kept, and of the kept ones that
is drawn in which u times their mass falls. Temperature 0 takes the first token.

The plain form computes in 32 bits (sampling in 64: a draw lies next to a border) and rounds
where the framework's bf16 chain does. ``exact`` computes in 64 bits with a rounding to e4m3 of
its own.
"""

import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
EPS = 1e-6
MOST = 2 * 8192 * 19456 * 2560   # operations of the largest listed projection


def listed():
    return [
        # a prompt's activations behind the MLP's norm
        dict(name="quant_prompt_norm", kind="quant", rows=8192, K=2560, norm=True, dtype="bf16"),
        # a weight of odd sizes, quantised at load
        dict(name="quant_weight_odd", kind="quant", rows=4099, K=9736, norm=False, dtype="bf16"),
        # one sequence's attention output projection: launch and call latency
        dict(name="lin_b1_o", kind="linear", M=1, N=2560, K=4096, norm=False, out="resid"),
        # a batch's MLP input, gate and up in one pass
        dict(name="lin_b16_gateup", kind="linear", M=16, N=9728, K=2560, norm=True, out="swiglu"),
        # the LM head of a small batch: memory speed
        dict(name="lin_b4_lm_head", kind="linear", M=4, N=151936, K=2560, norm=True, out="bf16"),
        # a full decode batch's MLP output
        dict(name="lin_b64_down", kind="linear", M=64, N=2560, K=9728, norm=False, out="resid"),
        # a short prompt's attention input, odd length
        dict(name="lin_prompt_511_qkv", kind="linear", M=511, N=6144, K=2560, norm=True,
             out="bf16"),
        # a batch of prompts through the MLP input: matrix speed
        dict(name="lin_prompt_8192_gateup", kind="linear", M=8192, N=9728, K=2560, norm=True,
             out="swiglu"),
        # one sequence with a chat model's usual settings: latency
        dict(name="sample_b1_topk", kind="sample", B=1, V=151936, dtype="bf16", rows="same",
             temperature=0.7, top_k=50, top_p=0.9, min_p=0.0),
        # a server's batch, every sequence with settings of its own
        dict(name="sample_b64_mixed", kind="sample", B=64, V=151936, dtype="bf16", rows="mixed",
             temperature=1.0, top_k=0, top_p=1.0, min_p=0.0),
        # nucleus sampling over a whole fp32 vocabulary
        dict(name="sample_b16_nucleus_f32", kind="sample", B=16, V=151936, dtype="f32",
             rows="same", temperature=1.0, top_k=0, top_p=0.95, min_p=0.0),
        # many rollouts of a smaller, odd vocabulary
        dict(name="sample_b256_minp", kind="sample", B=256, V=32003, dtype="bf16", rows="same",
             temperature=1.3, top_k=0, top_p=1.0, min_p=0.05),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("quant", "linear", "linear", "linear", "sample", "sample"))
    if kind == "quant":
        K = 8 * _log_int(rng, 1, 2048)
        dtype = rng.choice(("bf16", "bf16", "f32"))
        return dict(kind=kind, K=K, rows=_log_int(rng, 1, max(1, min(16384, 4099 * 9736 // K))),
                    norm=dtype == "bf16" and K <= 8192 and rng.random() < 0.5, dtype=dtype)
    if kind == "linear":
        out = rng.choice(("f32", "bf16", "resid", "swiglu"))
        K = rng.choice((2560, 4096, 9728, 8 * _log_int(rng, 8, 1216)))
        N = rng.choice((_log_int(rng, 16, 19456), 16 * _log_int(rng, 1, 1216)))
        M = rng.choice((_log_int(rng, 1, 64), _log_int(rng, 1, 8192)))
        M = max(1, min(M, MOST // (2 * N * K * (2 if out == "swiglu" else 1))))
        return dict(kind=kind, M=M, N=N, K=K, norm=K <= 8192 and rng.random() < 0.5, out=out)
    V = rng.choice((151936, _log_int(rng, 2, 200000)))
    return dict(kind=kind, V=V, B=_log_int(rng, 1, max(1, min(512, 64 * 151936 // V))),
                dtype=rng.choice(("bf16", "bf16", "f32")), rows=rng.choice(("same", "mixed")),
                temperature=rng.choice((0.0, 0.2, 0.7, 1.0, 1.0, 1.7)),
                top_k=rng.choice((0, 0, 1, 20, 50, _log_int(rng, 1, V))),
                top_p=rng.choice((1.0, 0.95, 0.8, rng.uniform(0.01, 1.0))),
                min_p=rng.choice((0.0, 0.0, 0.05, rng.uniform(0.0, 1.0))))


# ---------------------------------------------------------------------------
# The plain form.
# ---------------------------------------------------------------------------
def _pow2(e):
    """2^e in fp32 for whole e in -127 .. 127."""
    return torch.where(e < -126, (1 << 22) + 0 * e, (e + 127) << 23).to(torch.int32).view(F32)


def _quantise(x):
    """x [rows, K] fp32 -> e4m3 codes [rows, blocks, 128] and scales [rows, blocks, 1] fp32."""
    g = torch.nn.functional.pad(x, (0, -x.shape[1] % 128)).unflatten(1, (-1, 128))
    m, e = torch.frexp(g.abs().amax(-1, keepdim=True))     # 448 = 0.875 * 2^9
    e = torch.where(m == 0, -127, e - 9 + (m > 0.875).int()).clamp_min(-127)
    return (g * _pow2(-e)).to(torch.float8_e4m3fn), _pow2(e)


def _values(codes, scales, K):
    return (codes.float() * scales).flatten(1)[:, :K]


def _norm(x, w):
    """RMSNorm as the framework's bf16 chain has it: rounded before and behind the gain."""
    x = x.float()
    t = (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)).to(BF16)
    return (w.float() * t.float()).to(BF16).float()


def _linear(s):
    case = s["case"]
    x = _norm(s["x"], s["nw"]) if case["norm"] else s["x"].float()
    K, N = case["K"], case["N"]
    y = _values(*_quantise(x), K) @ _values(s["codes"], s["scales"], K).t()
    if case["out"] == "f32":
        return y
    y = y.to(BF16)
    if case["out"] == "resid":
        return (s["h"].float() + y.float()).to(BF16)
    if case["out"] == "swiglu":
        g, u = y[:, :N].float(), y[:, N:].float()
        return ((g / (1 + torch.exp(-g))).to(BF16).float() * u).to(BF16)
    return y


def _column(v, B):
    return (v if isinstance(v, torch.Tensor) else torch.full((B,), v, device=DEV))[:, None]


def _sample(s):
    x = s["logits"].double()
    B, V = x.shape
    t, k, p, mp = (_column(s[n], B) for n in ("temperature", "top_k", "top_p", "min_p"))
    t, p, mp = t.float().double(), p.float().double(), mp.float().double()
    x, order = torch.sort(x, dim=-1, descending=True, stable=True)
    z = (x - x[:, :1]) / torch.where(t > 0, t, 1.0)
    w = torch.exp(z)
    mass = w.cumsum(-1)
    rank = torch.arange(V, device=DEV)[None]
    k = torch.where(k > 0, k, V).clamp(max=V).long()
    kept = (rank < k) & ((p >= 1) | (mass - w < p * mass.gather(1, k - 1))) & (w >= mp)
    last = (kept.sum(-1, keepdim=True) - 1).clamp_min(0)
    last = torch.where(t > 0, last, 0)
    total = mass.gather(1, last)
    at = (mass <= s["u"].double()[:, None] * total).sum(-1, keepdim=True).minimum(last)
    logp = torch.where(t > 0, z.gather(1, at) - torch.log(total), 0.0)
    return order.gather(1, at)[:, 0], logp[:, 0].float()


def _plain(s):
    case = s["case"]
    if case["kind"] == "linear":
        return _linear(s)
    if case["kind"] == "sample":
        return _sample(s)
    x = _norm(s["x"], s["nw"]) if case["norm"] else s["x"].float()
    return _values(*_quantise(x), case["K"]).to(s["x"].dtype)


# ---------------------------------------------------------------------------
# Inputs.
# ---------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _activations(rows, K, g):
    """Rows as a residual stream has them: a few channels and values far above the others."""
    x = torch.randn(rows, K, device=DEV, generator=g)
    x *= 1 + 12 * (torch.rand(K, device=DEV, generator=g) < 0.004).float()
    return x * (0.5 + torch.rand(rows, 1, device=DEV, generator=g))


def _inputs(case, seed):
    g = _gen(seed)
    if case["kind"] == "sample":
        B, V = case["B"], case["V"]
        x = 2.5 * torch.randn(B, V, device=DEV, generator=g)
        # the next word's few likely tokens, in some rows well above the rest
        top = torch.randint(0, V, (B, 40), device=DEV, generator=g)
        lift = 9 * torch.rand(B, 40, device=DEV, generator=g)
        x.scatter_add_(1, top, lift * torch.rand(B, 1, device=DEV, generator=g))
        s = dict(logits=x.to(BF16 if case["dtype"] == "bf16" else F32),
                 u=torch.rand(B, device=DEV, generator=g))
        names = ("temperature", "top_k", "top_p", "min_p")
        if case["rows"] == "same":
            return dict(s, **{n: case[n] for n in names})

        def some(values, dtype):
            v = torch.tensor(values, device=DEV, dtype=dtype)
            return v[torch.randint(0, len(values), (B,), device=DEV, generator=g)]

        return dict(s, temperature=some((0.0, 0.3, 0.6, 0.7, 1.0, 1.0, 1.4), F32),
                    top_k=some((0, 0, 1, 20, 50, 1000), torch.int32),
                    top_p=some((1.0, 1.0, 0.95, 0.8, 0.3), F32),
                    min_p=some((0.0, 0.0, 0.02, 0.1), F32))
    K = case["K"]
    rows = case["rows"] if case["kind"] == "quant" else case["M"]
    x = _activations(rows, K, g)
    s = dict(x=x.to(F32 if case.get("dtype") == "f32" else BF16))
    if case["norm"]:
        s["nw"] = (1 + 0.2 * torch.randn(K, device=DEV, generator=g)).to(BF16)
    if case["kind"] == "linear":
        N = case["N"]
        s["w"] = (0.02 * torch.randn((2 if case["out"] == "swiglu" else 1) * N, K, device=DEV,
                                     generator=g)).to(BF16)
        if case["out"] == "resid":
            s["h"] = torch.randn(rows, N, device=DEV, generator=g).to(BF16)
    return s


def prepare(case, seed):
    s = dict(_inputs(case, seed), case=case)
    kind = case["kind"]
    if kind == "linear":
        w = s.pop("w")
        if not own:
            s["codes"], s["scales"] = _quantise(w.float())
            return s
        from kernel_optim_amd.kernels import fp8
        from kernel_optim_amd.kernels.gemv import EPI_BF16, EPI_F32, EPI_RESID, EPI_SWIGLU
        epi = dict(f32=EPI_F32, bf16=EPI_BF16, resid=EPI_RESID, swiglu=EPI_SWIGLU)[case["out"]]
        s["w"] = fp8.fp8_quantize(w, pair=case["out"] == "swiglu")
        s["op"] = fp8.Fp8Linear(case["M"], case["N"], case["K"], epi, case["norm"], eps=EPS)
        s["y"] = torch.empty(case["M"], case["N"], device=DEV,
                             dtype=F32 if case["out"] == "f32" else BF16)
    elif own and kind == "quant":
        from kernel_optim_amd.kernels import fp8
        s["op"] = fp8
        s["held"] = fp8.fp8_empty(case["rows"], case["K"], DEV)
        s["y"] = torch.empty_like(s["x"])
    elif own:
        from kernel_optim_amd.kernels.sampling import Sampler
        s["op"] = Sampler(case["B"], case["V"], DEV)
        s["ids"] = torch.empty(case["B"], dtype=torch.int64, device=DEV)
        s["logp"] = torch.empty(case["B"], dtype=F32, device=DEV)
    return s


def run(s):
    if not own:
        return _plain(s)
    kind = s["case"]["kind"]
    if kind == "linear":
        s["op"](s["x"], s["w"], y=s["y"], nw=s.get("nw"), h=s.get("h"))
        return s["y"]
    if kind == "quant":
        s["op"].fp8_quantize(s["x"], out=s["held"], nw=s.get("nw"), eps=EPS)
        s["op"].fp8_read(s["held"], s["y"])
        return s["y"]
    s["op"](s["logits"], s["u"], s["ids"], temperature=s["temperature"], top_k=s["top_k"],
            top_p=s["top_p"], min_p=s["min_p"], logprobs=s["logp"])
    return s["ids"], s["logp"]


# ---------------------------------------------------------------------------
# In 64 bits.
# ---------------------------------------------------------------------------
def _held64(x):
    """What 8 bits hold of x [rows, K] fp64, as fp64 values: the scale by comparing with
    448 times each power of two, the code by rounding to a multiple of its binade's step."""
    rows, K = x.shape
    out = torch.empty_like(x)
    for k in range(0, K, 128):
        b = x[:, k:k + 128]
        top = b.abs().amax(1, keepdim=True)
        e = torch.floor(torch.log2(top.clamp_min(2.0 ** -400))).clamp(-140, 128) - 8
        two = lambda n: ((n.long() + 1023) << 52).view(F64)
        e = torch.where(top > 448 * two(e), e + 1, e)
        e = torch.where(top <= 448 * two(e - 1), e - 1, e).clamp_min(-127)
        v = b / two(e)
        binade = torch.frexp(v)[1] - 1                 # 2^binade <= |v| < 2^(binade + 1)
        step = two(torch.where(v == 0, -6, binade).clamp_min(-6) - 3)
        out[:, k:k + 128] = torch.round(v / step) * step * two(e)
    return out


def _norm64(x, w):
    t = (x.double() / torch.sqrt(x.double().square().mean(-1, keepdim=True) + EPS)).to(BF16)
    return (w.double() * t.double()).to(BF16).double()


def _sample64(case, seed):
    s = {n: v.cpu().double().numpy() if isinstance(v, torch.Tensor) else v
         for n, v in _inputs(case, seed).items()}
    B, V = case["B"], case["V"]
    ids, logp = np.zeros(B, dtype=np.int64), np.zeros(B)
    at = lambda n, b: float(np.float32(s[n][b] if isinstance(s[n], np.ndarray) else s[n]))
    for b in range(B):
        x = s["logits"][b]
        t, k, p, mp = (at(n, b) for n in ("temperature", "top_k", "top_p", "min_p"))
        if t <= 0:
            ids[b] = int(np.argmax(x))
            continue
        order = np.argsort(-x, kind="stable")
        if 0 < k < V:
            order = order[:int(k)]
        z = (x[order] - x[order[0]]) / t
        w = np.exp(z)
        c = np.cumsum(w)
        n = len(w)
        if p < 1:
            n = min(n, int(np.searchsorted(c, p * c[-1], side="left")) + 1)
        if mp > 0:
            n = min(n, max(1, int(np.searchsorted(-w, -mp, side="right"))))
        i = min(int(np.searchsorted(c[:n], s["u"][b] * c[n - 1], side="right")), n - 1)
        ids[b] = order[i]
        logp[b] = z[i] - math.log(c[n - 1])
    return torch.from_numpy(ids), torch.from_numpy(logp)


def exact(case, seed):
    if case["kind"] == "sample":
        return _sample64(case, seed)
    s = _inputs(case, seed)
    x = _held64(_norm64(s["x"], s["nw"]) if case["norm"] else s["x"].double())
    if case["kind"] == "quant":
        return x
    w, N = s["w"], case["N"]
    y = torch.cat([x @ _held64(w[i:i + 16384].double()).t() for i in range(0, len(w), 16384)], 1)
    if case["out"] == "resid":
        return s["h"].double() + y
    if case["out"] == "swiglu":
        return y[:, :N] / (1 + torch.exp(-y[:, :N])) * y[:, N:]
    return y


def work(case):
    if case["kind"] == "sample":
        n = case["B"] * case["V"]
        return {"bytes": n * (2 if case["dtype"] == "bf16" else 4) + 32 * case["B"],
                "flops": 4 * n}   # a difference, a scaling, an exp and a sum for each token
    K, blocks = case["K"], -(-case["K"] // 128)
    if case["kind"] == "quant":
        rows, size = case["rows"], 2 if case["dtype"] == "bf16" else 4
        return {"bytes": rows * (2 * size * K + K + blocks), "flops": 3 * rows * K}
    M, N = case["M"], case["N"]
    wide = N * (2 if case["out"] == "swiglu" else 1)
    outs = M * N * dict(f32=4, bf16=2, resid=4, swiglu=2)[case["out"]]
    return {"bytes": 2 * M * K + wide * (K + blocks) + outs, "flops": 2 * M * wide * K}
