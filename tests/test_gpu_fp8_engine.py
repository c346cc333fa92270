"""GPU: the engine on 8-bit weights against the eager replay whose projections quantise both factors as
the oracle does. Drawn tokens are the Sampler's on the step's own logits.

Tolerance. Two evaluations that round differently differ by some d of a value (bf16: up to 2^-8) in
front of a quantiser whose step is s of it (e4m3: 2^-4 to 2^-3): a code then flips with probability d / s
and by s, so behind it they differ by sqrt(d s) in the mean square, where bf16 projections pass d
on: sqrt(s / d), 4 to 6 times as much. The bf16 tests' limit of 0.25 logits is no bound of that.
What is: the replay against itself with attention's probabilities rounded to bf16 in front of their
product with V, as the engine's attention kernels (tested by themselves) round them, by the
factor that the bf16 engine's full-depth test allows over its own such noise."""

from types import SimpleNamespace

import pytest
import torch
import torch.nn.functional as F

import oracle.qwen3 as Q
from kernel_optim_amd.engine import Engine, Sampling
from kernel_optim_amd.kernels.sampling import Sampler
from kernel_optim_amd.model import Qwen3Config, fp8_weights, random_weights, weights_to
from oracle import fp8 as O
from tests.test_gpu_engine import (FULL_NOISE_FACTOR, FULL_NOISE_SLACK, check_against_replay)
from tests.test_oracle_qwen3 import SMALL, perturbed_weights

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def prompts(cfg, B, S, seed=6):
    return torch.randint(0, cfg.vocab, (B, S), generator=torch.Generator().manual_seed(seed))


def replay(monkeypatch, cfg, w, prompt, toks, cap, round_p):
    """The eager replay with projections over what 8 bits hold of x and w."""
    held = {}

    def linear(x, w):
        key = (w.data_ptr(), tuple(w.shape))
        if key not in held:
            held[key] = O.held(w).float()
        y = O.held(x.reshape(-1, x.shape[-1])).float() @ held[key].t()
        return y.to(BF16).view(*x.shape[:-1], -1)

    soft = torch.softmax
    monkeypatch.setattr(Q, "F", SimpleNamespace(linear=linear, embedding=F.embedding, silu=F.silu))
    if round_p:
        monkeypatch.setattr(torch, "softmax", lambda s, dim: soft(s, dim=dim).to(BF16).float())
    out = Q.Qwen3Oracle(cfg, w, B=len(toks), cap=cap).teacher_forced(prompt, toks).float()
    monkeypatch.undo()
    return out


def check(monkeypatch, cfg, w, prompt, toks, logits, cap):
    a, b = (replay(monkeypatch, cfg, w, prompt, toks, cap, p) for p in (False, True))
    noise = (a - b).abs().max().item()
    _, err = check_against_replay(toks, logits, a)
    assert err <= FULL_NOISE_FACTOR * noise + FULL_NOISE_SLACK, (err, noise)


@pytest.mark.parametrize("B", [1, 3, 20])
def test_decode(dev, monkeypatch, B):
    cfg, n = SMALL, 24
    w = perturbed_weights(cfg, seed=5)
    prompt = prompts(cfg, B, 29)
    eng = Engine.from_weights(cfg, w, keep_logits=True, weight_format="fp8")
    toks, logits = eng.trace(prompt.tolist(), n)
    assert eng.step_kind == "fp8"
    check(monkeypatch, cfg, w, prompt, toks, logits, 64)
    for _ in range(2):   # generate() yields the same tokens, twice
        assert torch.equal(torch.tensor(list(eng.generate(prompt.tolist(), n))).T, toks)


def test_two_layers_at_full_width(dev, monkeypatch):
    cfg, n = Qwen3Config(layers=2, vocab=2000), 5
    w = random_weights(cfg, seed=2)
    prompt = prompts(cfg, 1, 70)
    eng = Engine.from_weights(cfg, w, keep_logits=True, weight_format="fp8")
    toks, logits = eng.trace(prompt.tolist(), n)
    check(monkeypatch, cfg, w, prompt, toks, logits, 80)


@pytest.mark.parametrize("S", [1, 2, 9])
def test_short_prompts(dev, monkeypatch, S):
    cfg, n = SMALL, 4
    w = perturbed_weights(cfg, seed=5)
    prompt = prompts(cfg, 2, S)
    toks, logits = Engine.from_weights(cfg, w, keep_logits=True, weight_format="fp8").trace(
        prompt.tolist(), n)
    check(monkeypatch, cfg, w, prompt, toks, logits, 16)


def test_weights_are_held_in_8_bits(dev):
    cfg = SMALL
    w = weights_to(perturbed_weights(cfg, seed=5), dev)
    h = fp8_weights(w)
    full = sum(l[k].numel() for l in w["layers"] for k in ("qkv", "o", "gu", "down"))
    assert sum(l[k].nbytes for l in h["layers"] for k in ("qkv", "o", "gu", "down")) <= 1.02 * full
    assert h["embed"] is w["embed"] and h["layers"][0]["w_in"] is w["layers"][0]["w_in"]
    assert w["layers"][0]["qkv"].dtype == BF16   # the caller's stay as they are


@pytest.mark.parametrize("B", [1, 3])
def test_with_the_4_bit_cache_and_speculation(dev, B):
    """Both run, and speculation yields the tokens of the one-token steps but for near-ties: here the
    repeated prompt makes drafts that are taken."""
    cfg, n = SMALL, 16
    w = perturbed_weights(cfg, seed=5)
    prompt = [(p * 4)[:30] for p in prompts(cfg, B, 8).tolist()]
    for kv in ("bf16", "kv4"):
        plain = Engine.from_weights(cfg, w, weight_format="fp8", kv_cache=kv)
        spec = Engine.from_weights(cfg, w, weight_format="fp8", kv_cache=kv, spec=True)
        a, b = list(plain.generate(prompt, n)), list(spec.generate(prompt, n))
        assert len(a) == len(b) == n and spec.spec_steps > 0
        assert a[0] == b[0]


@pytest.mark.parametrize("kw", [dict(weight_format="fp8"), dict(decode_graph="fused"),
                                dict(decode_graph="hipblaslt"), dict(kv_cache="kv4")])
def test_drawn_tokens(dev, kw):
    """generate() draws what Sampler draws from the step's logits with the same numbers."""
    cfg, B, n = SMALL, 3, 10
    w = perturbed_weights(cfg, seed=5)
    prompt = prompts(cfg, B, 21).tolist()
    eng = Engine.from_weights(cfg, w, keep_logits=True, **kw)
    s = Sampling(temperature=[0.8, 1.2, 0.0], top_k=[0, 20, 0], top_p=0.9, min_p=[0.0, 0.01, 0.0],
                 seed=3)
    numbers = torch.rand(n, B, generator=torch.Generator().manual_seed(3)).to(dev)
    columns = [c.to(dev) for c in s.columns(B)]
    draw, ids = Sampler(B, cfg.vocab, dev), torch.empty(B, dtype=torch.int64, device=dev)
    got = list(eng.generate(prompt, n, sampling=s))
    assert got == list(eng.generate(prompt, n, sampling=s))
    with torch.inference_mode():   # step by step, from the engine's own logits
        for t, v in zip(eng.settings, columns):
            t.copy_(v)
        eng.u.copy_(numbers[0])
        eng._prefill(torch.tensor(prompt, device=dev))
        for j in range(n):
            if j:
                eng.u.copy_(numbers[j])
                eng.step()
            draw(eng.logits, numbers[j], ids, *columns)
            torch.cuda.synchronize()
            assert ids.tolist() == eng.ids.tolist() == got[j]
    assert len({tuple(r) for r in got}) > 1


def test_drawing_greedily_is_greedy(dev):
    cfg, n = SMALL, 12
    eng = Engine.from_weights(cfg, perturbed_weights(cfg, seed=5), weight_format="fp8")
    prompt = prompts(cfg, 2, 17).tolist()
    greedy = list(eng.generate(prompt, n))
    assert list(eng.generate(prompt, n, sampling=Sampling(temperature=0.0))) == greedy
    assert list(eng.generate(prompt, n, sampling=Sampling(top_k=1, seed=9))) == greedy
    assert list(eng.generate(prompt, n)) == greedy
    a = list(eng.generate(prompt, n, sampling=Sampling(temperature=1.5, seed=1)))
    assert a != list(eng.generate(prompt, n, sampling=Sampling(temperature=1.5, seed=2)))


def test_refusals(dev):
    cfg = SMALL
    w = perturbed_weights(cfg, seed=5)
    with pytest.raises(ValueError):
        Engine.from_weights(cfg, w, weight_format="int8")
    with pytest.raises(ValueError):
        Engine.from_weights(cfg, w, weight_format="fp8", decode_graph="fused")
    eng = Engine.from_weights(cfg, w, weight_format="fp8")
    for bad in (Sampling(temperature=-1.0), Sampling(top_k=-1), Sampling(top_p=1.5), Sampling(min_p=-0.1),
                Sampling(temperature=[1.0, 1.0]), Sampling(top_k=0.5), Sampling(top_p=float("nan"))):
        with pytest.raises(ValueError):
            list(eng.generate([[1, 2, 3]], 2, sampling=bad))
