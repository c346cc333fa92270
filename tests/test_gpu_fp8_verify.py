"""GPU: the verify step on 8-bit weights, and 8-bit weights with the 4-bit cache, against the eager
replay whose projections quantise both factors as the oracle does.

The tolerance is that of test_gpu_fp8_engine.py: the replay against itself with attention's
probabilities rounded to bf16, by the bf16 engine's factor over its own such noise. The 4-bit
cache's attention rounds the products of its probabilities and scales instead, by as much."""

from types import SimpleNamespace

import pytest
import torch
import torch.nn.functional as F

import oracle.qwen3 as Q
from kernel_optim_amd.engine import Engine
from oracle import fp8 as O
from oracle.ops import argmax_first
from tests.test_gpu_engine import FULL_NOISE_FACTOR, FULL_NOISE_SLACK, check_against_replay
from tests.test_gpu_fp8_engine import prompts, replay
from tests.test_gpu_kv4_engine import replay_over
from tests.test_oracle_qwen3 import SMALL, perturbed_weights

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def limit(noise):
    return FULL_NOISE_FACTOR * noise + FULL_NOISE_SLACK


def replay_over_cache(monkeypatch, eng, w, run, round_p):
    """run(oracle) over the engine's 4-bit cache, projections over what 8 bits hold of x and w."""
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
    return replay_over(eng, w, monkeypatch, run).float()


def check_verify(vout, logits, want, noise):
    """Ids and logits of a verify step against the replay's logits [B, T, V] of its rows: logits
    within the limit, ids the first maxima of the step's own."""
    got = logits.view_as(want).float()
    err = (got - want).abs().max().item()
    assert err <= limit(noise), (err, noise)
    assert torch.equal(vout, argmax_first(logits).view(vout.shape))
    chosen = want.gather(2, vout[..., None])[..., 0]
    assert (want.max(-1).values - chosen <= 2 * err + 1e-6).all()


@pytest.mark.parametrize("B", [1, 3, 4, 8, 16])
def test_verify_step(dev, monkeypatch, B):
    """7, 21, 28, 40 and 80 rows: every kind of product. The rows are those that the one-token steps
    decoded, at the third generated position."""
    cfg, S, n = SMALL, 29, 12
    w = perturbed_weights(cfg, seed=41)
    prompt = prompts(cfg, B, S, 42)
    eng = Engine.from_weights(cfg, w, keep_logits=True, spec=True, weight_format="fp8")
    toks, _ = eng.trace(prompt.tolist(), n)
    T, j = eng.T, 2
    at = S - 1 + j
    rows = torch.cat((prompt, toks), 1)[:, at:at + T]
    vout, logits = eng.verify_step(rows, torch.full((B,), at))
    a, b = (replay(monkeypatch, cfg, w, prompt, toks, S + n, p) for p in (False, True))
    check_verify(vout, logits, a[:, j:j + T], (a - b).abs().max().item())


@pytest.mark.parametrize("B", [1, 3])
def test_the_4_bit_cache(dev, monkeypatch, B):
    """One-token steps and a verify step of drafts that nothing decoded."""
    cfg, S, n = SMALL, 20, 24
    w = perturbed_weights(cfg, seed=43)
    prompt = prompts(cfg, B, S, 44)
    eng = Engine.from_weights(cfg, w, keep_logits=True, spec=True, weight_format="fp8", kv_cache="kv4")
    toks, logits = eng.trace(prompt.tolist(), n)
    a, b = (replay_over_cache(monkeypatch, eng, w, lambda o: o.teacher_forced_decode(prompt, toks), p)
            for p in (False, True))
    noise = (a - b).abs().max().item()
    _, err = check_against_replay(toks, logits, a)
    assert err <= limit(noise), (err, noise)

    start = S + 8
    drafts = torch.randint(0, cfg.vocab, (B, eng.K), generator=torch.Generator().manual_seed(45))
    rows = torch.cat((toks[:, 8:9], drafts), 1)
    vout, logits = eng.verify_step(rows, torch.full((B,), start))

    def run(o):
        o.forward(prompt, 0)
        return o.forward(rows, start)

    a, b = (replay_over_cache(monkeypatch, eng, w, run, p) for p in (False, True))
    check_verify(vout, logits, a, max(noise, (a - b).abs().max().item()))


@pytest.mark.parametrize("B", [1, 3, 8])
def test_speculation_yields_the_same_tokens(dev, monkeypatch, B):
    """As the one-token steps', but for near-ties: where a sequence first differs, both steps have
    read the same tokens, each is within the limit of the replay, and either token is its own
    step's maximum, so that the one-token step's logits of the two are within four limits."""
    cfg, n = SMALL, 24
    w = perturbed_weights(cfg, seed=46)
    prompt = torch.tensor([(p * 4)[:30] for p in prompts(cfg, B, 8, 47).tolist()])
    plain = Engine.from_weights(cfg, w, keep_logits=True, weight_format="fp8")
    toks, logits = plain.trace(prompt.tolist(), n)
    a, b = (replay(monkeypatch, cfg, w, prompt, toks, 30 + n, p) for p in (False, True))
    most = 4 * limit((a - b).abs().max().item())
    spec = Engine.from_weights(cfg, w, weight_format="fp8", spec=True)
    spec.min_advance = 0.0   # verify steps to the end
    got = torch.tensor(list(spec.generate(prompt.tolist(), n))).T
    assert got.shape == toks.shape and spec.spec_steps > 0
    for s in range(B):
        off = (got[s] != toks[s]).nonzero()
        if len(off):
            row = logits[int(off[0])][s].float()
            assert row[toks[s, off[0]]] - row[got[s, off[0]]] <= most
