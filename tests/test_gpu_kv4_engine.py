"""GPU: the decode engine over a 4-bit KV cache. The eager replay attends to what the engine's own
cache holds (its own prompt attention is bf16, as the engine's), so what is left between
the two is the rounding that the bf16 engine's tests bound: their limits hold here."""

import pytest
import torch

import oracle.qwen3 as Q
from kernel_optim_amd.engine import Engine
from kernel_optim_amd.model import Qwen3Config, random_weights
from oracle import kv4 as O
from tests.test_gpu_engine import LOGIT_ATOL, check_against_replay
from tests.test_oracle_qwen3 import SMALL, perturbed_weights

pytestmark = pytest.mark.gpu


def held(eng, layer, group=32):
    n, s, c = O.unpack(eng.kv4[layer], eng.cfg.head_dim, group)
    return O.values(n, s, c, group, torch.float32)   # [2, B, nkv, slots, d]


def replay_over(eng, w, monkeypatch, run):
    """run(oracle) with the attention of every step behind the prompt reading the engine's cache."""
    cfg, L = eng.cfg, eng.cfg.layers
    kept = [held(eng, i) for i in range(L)]
    plain, calls = Q.attention_fp32, [0]

    def attention(q, k, v, start, scale):
        layer = calls[0] % L
        calls[0] += 1
        if start == 0:
            return plain(q, k, v, start, scale)
        k, v = kept[layer][:, :, :, :start + q.shape[2]]
        return plain(q, k, v, start, scale)

    monkeypatch.setattr(Q, "attention_fp32", attention)
    out = run(Q.Qwen3Oracle(cfg, w, B=eng.B, cap=eng.cap))
    monkeypatch.undo()
    return out


@pytest.mark.parametrize("graph,B", [("fused", 1), ("fused", 3), ("hipblaslt", 2)])
def test_decode(dev, monkeypatch, graph, B):
    cfg, n = SMALL, 40
    w = perturbed_weights(cfg, seed=5)
    prompt = torch.randint(0, cfg.vocab, (B, 29), generator=torch.Generator().manual_seed(6))
    eng = Engine.from_weights(cfg, w, keep_logits=True, decode_graph=graph, kv_cache="kv4")
    toks, logits = eng.trace(prompt.tolist(), n)
    assert eng.step_kind == graph and eng.k_cache is None
    replay = replay_over(eng, w, monkeypatch, lambda o: o.teacher_forced_decode(prompt, toks))
    _, err = check_against_replay(toks, logits, replay)
    assert err < LOGIT_ATOL
    # generate() yields the same tokens, twice
    for _ in range(2):
        assert torch.equal(torch.tensor(list(eng.generate(prompt.tolist(), n))).T, toks)


def test_two_layers_at_full_width(dev, monkeypatch):
    cfg, n = Qwen3Config(layers=2), 8
    w = random_weights(cfg, seed=7)
    prompt = torch.randint(0, cfg.vocab, (2, 50), generator=torch.Generator().manual_seed(8))
    eng = Engine.from_weights(cfg, w, keep_logits=True, kv_cache="kv4")
    toks, logits = eng.trace(prompt.tolist(), n)
    replay = replay_over(eng, w, monkeypatch, lambda o: o.teacher_forced_decode(prompt, toks))
    _, err = check_against_replay(toks, logits, replay)
    assert err < LOGIT_ATOL


def test_the_prompt_is_quantised_from_bf16(dev):
    cfg = SMALL
    w = perturbed_weights(cfg, seed=9)
    prompt = torch.randint(0, cfg.vocab, (2, 45), generator=torch.Generator().manual_seed(10)).tolist()
    full, eng = (Engine.from_weights(cfg, w, kv_cache=k) for k in ("bf16", "kv4"))
    assert list(full.generate(prompt, 1)) == list(eng.generate(prompt, 1))   # a bf16 prompt pass
    k, v = (c[0, :, :, :45].cpu() for c in (full.k_cache, full.v_cache))
    n, s, c = O.unpack(eng.kv4[0], cfg.head_dim, 32)
    for i, x in enumerate((k, v)):
        for got, want in zip((n, s, c), O.quantise(x, 32)):
            assert torch.equal(got[i][:, :, :45], want)


def test_verify_step(dev, monkeypatch):
    """Speculation's verify step: B * (K + 1) rows appended and attended at each sequence's own
    position, and speculative decoding to the end."""
    cfg, S, n = SMALL, 20, 24
    w = perturbed_weights(cfg, seed=11)
    prompt = torch.randint(0, cfg.vocab, (2, S), generator=torch.Generator().manual_seed(12))
    eng = Engine.from_weights(cfg, w, keep_logits=True, spec=True, kv_cache="kv4")
    toks, _ = eng.trace(prompt.tolist(), n)
    rows = torch.cat((toks[:, 8:9], torch.randint(0, cfg.vocab, (2, eng.K))), 1)
    start = S + 8
    got, logits = eng.verify_step(rows, torch.tensor([start, start]))

    def run(o):
        # every position in front of the step, then the step's rows in one forward
        o.forward(prompt, 0)
        return o.forward(rows, start)

    want = replay_over(eng, w, monkeypatch, run).float()
    diff = (logits.view_as(want).float() - want).abs().max()
    assert diff < LOGIT_ATOL
    chosen = want.gather(2, got[:, :, None])[..., 0]
    assert (want.max(-1).values - chosen <= 2 * diff + 1e-6).all()
    assert len(list(eng.generate(prompt.tolist(), n))) == n


def test_refusals(monkeypatch):
    cfg = SMALL
    w = perturbed_weights(cfg, seed=1)
    with pytest.raises(ValueError):
        Engine.from_weights(cfg, w, kv_cache="int8")
    monkeypatch.setattr("kernel_optim_amd.engine.KV_GROUP", 48)
    with pytest.raises(ValueError):
        Engine.from_weights(cfg, w, kv_cache="kv4")
