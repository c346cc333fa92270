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


# ---------------------------------------------------------------------------
# What the engine puts into its cache. The replays above read it in place of the oracle's own K and
# V, so they agree whatever it holds.
# ---------------------------------------------------------------------------
def check_rows(eng, layer, which, got, want, step):
    """Cached rows against the oracle's bf16 ones, in 2-norm over a layer and forward. The quantiser is
    off by step / sqrt(12) a value (even in [-s/2, s/2]); 1.25 of that lies 4 deviations out for the
    256 values of the smallest rows. Beside it the two ways to the row, some 13 bf16 roundings each
    (two layers of norms, projections, residual adds, activation, RoPE), of at most 2^-8 / sqrt(3) =
    0.0023 in 2-norm: 0.0115 for all of them, and a factor of 4 for what gains and activations make
    of them. Rows of another slot, layer or weight are off by 0.2 (RoPE one position off) to 1.4."""
    rms = lambda x: x.double().square().mean().sqrt()
    limit = ((1.25 * rms(step) / 12 ** 0.5) ** 2 + (0.05 * rms(want)) ** 2).sqrt()
    err = rms(got.double() - want.double())
    assert err <= limit, f"layer {layer} {'KV'[which]}: {err / rms(want):.3f} of the rows"


def replay_and_check_rows(eng, w, monkeypatch, run):
    """replay_over, with every forward's own K and V, the prompt's included, against what the engine
    cached at those positions. Returns run's result and the forwards checked."""
    cfg, L, group = eng.cfg, eng.cfg.layers, eng.kv_group
    kept = [O.unpack(eng.kv4[i], cfg.head_dim, group) for i in range(L)]
    values = [O.values(n, s, c, group, torch.float32) for n, s, c in kept]
    plain, calls = Q.attention_fp32, [0]

    def attention(q, k, v, start, scale):
        layer = calls[0] % L
        calls[0] += 1
        new = slice(start, start + q.shape[2])
        for which, x in enumerate((k, v)):
            check_rows(eng, layer, which, values[layer][which, :, :, new], x[:, :, new],
                       kept[layer][1][which, :, :, new])
        if start == 0:
            return plain(q, k, v, start, scale)
        k, v = values[layer][:, :, :, :start + q.shape[2]]
        return plain(q, k, v, start, scale)

    monkeypatch.setattr(Q, "attention_fp32", attention)
    out = run(Q.Qwen3Oracle(cfg, w, B=eng.B, cap=eng.cap))
    monkeypatch.undo()
    assert calls[0] % L == 0
    return out, calls[0] // L


def check_last_layer(eng, qkv, at, T):
    """The last layer's appended slots against its own projection rows, which the step leaves: V to the
    bit, K within kv4_append's bound."""
    cfg, i, group = eng.cfg, eng.cfg.layers - 1, eng.kv_group
    nq, nkv, d, lw = cfg.nq, cfg.nkv, cfg.head_dim, eng.w["layers"][i]
    n, s, c = O.unpack(eng.kv4[i], d, group)
    x = qkv.cpu().view(eng.B, T, nq + 2 * nkv, d)
    for b in range(eng.B):
        for t in range(T):
            p = at + t
            for got, want in zip((n, s, c), O.quantise(x[b, t, nq + nkv:], group)):
                assert torch.equal(got[1, b, :, p], want)
            k = O.norm_rope(x[b, t, nq:nq + nkv], lw["k_norm"].cpu(), eng._cos[p].cpu(),
                            eng._sin[p].cpu(), cfg.eps)
            sk = O.quantise(k, group)[1].double().repeat_interleave(group, -1)
            got = O.values(n[0, b, :, p], s[0, b, :, p], c[0, b, :, p], group)
            # half a step of an s one bf16 step off, 8 s 2^-8 at the ends, fp32's norm and rotation
            assert ((got - k).abs() <= sk * (0.5 + 2.0 ** -7 + 2.0 ** -5 + 2.0 ** -10)).all()


@pytest.mark.parametrize("graph,B", [("fused", 1), ("fused", 3), ("hipblaslt", 2)])
def test_decode_caches_the_right_rows(dev, monkeypatch, graph, B):
    cfg, n, S = SMALL, 40, 29
    w = perturbed_weights(cfg, seed=25)
    prompt = torch.randint(0, cfg.vocab, (B, S), generator=torch.Generator().manual_seed(26))
    eng = Engine.from_weights(cfg, w, keep_logits=True, decode_graph=graph, kv_cache="kv4")
    toks, _ = eng.trace(prompt.tolist(), n)
    assert eng.step_kind == graph
    check_last_layer(eng, eng.qkv, S + n - 2, 1)
    _, forwards = replay_and_check_rows(eng, w, monkeypatch,
                                        lambda o: o.teacher_forced_decode(prompt, toks))
    assert forwards == n


def test_full_width_caches_the_right_rows(dev, monkeypatch):
    cfg, n = Qwen3Config(layers=2), 8
    w = random_weights(cfg, seed=27)
    prompt = torch.randint(0, cfg.vocab, (2, 50), generator=torch.Generator().manual_seed(28))
    eng = Engine.from_weights(cfg, w, keep_logits=True, kv_cache="kv4")
    toks, _ = eng.trace(prompt.tolist(), n)
    check_last_layer(eng, eng.qkv, 50 + n - 2, 1)
    _, forwards = replay_and_check_rows(eng, w, monkeypatch,
                                        lambda o: o.teacher_forced_decode(prompt, toks))
    assert forwards == n


@pytest.mark.parametrize("B", [1, 2])
def test_verify_caches_the_right_rows(dev, monkeypatch, B):
    cfg, S, n = SMALL, 20, 24
    w = perturbed_weights(cfg, seed=29)
    prompt = torch.randint(0, cfg.vocab, (B, S), generator=torch.Generator().manual_seed(30))
    eng = Engine.from_weights(cfg, w, keep_logits=True, spec=True, kv_cache="kv4")
    toks, _ = eng.trace(prompt.tolist(), n)
    rows = torch.cat((toks[:, 8:9], torch.randint(0, cfg.vocab, (B, eng.K))), 1)
    start = S + 8
    eng.verify_step(rows, torch.full((B,), start))
    check_last_layer(eng, eng.qkvT, start, eng.K + 1)

    def run(o):
        o.teacher_forced_decode(prompt, toks[:, :9])   # up to the position in front of the step
        return o.forward(rows, start)

    _, forwards = replay_and_check_rows(eng, w, monkeypatch, run)
    assert forwards == 10


def test_every_layer_of_the_prompt_is_quantised_from_bf16(dev):
    cfg, B, S = SMALL, 2, 45
    w = perturbed_weights(cfg, seed=31)
    prompt = torch.randint(0, cfg.vocab, (B, S), generator=torch.Generator().manual_seed(32)).tolist()
    full, eng = (Engine.from_weights(cfg, w, kv_cache=k) for k in ("bf16", "kv4"))
    assert list(full.generate(prompt, 1)) == list(eng.generate(prompt, 1))
    for i in range(cfg.layers):
        n, s, c = O.unpack(eng.kv4[i], cfg.head_dim, eng.kv_group)
        for j, x in enumerate((full.k_cache, full.v_cache)):
            for got, want in zip((n, s, c), O.quantise(x[i, :, :, :S].cpu(), eng.kv_group)):
                assert torch.equal(got[j][:, :, :S], want)


def test_engines_of_different_groups(dev, monkeypatch):
    """Three engines at once, each with its own group size, against the replay over its cache; then the
    first again."""
    cfg, B, S, n = SMALL, 2, 33, 20
    w = perturbed_weights(cfg, seed=33)
    prompt = torch.randint(0, cfg.vocab, (B, S), generator=torch.Generator().manual_seed(34))
    engines = [Engine.from_weights(cfg, w, keep_logits=True, kv_cache="kv4", kv_group=g)
               for g in (None, 64, 128)]
    assert [e.kv_group for e in engines] == [32, 64, 128]
    traced = [e.trace(prompt.tolist(), n) for e in engines]
    assert [e.kv4.shape[-1] for e in engines] == [5120, 4608, 4352]
    for eng, (toks, logits) in zip(engines, traced):
        replay, _ = replay_and_check_rows(eng, w, monkeypatch,
                                          lambda o: o.teacher_forced_decode(prompt, toks))
        _, err = check_against_replay(toks, logits, replay)
        assert err < LOGIT_ATOL
    assert torch.equal(engines[0].trace(prompt.tolist(), n)[0], traced[0][0])
    with pytest.raises(ValueError):
        Engine.from_weights(cfg, w, kv_cache="kv4", kv_group=16)
