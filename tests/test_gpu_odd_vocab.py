"""GPU: vocabularies that are no multiple of 8, whose logits' rows begin at any bf16: greedy ids of such
rows, and engines on bf16 and 8-bit weights."""

import pytest
import torch

from dataclasses import replace

from kernel_optim_amd.engine import Engine, Sampling
from kernel_optim_amd.kernels.gemv import argmax_rows
from oracle.ops import argmax_first
from tests.test_gpu_fp8_engine import check, prompts
from tests.test_oracle_qwen3 import SMALL, perturbed_weights

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.mark.parametrize("M,N", [(1, 1), (9, 3), (5, 7), (4, 9), (17, 15), (3, 1001), (33, 32003),
                                 (8, 65539), (2, 151937)])
@pytest.mark.parametrize("skip", [0, 1, 6])
def test_argmax_of_rows_at_any_alignment(dev, M, N, skip):
    """Rows of a matrix without padding and of one with ``skip`` columns in front; ties at the row's ends,
    which lie in front of and behind the 16-byte loads."""
    g = torch.Generator().manual_seed(M + N)
    wide = torch.randn(M, N + skip, generator=g).to(BF16)
    x = wide[:, skip:]
    x[::3, 0] = x[::3, -1] = 9.0
    x[1::3, -1] = 9.0
    x[M - 1] = float("-inf")
    want = argmax_first(x)
    ids = torch.full((M,), -7, dtype=torch.int64, device=dev)
    argmax_rows(wide.to(dev)[:, skip:], ids)
    assert torch.equal(ids.cpu(), want)


@pytest.mark.parametrize("kw", [dict(weight_format="fp8"), dict(weight_format="fp8", kv_cache="kv4"),
                                dict(decode_graph="hipblaslt"), dict(decode_graph="fused")])
@pytest.mark.parametrize("B", [1, 3])
def test_engine(dev, kw, B):
    """Decode, draw and speculate; every greedy id is the first maximum of its own logits."""
    cfg, n = replace(SMALL, vocab=1003), 8
    w = perturbed_weights(cfg, seed=51)
    prompt = [(p * 4)[:21] for p in prompts(cfg, B, 6, 52).tolist()]
    eng = Engine.from_weights(cfg, w, keep_logits=True, spec=True, **kw)
    toks, logits = eng.trace(prompt, n)
    assert torch.equal(toks, torch.stack([argmax_first(l) for l in logits], 1))
    vout, logits = eng.verify_step(torch.cat((toks, toks), 1)[:, :eng.T], torch.full((B,), 21))
    assert torch.equal(vout, argmax_first(logits).view(B, eng.T))
    assert len(list(eng.generate(prompt, n))) == n
    drawn = list(eng.generate(prompt, n, sampling=Sampling(temperature=1.3, top_k=50, seed=2)))
    assert len(drawn) == n and all(0 <= t < cfg.vocab for row in drawn for t in row)


def test_logits_against_the_replay(dev, monkeypatch):
    cfg, n, B = replace(SMALL, vocab=1001), 10, 3
    w = perturbed_weights(cfg, seed=53)
    prompt = prompts(cfg, B, 19, 54)
    toks, logits = Engine.from_weights(cfg, w, keep_logits=True, weight_format="fp8").trace(
        prompt.tolist(), n)
    check(monkeypatch, cfg, w, prompt, toks, logits, 32)
