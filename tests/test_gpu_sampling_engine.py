"""GPU: drawn generation where the model gives no numbers."""

import pytest
import torch

from kernel_optim_amd.engine import Engine, Sampling
from tests.test_oracle_qwen3 import SMALL, perturbed_weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kw", [dict(weight_format="fp8"), dict(decode_graph="fused"),
                                dict(decode_graph="hipblaslt"), dict(kv_cache="kv4")])
def test_sequences_without_numbers_get_no_token(dev, kw):
    """A NaN in the last norm's gain: every logit is NaN, every id -1, whose embedding is zeros, and the
    engine goes on."""
    w = perturbed_weights(SMALL, seed=5)
    w["final_norm"][3] = float("nan")
    eng = Engine.from_weights(SMALL, w, **kw)
    prompt = [[1, 2, 3, 4], [9, 8, 7, 6]]
    assert list(eng.generate(prompt, 5, sampling=Sampling(temperature=0.8, top_p=0.9, seed=1))) == [[-1, -1]] * 5
    torch.cuda.synchronize()
    good = Engine.from_weights(SMALL, perturbed_weights(SMALL, seed=5), **kw)
    out = list(good.generate(prompt, 5, sampling=Sampling(seed=1)))
    assert all(0 <= t < SMALL.vocab for row in out for t in row)
