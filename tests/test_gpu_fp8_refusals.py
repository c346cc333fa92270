"""GPU: calls of the 8-bit ops that are refused with ValueError before anything is launched."""

import pytest
import torch

from kernel_optim_amd.kernels.fp8 import Fp8Linear, fp8_quantize
from kernel_optim_amd.kernels.gemv import EPI_BF16

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def test_out_that_is_no_fp8_tensor(dev):
    x, nw = torch.zeros(4, 8, dtype=BF16, device=dev), torch.zeros(8, dtype=BF16, device=dev)
    for kw in (dict(), dict(nw=nw), dict(pair=True)):
        with pytest.raises(ValueError):
            fp8_quantize(x, out=x, **kw)


@pytest.mark.parametrize("M,K", [(3, 256), (40, 8704), (200, 256)])
def test_held_objects_take_held_rows_alone(dev, M, K):
    """Without a copy of x's codes: their workspace holds the sums' scratch at most, and the results are
    those of an object that has one."""
    g = torch.Generator().manual_seed(M)
    x, w = (torch.randn(n, K, generator=g).to(BF16).to(dev) for n in (M, 48))
    w, xq = fp8_quantize(w), fp8_quantize(x)
    y, z = (torch.empty(M, 48, dtype=BF16, device=dev) for _ in range(2))
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    held = Fp8Linear(M, 48, K, EPI_BF16, False, device=dev, held=True)
    scratch = held._scratch.numel()
    assert torch.cuda.memory_allocated() - before <= scratch + 512
    held(xq, w, y=y)
    Fp8Linear(M, 48, K, EPI_BF16, False)(x, w, y=z)
    assert torch.equal(y, z)
    with pytest.raises(ValueError):
        held(x, w, y=y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held(xq, w, y=y)
    for i in range(3):
        fp8_quantize(x * (i + 2), out=xq)
        y.fill_(7)
        graph.replay()
        Fp8Linear(M, 48, K, EPI_BF16, False)(x * (i + 2), w, y=z)
        torch.cuda.synchronize()
        assert torch.equal(y, z)


def test_prompts_hold_no_copies_of_their_rows_for_q_k_and_v(dev, monkeypatch):
    """The prompt's q, k and v products share one quantised copy of their rows, and have no workspace
    for another."""
    import kernel_optim_amd.prefill as prefill
    from kernel_optim_amd.engine import Engine
    from tests.test_oracle_qwen3 import SMALL, perturbed_weights
    made = []

    class Noted(Fp8Linear):
        def __init__(self, *args, **kw):
            super().__init__(*args, **kw)
            made.append(self)

    monkeypatch.setattr(prefill, "Fp8Linear", Noted)
    eng = Engine.from_weights(SMALL, perturbed_weights(SMALL, seed=5), weight_format="fp8")
    list(eng.generate([list(range(80))], 1))
    qkv = [op for op in made if not op.norm and op.K == SMALL.hidden and op.epi == EPI_BF16]
    assert len(qkv) == 3 and all(op._xq is None for op in qkv)
