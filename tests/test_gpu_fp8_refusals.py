"""GPU: calls of the 8-bit ops that are refused with ValueError before anything is launched."""

import pytest
import torch

from kernel_optim_amd.kernels.fp8 import fp8_quantize

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def test_out_that_is_no_fp8_tensor(dev):
    x, nw = torch.zeros(4, 8, dtype=BF16, device=dev), torch.zeros(8, dtype=BF16, device=dev)
    for kw in (dict(), dict(nw=nw), dict(pair=True)):
        with pytest.raises(ValueError):
            fp8_quantize(x, out=x, **kw)
