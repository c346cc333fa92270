"""Oracle of sampling: one row at a time, in 64 bits, by sorting. The rule is stated in
kernel_optim_amd/kernels/sampling.py."""

import math

import numpy as np
import torch


def order(x):
    """x fp64 numpy [V] -> indices by falling logit, the lowest index first; no -infinity, no NaN."""
    at = np.flatnonzero(x > -math.inf)
    return at[np.argsort(-x[at], kind="stable")]


def weights(x, o, t):
    """The ordered tokens' probabilities over the largest one, fp64."""
    if x[o[0]] == math.inf:
        return (x[o] == math.inf).astype(np.float64)
    with np.errstate(over="ignore"):
        return np.exp((x[o] - x[o[0]]) / t)


def kept(w, k, p, mp):
    """How many of the ordered weights the filters keep."""
    n = len(w)
    if 0 < k < n:
        n = k
    if p < 1:
        before = np.cumsum(w[:n]) - w[:n]
        n = min(n, max(1, int((before < p * w[:n].sum()).sum())))
    if mp > 0:
        n = min(n, max(1, int((w >= mp).sum())))
    return n


def sample(logits, u, t, k, p, mp):
    """logits [V] -> (id, log-probability)."""
    x = logits.double().cpu().numpy()
    t, p, mp, u = (float(np.float32(v)) for v in (t, p, mp, u))
    o = order(x)
    if len(o) == 0:
        return -1, -math.inf
    if not t > 0:
        return int(o[0]), 0.0
    w = weights(x, o, t)
    n = kept(w, k, p, mp)
    c = np.cumsum(w[:n])
    u = u if u > 0 else 0.0
    i = min(int((c <= u * c[-1]).sum()), n - 1)
    return int(o[i]), math.log(w[i] / c[-1]) if w[i] > 0 else -math.inf


def rows(logits, u, t, k, p, mp):
    """sample for every row; settings are numbers or [B] tensors."""
    B = logits.shape[0]
    at = lambda v, b: v[b].item() if isinstance(v, torch.Tensor) else v
    out = [sample(logits[b], u[b].item(), *(at(v, b) for v in (t, k, p, mp))) for b in range(B)]
    return torch.tensor([i for i, _ in out]), torch.tensor([l for _, l in out], dtype=torch.float64)
