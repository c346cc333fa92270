"""The oracle of sampling against the filters' own statements, on distributions that can be
counted by hand."""

import math

import numpy as np
import pytest
import torch

from oracle import sampling as O


def test_filters():
    w = np.array([8, 4, 2, 1, 1]) / 8
    assert O.kept(w, 0, 1.0, 0.0) == 5 and O.kept(w, 2, 1.0, 0.0) == 2 and O.kept(w, 9, 1.0, 0.0) == 5
    assert O.kept(w, 0, 0.5, 0.0) == 1      # the second has 8 of 16 before it: not below 8
    assert O.kept(w, 0, 0.51, 0.0) == 2 and O.kept(w, 0, 0.0, 0.0) == 1
    assert O.kept(w, 3, 0.9, 0.0) == 3      # of 14: 12 before the third, below 12.6
    assert O.kept(w, 0, 1.0, 0.25) == 3 and O.kept(w, 0, 1.0, 0.3) == 2 and O.kept(w, 0, 1.0, 1.0) == 1


@pytest.mark.parametrize("u,want", [(0.0, 2), (0.49, 2), (0.51, 0), (0.74, 0), (0.76, 3), (0.99, 3),
                                    (1.0, 3), (-1.0, 2), (float("nan"), 2)])
def test_draw_runs_in_falling_order(u, want):
    x = torch.tensor([math.log(2), -math.inf, math.log(4), math.log(2), float("nan")])
    i, logp = O.sample(x, u, 1.0, 0, 1.0, 0.0)
    assert i == want and logp == pytest.approx(math.log(0.5 if want == 2 else 0.25))


def test_ends():
    x = torch.tensor([1.0, 3.0, 3.0])
    assert O.sample(x, 0.9, 0.0, 0, 1.0, 0.0) == (1, 0.0)
    assert O.sample(torch.full((4,), -math.inf), 0.5, 1.0, 0, 1.0, 0.0) == (-1, -math.inf)
    assert O.sample(torch.tensor([0.0, math.inf, math.inf]), 0.6, 1.0, 0, 1.0, 0.0)[0] == 2
    assert O.sample(torch.tensor([-0.0, 0.0, 0.0]), 0.0, 1.0, 1, 1.0, 0.0)[0] == 0
