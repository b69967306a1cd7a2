"""Orthogonalised updates at the limits of what is accepted: many steps, other coefficients, matrices whose entries are alike, norms under eps."""
import math

import pytest
import torch

from test_gpu_muon import A, B, C, DEV, DTYPES, distance, exact, half_step, plain32

pytestmark = pytest.mark.gpu


def test_numbers_that_do_not_fit_are_refused():
    """By the operators too, which `Muon.step` calls with a group's settings as they are now."""
    import trl_amd

    x = torch.ones((4, 5), device=DEV)
    m = torch.zeros_like(x)
    for steps in (2**32 + 5, 0, 101):
        with pytest.raises(ValueError):
            trl_amd.ops.orthogonalize([x], [A, B, C], steps, 1e-7)
        with pytest.raises(ValueError):
            trl_amd.ops.muon_step_([x], [x.clone()], [m], [], [0.1, 0.9, 0.0, 1.0, 0.0], [], [A, B, C], steps, 1e-7)
    for group in (2**32, 1, -1):
        with pytest.raises(ValueError):
            trl_amd.ops.muon_step_([x], [x.clone()], [m], [group], [0.1, 0.9, 0.0, 1.0, 0.0], [], [A, B, C], 5, 1e-7)
    assert bool((x == 1).all()) and not m.any()
