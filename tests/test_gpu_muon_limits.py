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


def low_rank(shape, rank, gen, whole=False):
    draw = (lambda s: torch.randint(-8, 9, s, generator=gen, device=DEV).float()) if whole else (lambda s: torch.randn(s, generator=gen, device=DEV))
    return draw((shape[0], rank)) @ draw((rank, shape[1]))


def exact_of_rank(u, rank, steps, coefficients=(A, B, C), eps=1e-7):
    """By singular values, those behind the rank being zero, not what rounding has left of them."""
    a, b, c = coefficients
    left, s, right = torch.linalg.svd(u.double().cpu(), full_matrices=False)
    s = s / max(float(s.norm()), eps)
    s[rank:] = 0
    for _ in range(steps):
        s = a * s + b * s**3 + c * s**5
    return ((left * s) @ right).to(u.device)


@pytest.mark.parametrize("steps", [5, 12, 17, 18, 20, 30, 100])
@pytest.mark.parametrize("shape", [(1, 9), (16, 500), (40, 70), (64, 900), (900, 48), (33, 40000)])
def test_narrow_matrices_of_low_rank_and_many_steps(shape, steps):
    """64 rows or fewer go by the Gram matrix, whose rounding moves eigenvalues of zero either way.  Whole numbers of rank one are exactly of that rank in every type:
    the result is u / |u| times one number, which 64 bits hold to 1e-12 after five steps and, the usual polynomial's cycle attracting, to 2e-7 after 100.  A direction
    that is not the matrix's own is taken for one of size 2^-23, grows to size one and stays there (0.68 to 1.13): 1.7 2^23 in all, times the 64 2^-53 of
    the matrix that rounding leaves in it is 1e-7.  So 1e-5 has room for both."""
    import trl_amd

    gen = torch.Generator(device=DEV).manual_seed(shape[0] + steps)
    for dtype in DTYPES.values():
        u = low_rank(shape, 1, gen, whole=True).to(dtype)
        got, want = trl_amd.orthogonalize(u, ns_steps=steps), exact_of_rank(u, 1, steps)
        assert distance(got, want) <= (1e-5 + half_step(dtype)) * float(want.norm()) + 1e-30, dtype
    # of rank four, rounded to fp32: what the rounding adds is at 2^-24, and comes up by itself from 12 steps on.  Then only the size is known.
    u = low_rank(shape, 4, gen)
    got = trl_amd.orthogonalize(u, ns_steps=steps)
    assert float(torch.linalg.matrix_norm(got.double().cpu(), 2)) <= 1.1337 * 1.01  # the polynomial's largest value on its way
    if steps <= 12:
        want = exact(u, steps=steps)
        assert distance(got, want) <= 4 * distance(plain32(u, steps=steps), want) + 1e-6 * float(want.norm())
