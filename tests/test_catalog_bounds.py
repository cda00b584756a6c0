"""The bounds that the catalog's GPU tests use, on the CPU: the kernels' rounding restated stays inside them, and mistakes
that they are there for do not."""
import pytest
import torch

import catalog_bounds as cb

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _ratios(dtype, items, gap, user_zero, dim=64, users=66, same=False, **planted):
    c = cb.case(dtype, users, items, dim, gap, 0.0, items, 'cpu', user_zero, same)
    want, tol = cb.reference(*c)
    got = cb.emulate(*c, **planted)
    return [cb.worst(x, want[n], tol[n]) for n, x in zip(('g_user', 'g_item'), got)]


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('items', [1, 2, 8, 40])
@pytest.mark.parametrize('gap', [1.0, 4.6, 6.9, 11.5])
def test_the_rounding_is_inside(dtype, items, gap):
    for user_zero in (False, True):
        for same in (False, True):
            assert max(_ratios(dtype, items, gap, user_zero, same=same)) <= 1.0


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('gap', [6.9, 9.2, 11.5])
def test_a_target_whose_two_halves_are_rounded_apart_is_outside(dtype, gap):
    """g whole and -g p in pieces: what a cut leaves out of -g p stands where g (1 - p) should."""
    assert _ratios(dtype, 2, gap, True, whole_target=False)[0] > 1.5
    if dtype == torch.bfloat16:
        assert _ratios(dtype, 2, gap, False, same=True, whole_target=False)[1] > 1.5
