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


@pytest.mark.parametrize('dim', [32, 64, 128, 256])
def test_gradients_of_fp32_in_two_pieces_are_outside(dim):
    """Two rows to sum: the bound is a few roundings, what a third piece holds is more."""
    for user_zero, which, users in ((True, 0, 200), (False, 1, 2)):
        ratio = _ratios(torch.float32, 2, 1.0, user_zero, dim=dim, users=users, pieces=2)[which]
        assert ratio > 1.2, (user_zero, ratio)


def test_scores_of_fp32_in_two_pieces_are_outside():
    user, item = cb.thin_tables(200, 3, 32, 1, 'cpu')
    z, tol = cb.thin_scores(user, item, 1.5)
    assert cb.worst(cb.cut_scores(user, item, 1.5, 3), z, tol) <= 0.1
    assert cb.worst(cb.cut_scores(user, item, 1.5, 2), z, tol) > 1.5
