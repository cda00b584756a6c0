"""Targets that are predicted well: g (1 - p) is what is left of g and -g p, and stays as exact as fp32 holds it whatever the
tables' type -- needs a GPU.  Bounds: catalog_bounds.py (checked on the CPU in test_catalog_bounds.py)."""
import pytest
import torch

import catalog_bounds as cb
from graphsage_amd import kernels

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _run(case):
    user, item, target, bias, scale, g_log_prob, g_entropy = case
    r = kernels.catalog_log_probs(user, item, target, bias, scale)
    g = kernels.catalog_log_probs_bwd(user, item, target, bias, scale, r.lse, r.entropy, g_log_prob, g_entropy)
    return dict(lse=r.lse, entropy=r.entropy, g_user=g[0], g_item=g[1], g_bias=g[2])


def _check(case):
    want, tol = cb.reference(*case)
    for name, got in _run(case).items():
        off = cb.worst(got, want[name], tol[name])
        assert off <= 1.0, "%s: %.3g times the bound" % (name, off)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('items', [1, 2, 8, 40])
@pytest.mark.parametrize('gap', [1.0, 4.6, 6.9, 9.2, 11.5])            # p of 0.99, 0.999, 0.9999, 0.99999 with two items
def test_gradients_of_well_predicted_targets(cuda, dtype, items, gap):
    for user_zero in (False, True):
        for same in (False, True):
            _check(cb.case(dtype, 66, items, 64, gap, 0.0, items, 'cuda', user_zero, same))
    _check(cb.case(dtype, 5, items, 200, gap, 3.0, items, 'cuda', True))
    _check(cb.case(dtype, 300, items, 19, gap, -2.0, items, 'cuda', False, True))


@pytest.mark.parametrize('dtype', DTYPES)
def test_one_item_leaves_next_to_nothing(cuda, dtype):
    """p is 1 within the rounding of the lse that comes back: |lse| u and the two conversions beside it."""
    g = torch.Generator(device='cuda').manual_seed(1)
    user, item = (torch.randn((n, 40), generator=g, device='cuda').to(dtype) for n in (50, 1))
    target = torch.zeros(50, dtype=torch.int32, device='cuda')
    g_log_prob = -torch.rand(50, generator=g, device='cuda')
    r = kernels.catalog_log_probs(user, item, target, None, 3.0)
    g_user, g_item, _ = kernels.catalog_log_probs_bwd(user, item, target, None, 3.0, r.lse, r.entropy, g_log_prob)
    left = g_log_prob.double().abs() * cb.U * (8 * r.lse.double().abs() + 8)
    tiny = 2.0 ** -24 if dtype == torch.float16 else 0.0
    assert bool((g_user.double().abs() <= 3.0 * left[:, None] * item.double().abs() * 1.01 + tiny).all())
    assert bool((g_item.double().abs() <= 3.0 * (left[:, None] * user.double().abs()).sum(0) * 1.01 + tiny).all())


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('users', [5, 66, 300])
@pytest.mark.parametrize('shift', [0.0, 40.0, -300.0])
def test_log_probs_of_well_predicted_targets_far_from_zero(cuda, dtype, users, shift):
    """log p of -1e-2 to -1e-5: as exact as the sum beside the largest score, not as the scores themselves."""
    for items in (1, 2, 8, 40):
        for gap in (4.6, 9.2, 11.5):
            case = cb.case(dtype, users, items, 64, gap, shift, items, 'cuda', True)
            want, tol = cb.reference(*case)
            user, item, target, bias, scale = case[:5]
            got = kernels.catalog_log_probs(user, item, target, bias, scale).log_prob
            off = cb.worst(got, want['log_prob'], tol['log_prob'])
            assert off <= 1.0, "%d items, gap %g: %.3g times the bound" % (items, gap, off)
