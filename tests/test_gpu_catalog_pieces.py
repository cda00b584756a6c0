"""Every piece of an fp32 element counts: rows and sums so short that the bounds are a few roundings, less than the third
piece holds (test_catalog_bounds.py shows on the CPU that two pieces exceed them) -- needs a GPU."""
import pytest
import torch

import catalog_bounds as cb
from graphsage_amd import kernels

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dim', [2, 19, 32, 33, 64, 100, 128, 129, 200, 256])
def test_gradients(cuda, dim):
    for user_zero, users in ((True, 200), (False, 2), (False, 1), (True, 1)):
        for seed in range(3):
            case = cb.case(torch.float32, users, 2, dim, 1.0, 0.0, seed, 'cuda', user_zero)
            want, tol = cb.reference(*case)
            user, item, target, bias, scale, g_log_prob, g_entropy = case
            r = kernels.catalog_log_probs(user, item, target, bias, scale)
            g = kernels.catalog_log_probs_bwd(user, item, target, bias, scale, r.lse, r.entropy, g_log_prob, g_entropy)
            for name, got in (('g_user', g[0]), ('g_item', g[1]), ('g_bias', g[2])):
                off = cb.worst(got, want[name], tol[name])
                assert off <= 1.0, "%s: %.3g times the bound" % (name, off)


@pytest.mark.parametrize('users', [1, 20, 40, 200])
@pytest.mark.parametrize('dim', [2, 19, 32, 33, 64, 100, 128, 129, 200, 256])
def test_scores(cuda, users, dim):
    user, item = cb.thin_tables(users, 1, dim, users + dim, 'cuda')
    z, tol = cb.thin_scores(user, item, 1.5)
    r = kernels.catalog_log_probs(user, item, None, None, 1.5)
    assert cb.worst(r.lse, z[:, 0], tol[:, 0]) <= 1.0        # one item: the lse is its score

    # the gradients' own scores, against a statistic that the caller sets: dz = -g p (log p + entropy), one user at a time
    bias = torch.zeros(1, device='cuda')
    for n in range(min(users, 4)):
        lse = (z[n] + 1.0).float()
        g = torch.tensor([0.7], device='cuda')
        entropy = torch.zeros(1, device='cuda')
        _, _, g_bias = kernels.catalog_log_probs_bwd(user[n:n + 1].contiguous(), item, None, bias, 1.5, lse, entropy, None, g)
        lp = z[n] - lse.double()
        p = torch.exp(lp)
        want = -0.7 * p * lp
        # d(p log p) = p (1 + log p): the score's bound, the lse's conversion (2 u), the exponential (2 u), three products
        slack = p * (1 + lp.abs()) * (tol[n] + 4 * cb.U * lse.double().abs()) + 8 * cb.U * want.abs() + 4 * cb.U * p
        assert cb.worst(g_bias, want, 0.7 * slack + 2.0 ** -26) <= 1.0
