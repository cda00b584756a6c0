"""More rows and elements than one launch has threads for -- needs a GPU (of 288 GB: up to 60 GB are used)."""
import pytest
import torch

from graphsage_amd import kernels

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _give_back():
    yield
    torch.cuda.empty_cache()


def _rows(n, dim, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    return torch.randn((n, dim), generator=g, device='cuda', dtype=torch.bfloat16)


def test_gradients_of_more_than_2_to_the_29_elements(cuda):
    n, items, dim = 2_100_000, 40, 256                # 8 threads an element join them: 2^29 elements are 2^32 threads
    user, item = _rows(n, dim, 1), _rows(items, dim, 2) / 16
    target = (torch.arange(n, device='cuda') % items).to(torch.int32)
    r = kernels.catalog_log_probs(user, item, target, None, 0.5)
    g = torch.full((n,), -1.0, device='cuda')
    g_user, _, _ = kernels.catalog_log_probs_bwd(user, item, target, None, 0.5, r.lse, r.entropy, g, None, need_item=False)
    for at in (0, 1_000_000, (1 << 29) // dim - 3, (1 << 29) // dim, n - 33):
        u = user[at:at + 33].double().requires_grad_()
        logp = torch.log_softmax(0.5 * u @ item.double().T, 1)
        lp = logp.gather(1, target[at:at + 33].long()[:, None])[:, 0]
        (-lp).sum().backward()
        assert float((r.log_prob[at:at + 33].double() - lp.detach()).abs().max()) <= 1e-4
        # dz to 2^-8 of p against rows of about 1, 40 of them, rounded to bf16
        size = 0.5 * (torch.softmax(0.5 * user[at:at + 33].double() @ item.double().T, 1) @ item.double().abs())
        assert bool(((g_user[at:at + 33].double() - u.grad).abs() <= 2.0 ** -8 * size + 2.0 ** -8 * u.grad.abs() + 1e-5).all())


def test_more_than_2_to_the_29_users(cuda):
    n = (1 << 29) + 4177                              # a block lays 32 rows out, a wave joins a user
    base = torch.linspace(-2, 2, 1021, device='cuda').to(torch.bfloat16)
    user = torch.empty(n, 1, dtype=torch.bfloat16, device='cuda')
    for lo in range(0, n, 1021 << 16):
        m = min(n - lo, 1021 << 16)
        user[lo:lo + m, 0] = base.repeat((m + 1020) // 1021)[:m]
    item = torch.tensor([[1.0], [-0.5], [0.25]], device='cuda').to(torch.bfloat16)
    r = kernels.catalog_log_probs(user, item)
    for lo in (0, (1 << 26) - 500, (1 << 28), (1 << 29) - 500, n - 1021):
        z = user[lo:lo + 1021].double() @ item.double().T
        lse = torch.logsumexp(z, 1)
        p = torch.softmax(z, 1)
        assert float((r.lse[lo:lo + 1021].double() - lse).abs().max()) <= 1e-5
        assert float((r.entropy[lo:lo + 1021].double() + (p * torch.log(p)).sum(1)).abs().max()) <= 1e-5


def test_best_items_of_an_empty_catalog_for_many_users(cuda):
    n = (1 << 24) + 5
    user, item = torch.zeros((n, 1), dtype=torch.bfloat16, device='cuda'), torch.zeros((0, 1), dtype=torch.bfloat16, device='cuda')
    r = kernels.catalog_log_probs(user, item, top_k=1)
    assert bool((r.top_ids == -1).all()) and bool((r.top_log_prob == -float('inf')).all()) and bool((r.lse == -float('inf')).all())
