"""Gradients of gradients through the operators' autograd functions: right, or refused, never silently incomplete.  On the
CPU: the kernels are replaced by plain formulas, what is tested is the functions around them."""
import pytest
import torch

from graphsage_amd import autograd, kernels

MASK = torch.tensor([0.0, 2.0, 2.0, 0.0, 2.0], dtype=torch.float64)


def test_dropout(monkeypatch):
    monkeypatch.setattr(kernels, 'dropout', lambda x, rate, seed, offset: x.detach() * MASK)
    x = torch.randn(5, dtype=torch.float64, requires_grad=True)
    y = autograd.Dropout.apply(x * x * x, 0.5, 3, 0)
    (g,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    torch.testing.assert_close(g, 3 * x * x * MASK)
    (g * g).sum().backward()                                  # sum (3 x^2 m)^2 -> 36 x^3 m^2
    torch.testing.assert_close(x.grad, 36 * x.detach() ** 3 * MASK ** 2)

    # a function of the gradient that came in
    x = torch.randn(5, dtype=torch.float64, requires_grad=True)
    c = torch.randn(5, dtype=torch.float64, requires_grad=True)
    y = autograd.Dropout.apply(x, 0.5, 3, 0)
    (g,) = torch.autograd.grad(y, x, c, create_graph=True)
    g.sum().backward()
    assert torch.equal(c.grad, MASK)


def test_dropout_seed_in_memory_is_the_drawn_one(monkeypatch):
    seen = []
    monkeypatch.setattr(kernels, 'dropout', lambda x, rate, seed, offset: seen.append(int(seed)) or x.detach() * MASK)
    seed = torch.tensor([6])
    x = torch.randn(5, dtype=torch.float64, requires_grad=True)
    y = autograd.Dropout.apply(x * x, 0.5, seed, 0)
    seed.fill_(9)
    (g,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    (g * g).sum().backward()
    assert set(seen) == {6} and len(seen) == 2


def _catalog(user, item, targets, bias, scale, **_):
    logp = torch.log_softmax(scale * user.detach() @ item.detach().T, 1)
    lse = torch.logsumexp(scale * user.detach() @ item.detach().T, 1)
    return kernels.CatalogLogProbs(logp.gather(1, targets.long()[:, None])[:, 0], -(logp.exp() * logp).sum(1), lse, None, None)


def test_catalog_is_refused(monkeypatch):
    monkeypatch.setattr(kernels, 'catalog_log_probs', _catalog)
    monkeypatch.setattr(kernels, 'catalog_log_probs_bwd', lambda user, item, *a, **k: (torch.ones_like(user), torch.ones_like(item), None))
    user, item = torch.randn(3, 4, requires_grad=True), torch.randn(6, 4, requires_grad=True)
    log_prob, entropy = autograd.CatalogLogProbs.apply(user * user, item, torch.tensor([0, 1, 2], dtype=torch.int32), None, 2.0)
    g_user, g_item = torch.autograd.grad((log_prob + entropy).sum(), (user, item), create_graph=True)
    with pytest.raises(RuntimeError, match='cannot be differentiated again'):
        ((g_user ** 2).sum() + (g_item ** 2).sum()).backward()
    log_prob, entropy = autograd.CatalogLogProbs.apply(user * user, item, torch.tensor([0, 1, 2], dtype=torch.int32), None, 2.0)
    (log_prob + entropy).sum().backward()                     # once is as before
    assert torch.equal(item.grad, torch.ones_like(item))


def test_attention_is_refused(monkeypatch):
    monkeypatch.setattr(kernels, 'neighbor_attention', lambda q, *a: (q.detach() + 1, torch.zeros(q.shape[:2])))
    monkeypatch.setattr(kernels, 'neighbor_attention_bwd', lambda q, k, *a, **kw: (torch.ones_like(q), torch.ones_like(k), None))
    q, k = torch.randn(3, 2, 4, requires_grad=True), torch.randn(6, 1, 4, requires_grad=True)
    out, _ = autograd.NeighborAttention.apply(q * q, k, None, None, 2, 0, None, None, None)
    g_q, g_k = torch.autograd.grad(out.sum(), (q, k), create_graph=True)
    with pytest.raises(RuntimeError, match='cannot be differentiated again'):
        ((g_q ** 2).sum() + (g_k ** 2).sum()).backward()
    out, _ = autograd.NeighborAttention.apply(q * q, k, None, None, 2, 0, None, None, None)
    out.sum().backward()
    assert torch.equal(k.grad, torch.ones_like(k))
