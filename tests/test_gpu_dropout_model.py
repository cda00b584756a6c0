"""A model with a ``dropout_seed`` under activation checkpointing: the pass that runs again draws the masks of the first
one, or is refused -- needs a GPU."""
import numpy as np
import pytest
import torch
from torch.utils.checkpoint import checkpoint

import graphsage_amd as ga
from graphsage_amd import _lib

pytestmark = pytest.mark.gpu


def _toy(agg_option, dropout=0.4):
    rng = np.random.default_rng(0)
    nu, ni = 60, 20
    u = np.concatenate([rng.integers(0, nu, 900), np.arange(nu)])
    it = np.concatenate([rng.integers(0, ni, 900), np.arange(nu) % ni]) + nu
    e = np.stack([u, it])
    feats = {'user': rng.standard_normal((nu, 12)).astype(np.float32), 'item': rng.standard_normal((ni, 9)).astype(np.float32)}
    g = ga.Graph(feats, {'user': list(range(nu)), 'item': list(range(nu, nu + ni))}, np.concatenate([e, e[::-1]], axis=1))
    gen = ga.GraphSAGEGenerator(g, 16, [5, 3], head_node_types=['user', 'item'], seed=4)
    links = [(int(a), int(b) + nu) for a, b in zip(rng.integers(0, nu, 16), rng.integers(0, ni, 16))]
    batch, _ = gen.flow(links, targets=np.zeros(16), shuffle=False)[0]
    return ga.GraphSAGE([16, 8], gen, agg_option=agg_option, dropout=dropout, dropout_seed=11, seed=6).build(), batch


def _grads(model, embeddings):
    user, item = embeddings
    return torch.autograd.grad((user * item).sum(), model.parameters())


@pytest.mark.parametrize('agg_option', ['mean', 'attention'])
def test_gradients_under_checkpointing_are_those_without(cuda, agg_option):
    model, batch = _toy(agg_option)
    plain = model(batch, dropout_offset=1 << 30)
    want = _grads(model, plain)
    again = checkpoint(lambda: model(batch, dropout_offset=1 << 30), use_reentrant=False)
    for a, b in zip(again, plain):
        assert torch.equal(a, b)
    for a, b in zip(_grads(model, again), want):
        assert torch.equal(a, b)
    other = model(batch, dropout_offset=2 << 30)
    assert not torch.equal(other[0], plain[0]) and model._dropout_drawn == 0

    with pytest.raises(_lib.GsageError, match='dropout_offset'):
        _grads(model, checkpoint(lambda: model(batch), use_reentrant=False))


def test_without_dropout_checkpointing_needs_no_place(cuda):
    model, batch = _toy('attention')
    model.eval()
    want = _grads(model, model(batch))
    for a, b in zip(_grads(model, checkpoint(lambda: model(batch), use_reentrant=False)), want):
        assert torch.equal(a, b)


def test_a_captured_pass_draws_by_the_seed_in_memory(cuda):
    model, batch = _toy('attention')
    slots = [batch[i] for i in range(len(batch))]
    model.dropout_seed = torch.tensor([3], dtype=torch.int64, device='cuda')
    with torch.no_grad():
        model(slots, dropout_offset=5)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = model(slots, dropout_offset=5)
        seen = []
        for seed in (3, 4, 3, 5):
            model.dropout_seed.fill_(seed)
            graph.replay()
            torch.cuda.synchronize()
            want = model(slots, dropout_offset=5)
            for a, b in zip(out, want):
                assert torch.equal(a, b)
            seen.append(out[0].clone())
    assert torch.equal(seen[0], seen[2]) and not torch.equal(seen[0], seen[1]) and not torch.equal(seen[0], seen[3])
