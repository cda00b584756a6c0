"""Where a model's masks under a ``dropout_seed`` begin, on the CPU: the kernel is replaced by a formula of seed, block and
position."""
import threading

import numpy as np
import pytest
import torch
from torch.utils.checkpoint import checkpoint

import graphsage_amd as ga
from graphsage_amd import _lib, kernels


def _plain(x, rate, seed, offset):
    at = torch.arange(x.numel()) + 8 * offset + 1_000_003 * seed
    keep = ((at * 2654435761) % 4294967296 >> 16) >= rate * 65536
    return x.detach() * keep.reshape(x.shape) / (1 - rate)


@pytest.fixture
def model(monkeypatch):
    monkeypatch.setattr(kernels, 'dropout', _plain)
    edges = np.array([[0, 1, 2, 3, 4, 3], [3, 4, 3, 0, 1, 2]])
    g = ga.Graph({'user': np.zeros((3, 2)), 'item': np.zeros((2, 2))}, {'user': [0, 1, 2], 'item': [3, 4]}, edges)
    gen = ga.GraphSAGEGenerator(g, 2, [2, 2], head_node_types=['user', 'item'], seed=3)
    return ga.GraphSAGE([4, 4], gen, dropout=0.5, dropout_seed=7)


def _two_layers(drop, x):
    return drop(torch.tanh(drop(x) * 1.5)).sum()


@pytest.mark.parametrize('reentrant', [False, True])
def test_a_forward_pass_run_again_draws_the_masks_it_drew(model, reentrant):
    x = torch.randn(4, 25, dtype=torch.float64, requires_grad=True)
    loss = _two_layers(model._dropper(40), x)
    (want,) = torch.autograd.grad(loss, x)
    again = checkpoint(lambda x: _two_layers(model._dropper(40), x), x, use_reentrant=reentrant)
    assert torch.equal(again, loss)
    again.backward()
    assert torch.equal(x.grad, want) and model._dropout_drawn == 0


@pytest.mark.parametrize('reentrant', [False, True])
def test_without_a_place_it_is_refused(model, reentrant):
    x = torch.randn(4, 25, dtype=torch.float64, requires_grad=True)
    loss = checkpoint(lambda x: _two_layers(model._dropper(), x), x, use_reentrant=reentrant)
    with pytest.raises(_lib.GsageError, match='dropout_offset'):
        loss.backward()


def test_calls_go_on_where_the_last_one_ended(model):
    x = torch.ones(4, 25, dtype=torch.float64)
    first, second = model._dropper(), model._dropper()
    a, b, c = first(x), second(x), first(x)
    assert model._dropout_drawn == 39                         # 13 blocks of eight each
    for got, at in ((a, 0), (b, 13), (c, 26)):
        assert torch.equal(got, _plain(x, 0.5, 7, at))
    drop = model._dropper(100)
    assert torch.equal(drop(x), _plain(x, 0.5, 7, 100)) and torch.equal(drop(x), _plain(x, 0.5, 7, 113))
    assert model._dropout_drawn == 39                         # a call with a place of its own counts nothing


def test_threads_draw_from_stretches_that_do_not_meet(model, monkeypatch):
    seen = []
    monkeypatch.setattr(kernels, 'dropout', lambda x, rate, seed, offset: seen.append(offset) or x)
    x = torch.ones(3)

    def work():
        for _ in range(500):
            model._dropper()(x)
    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert sorted(seen) == list(range(2000)) and model._dropout_drawn == 2000


def test_refusals(model):
    with pytest.raises(ValueError):
        model._dropper(-1)
    model.dropout_seed = None
    with pytest.raises(ValueError, match='dropout_seed'):
        model._dropper(0)
    assert model._dropper()(torch.ones(4)).shape == (4,)
    model.eval()
    x = torch.ones(4)
    assert model._dropper()(x) is x
