"""What ``fit`` and ``evaluate`` report as the loss of a head that has one of its own -- needs a GPU."""
import numpy as np
import pytest
import torch

import graphsage_amd as ga
from graphsage_amd.link_utils import CatalogHead
from graphsage_amd.train import LinkHead, Trainer

pytestmark = pytest.mark.gpu


def _toy(seed=0, nu=120, ni=35):
    rng = np.random.default_rng(seed)
    u = np.concatenate([rng.integers(0, nu, 3000), np.arange(nu)])
    it = np.concatenate([rng.integers(0, ni, 3000), np.arange(nu) % ni]) + nu
    e = np.stack([u, it])
    feats = {'user': rng.standard_normal((nu, 24)).astype(np.float32), 'item': rng.standard_normal((ni, 19)).astype(np.float32)}
    g = ga.Graph(feats, {'user': list(range(nu)), 'item': list(range(nu, nu + ni))}, np.concatenate([e, e[::-1]], axis=1))
    links = [(int(a), int(b) + nu) for a, b in zip(rng.integers(0, nu, 230), rng.integers(0, ni, 230))]
    return g, links, (rng.random(230) < 0.6).astype(np.float32)


def _own(tr, seq):
    """The head's loss of every batch, in 64 bits, weighted by the batches' sizes."""
    total = count = 0.0
    for i in range(len(seq)):
        batch, y = seq[i]
        user, item = (x.detach().double() for x in tr.model(batch))
        logp = torch.log_softmax(tr.head.scale * user @ item.T, 1)
        pos = torch.from_numpy(np.asarray(y) > 0.5)
        loss = -logp.diagonal()[pos].sum() / max(int(pos.sum()), 1) + tr.head.entropy_weight * (logp.exp() * logp).sum(1).mean()
        total, count = total + float(loss) * len(y), count + len(y)
    return total / count


@pytest.mark.parametrize('agg_option,sizes', [('attention', [16, 8]), ('mean', [32, 32])])
@pytest.mark.parametrize('entropy_weight', [0.0, 0.1])
def test_evaluate_reports_the_loss_that_is_trained(cuda, agg_option, sizes, entropy_weight):
    g, links, targets = _toy()
    gen = ga.GraphSAGEGenerator(g, 50, [5, 3], head_node_types=['user', 'item'], seed=4)
    model = ga.GraphSAGE(sizes, gen, agg_option=agg_option, seed=6)
    tr = Trainer(model, head=CatalogHead(8.0, entropy_weight), lr=1e-2, graph=g, batch_size=50)
    seq = gen.flow(links, targets=targets, shuffle=False)        # four full batches and one of 30
    got, want = tr.evaluate(seq)['loss'], _own(tr, seq)
    assert abs(got - want) <= 1e-5 * abs(want)                   # fp32 embeddings and scores of at most 8
    history = tr.fit(gen.flow(links, targets=targets, seed=1), validation_data=seq, epochs=1, verbose=0)
    assert abs(history['val_loss'][0] - _own(tr, seq)) <= 1e-5 * abs(want)
    assert tr.predict(seq).shape == (230, 1)


def test_heads_without_a_loss_report_the_squared_error(cuda):
    g, links, targets = _toy()
    gen = ga.GraphSAGEGenerator(g, 50, [5, 3], head_node_types=['user', 'item'], seed=4)
    model = ga.GraphSAGE([32, 32], gen, seed=6).build()
    tr = Trainer(model, head=LinkHead(32, cuda, seed=1), lr=1e-2, graph=g, batch_size=50)
    seq = gen.flow(links, targets=targets, shuffle=False)
    want = float(((tr.predict(seq).double().cpu().reshape(-1) - torch.from_numpy(targets).double()) ** 2).mean())
    assert abs(tr.evaluate(seq)['loss'] - want) <= 1e-6


@pytest.mark.parametrize('agg_option,sizes', [('attention', [16, 8]), ('mean', [32, 32])])
def test_a_bias_of_the_catalog_reaches_every_batch(cuda, agg_option, sizes):
    g, links, targets = _toy()
    gen = ga.GraphSAGEGenerator(g, 50, [5, 3], head_node_types=['user', 'item'], seed=4)
    model = ga.GraphSAGE(sizes, gen, agg_option=agg_option, seed=6)
    count = np.bincount([b - 120 for _, b in links], minlength=35) + 1.0
    bias = -np.log(count)
    tr = Trainer(model, head=CatalogHead(8.0, item_bias=bias), lr=1e-2, graph=g, batch_size=50)
    seq = gen.flow(links, targets=targets, shuffle=False)
    total = 0.0
    for i in range(len(seq)):
        batch, y = seq[i]
        rows = torch.tensor([b - 120 for _, b in links[50 * i:50 * i + 50]])
        leaves = [x.detach().double().requires_grad_() for x in model(batch)]
        logp = torch.log_softmax(8.0 * leaves[0] @ leaves[1].T + torch.from_numpy(bias).cuda()[rows.cuda()], 1)
        pos = torch.from_numpy(y > 0.5)
        loss = -logp.diagonal()[pos].sum() / int(pos.sum())
        got, _ = tr.loss(batch, y)
        assert abs(float(got.detach()) - float(loss.detach())) <= 1e-5 * abs(float(loss.detach()))
        total += float(loss.detach()) * len(y)
    assert abs(tr.evaluate(seq)['loss'] - total / 230) <= 1e-5 * abs(total / 230)
    assert np.isfinite(tr.fit(gen.flow(links, targets=targets, seed=1), epochs=1, verbose=0)['loss'][0])


def test_refusals_of_a_catalog_bias(cuda):
    g, links, targets = _toy()
    gen = ga.GraphSAGEGenerator(g, 50, [5, 3], head_node_types=['user', 'item'], seed=4)
    model = ga.GraphSAGE([16, 8], gen, agg_option='attention', seed=6)
    batch, y = gen.flow(links, targets=targets, shuffle=False)[0]
    with pytest.raises(ValueError, match='35 items'):
        Trainer(model, head=CatalogHead(8.0, item_bias=np.zeros(34)), graph=g, batch_size=50).loss(batch, y)
    tr = Trainer(model, head=CatalogHead(8.0, item_bias=np.zeros(35)), graph=g, batch_size=50)
    with pytest.raises(TypeError, match='ids'):
        tr.loss([batch[i] for i in range(len(batch))], y)
    emb = model(batch)
    with pytest.raises(ValueError, match='items'):
        tr.head.loss(emb, y)
    with pytest.raises(ValueError, match='links'):
        tr.head.loss(emb, y, items=torch.zeros(49, dtype=torch.int64, device='cuda'))
    far = torch.full((50,), 35, dtype=torch.int64, device='cuda')
    assert bool(tr.head.loss(emb, y, items=far)[0].isnan())


@pytest.mark.parametrize('with_bias', [False, True])
def test_distinct_items_are_one_choice_each(cuda, with_bias):
    g, links, targets = _toy()
    gen = ga.GraphSAGEGenerator(g, 50, [5, 3], head_node_types=['user', 'item'], seed=4)
    model = ga.GraphSAGE([16, 8], gen, agg_option='attention', seed=6)
    bias = np.linspace(-1, 1, 35) if with_bias else None
    tr = Trainer(model, head=CatalogHead(8.0, 0.1, bias, distinct_items=True), lr=1e-2, graph=g, batch_size=50)
    seq = gen.flow(links, targets=targets, shuffle=False)
    batch, y = seq[0]
    rows = [b - 120 for _, b in links[:50]]
    distinct = sorted(set(rows), key=rows.index)
    assert len(distinct) < 40                                    # 50 links, 35 items
    places = torch.tensor([rows.index(r) for r in distinct], device='cuda')
    own = torch.tensor([distinct.index(r) for r in rows], device='cuda')
    emb = [x.detach().requires_grad_() for x in model(batch)]
    loss, pred = tr.head.loss(emb, y, items=torch.tensor(rows, device='cuda'))
    loss.backward()
    leaves = [x.detach().double().requires_grad_() for x in emb]
    z = 8.0 * torch.matmul(leaves[0], leaves[1][places].T.contiguous())
    if with_bias:
        z = z + torch.from_numpy(bias).cuda()[torch.tensor(distinct).cuda()]
    logp = torch.log_softmax(z, 1)
    pos = torch.from_numpy(y > 0.5).cuda()
    want = -logp.gather(1, own[:, None])[pos].sum() / int(pos.sum()) + 0.1 * (logp.exp() * logp).sum(1).mean()
    want.backward()
    # fp32 scores of at most 9: 1e-5 of the loss, 1e-4 of the largest gradient
    assert abs(float(loss.detach()) - float(want.detach())) <= 1e-5 * abs(float(want.detach())) and pred.shape == (50, 1)
    for a, b in zip(emb, leaves):
        assert float((a.grad.double() - b.grad).abs().max()) <= 1e-4 * float(b.grad.abs().max())
    repeated = [i for i in range(50) if rows.index(rows[i]) != i]
    assert not emb[1].grad[repeated].any()
    assert abs(float(tr.loss(batch, y)[0].detach()) - float(want.detach())) <= 1e-5 * abs(float(want.detach()))
    assert np.isfinite(tr.evaluate(seq)['loss'])
    assert np.isfinite(tr.fit(gen.flow(links, targets=targets, seed=1), epochs=1, verbose=0)['loss'][0])
