"""What the operators around learning and ranking cost, and what they have to return.

Three families, each over the range that a user of the package meets:

* ``attention``: every parent attends over its neighbors' rows, in place of their mean.  The neighbors are rows of a
  table read by id (a sampled batch, or the whole adjacency), or the rows of a layer's own output; forward alone
  (inference) or with the gradients (training);
* ``catalog``: users against every item: log probabilities of given items, the entropy and the best items, with the
  gradients for training;
* ``dropout``: a counter-based keep mask that is never stored.

``run`` computes them from elementary torch operations, or, where ``own`` is true, calls the package.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}
BYTES = {'fp32': 4, 'bf16': 2, 'fp16': 2}


# ---- the cases -------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one user, asked for at once, over its whole history of 20 000 items: latency counts
        {'name': 'attention one long history', 'op': 'attention', 'dtype': 'fp32', 'parents': 1, 'child': 20000,
         'edges': 20000, 'rows': 100000, 'heads': 4, 'kv': 1, 'dim': 64, 'ids': True, 'shared': True, 'train': False},
        # the benchmark's batch: 4096 walks with fan-outs 25 and 10, the hop-1 nodes over their sampled neighbors' features
        {'name': 'attention sampled batch', 'op': 'attention', 'dtype': 'fp32', 'parents': 102400, 'child': 10,
         'edges': 1024000, 'rows': 100000, 'heads': 1, 'kv': 1, 'dim': 64, 'ids': True, 'shared': True, 'train': False},
        # inference over a whole graph: ragged histories, popular nodes first, projected keys and values in 16 bits
        {'name': 'attention whole graph', 'op': 'attention', 'dtype': 'bf16', 'parents': 50000, 'child': 0,
         'edges': 2000000, 'rows': 100000, 'heads': 8, 'kv': 2, 'dim': 64, 'ids': True, 'shared': False, 'train': False},
        # a training step's second layer: 8192 heads over the 25 rows that the first layer gave each of them
        {'name': 'attention layer training', 'op': 'attention', 'dtype': 'fp32', 'parents': 8192, 'child': 25,
         'edges': 204800, 'rows': 204800, 'heads': 4, 'kv': 1, 'dim': 32, 'ids': False, 'shared': True, 'train': True},
        # training of an embedding table through a ragged adjacency, an odd width
        {'name': 'attention table training', 'op': 'attention', 'dtype': 'fp16', 'parents': 6040, 'child': 0,
         'edges': 226000, 'rows': 3700, 'heads': 2, 'kv': 2, 'dim': 33, 'ids': True, 'shared': False, 'train': True},
        # one user against the benchmark's 100 000 items, the ten best: latency counts
        {'name': 'catalog one user', 'op': 'catalog', 'dtype': 'fp32', 'users': 1, 'items': 100000, 'dim': 32,
         'scale': 10.0, 'bias': False, 'top': 10, 'train': False},
        # a small batch against a small catalog
        {'name': 'catalog small batch', 'op': 'catalog', 'dtype': 'fp32', 'users': 100, 'items': 3700, 'dim': 32,
         'scale': 10.0, 'bias': False, 'top': 0, 'train': True},
        # the benchmark's batch, every user against the items of the batch, corrected by how often each is drawn
        {'name': 'catalog in-batch training', 'op': 'catalog', 'dtype': 'fp32', 'users': 4096, 'items': 4096, 'dim': 32,
         'scale': 10.0, 'bias': True, 'top': 0, 'train': True},
        # the same against the whole catalog, in 16 bits
        {'name': 'catalog full training', 'op': 'catalog', 'dtype': 'bf16', 'users': 4096, 'items': 100000, 'dim': 64,
         'scale': 10.0, 'bias': True, 'top': 0, 'train': True},
        # ranking for a block of users
        {'name': 'catalog ranking', 'op': 'catalog', 'dtype': 'fp32', 'users': 512, 'items': 100000, 'dim': 64,
         'scale': 10.0, 'bias': True, 'top': 20, 'train': False},
        # the aggregator inputs of a small batch: 100 links, 32 deepest neighbors of 19 features
        {'name': 'dropout small batch', 'op': 'dropout', 'dtype': 'fp32', 'count': 100 * 32 * 19, 'rate': 0.3},
        # the deepest hop of the benchmark's batch: 4096 walks of 250 rows of 64
        {'name': 'dropout deepest hop', 'op': 'dropout', 'dtype': 'bf16', 'count': 4096 * 250 * 64, 'rate': 0.5},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(['attention', 'attention', 'catalog', 'catalog', 'dropout'])
    dtype = rng.choice(['fp32', 'bf16', 'fp16'])
    if op == 'dropout':
        return {'op': op, 'dtype': dtype, 'count': _spread(rng, 1000, 1 << 25), 'rate': round(rng.uniform(0.05, 0.9), 3)}
    if op == 'catalog':
        train = rng.random() < 0.6
        users = _spread(rng, 1, 4096)
        items = _spread(rng, 300, min(100000, (200000000 if train else 30000000) // users))
        return {'op': op, 'dtype': dtype, 'users': users, 'items': items,
                'dim': rng.choice([8, 16, 19, 32, 33, 48, 64, 64, 100, 128, 200, 256]),
                'scale': rng.choice([1.0, 4.0, 8.0, 10.0]), 'bias': rng.random() < 0.5,
                'top': 0 if train else rng.choice([1, 5, 10, 20, 50, 64]), 'train': train}
    kv = rng.choice([1, 1, 1, 2, 3])
    heads = kv * rng.choice([1, 1, 2, 4, 5])
    dim = rng.choice([8, 16, 19, 32, 33, 64, 64, 100, 128, 200, 256])
    most = min(1000000, 128000000 // (heads * dim))
    train = rng.random() < 0.5
    shared = rng.random() < 0.5
    if rng.random() < 0.5:                                  # as many neighbors for each
        child = _spread(rng, 1, 64)
        parents = _spread(rng, 1, most // child)
        edges, ids = parents * child, rng.random() < 0.5
    else:                                                   # ragged, some without any
        child, parents = 0, _spread(rng, 1, 20000)
        edges, ids = _spread(rng, 1000, most), rng.random() < 0.7
    rows = _spread(rng, 100, 100000) if ids else edges
    return {'op': op, 'dtype': dtype, 'parents': parents, 'child': child, 'edges': edges, 'rows': rows, 'heads': heads,
            'kv': kv, 'dim': dim, 'ids': ids, 'shared': shared, 'train': train}


def work(case):
    e = BYTES[case['dtype']]
    if case['op'] == 'dropout':
        return {'bytes': 2 * e * case['count'], 'flops': case['count']}
    if case['op'] == 'catalog':
        n, v, d = case['users'], case['items'], case['dim']
        tables = (n + v) * d * e + (4 * v if case['bias'] else 0)
        if case['train']:                                   # tables, targets, gradients in; losses and gradients out
            return {'bytes': 2 * tables + n * (4 + 8 + 8), 'flops': 6 * n * v * d}
        return {'bytes': tables + n * (4 + 8 * case['top']), 'flops': 2 * n * v * d}
    p, h, kv, d, n = case['parents'], case['heads'], case['kv'], case['dim'], case['edges']
    tables = 1 if case['shared'] else 2
    rows = min(case['rows'], n) * kv * d * e * tables
    index = (4 * n if case['ids'] else 0) + (0 if case['child'] else 8 * (p + 1))
    moved = 2 * p * h * d * e + 4 * p * h + rows + index
    if not case['train']:
        return {'bytes': moved, 'flops': 4 * n * h * d}
    written = case['rows'] * kv * d * e * tables            # the table's gradient is whole
    return {'bytes': moved + 2 * p * h * d * e + written, 'flops': 14 * n * h * d}


# ---- the inputs ------------------------------------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device='cuda').manual_seed(int(seed))


def prepare(case, seed):
    g = _generator(seed)
    dev, dtype = 'cuda', DTYPES[case['dtype']]

    def normal(*shape):
        return torch.randn(shape, generator=g, device=dev)

    def uniform(*shape):
        return torch.rand(shape, generator=g, device=dev)

    if case['op'] == 'dropout':
        return {'case': case, 'x': normal(case['count']).to(dtype), 'seed': 0x9E3779B97F4A7C15 ^ int(seed), 'offset': int(seed) % 1000}

    if case['op'] == 'catalog':
        n, v, d = case['users'], case['items'], case['dim']
        item = normal(v, d)
        item = item / item.norm(dim=1, keepdim=True)
        target = (v * uniform(n) ** 2).to(torch.int64).clamp_(max=v - 1)          # popular items first
        user = item[target] + 2.0 * normal(n, d) / math.sqrt(d)                   # a user leans to what it chose
        user = user / user.norm(dim=1, keepdim=True)
        state = {'case': case, 'user': user.to(dtype), 'item': item.to(dtype), 'bias': None}
        if case['bias']:
            # minus the logarithm of how often an item is drawn; one in a hundred is not on offer, no target among them
            bias = 0.5 * torch.log((torch.arange(v, device=dev) + 1.0) / v)
            off = uniform(v) < 0.01
            off[target] = False
            state['bias'] = torch.where(off, torch.full_like(bias, -math.inf), bias)
        if case['train']:
            skip = uniform(n) < 0.05                                               # negative links teach nothing here
            skip[0] = False
            state['target'] = torch.where(skip, torch.full_like(target, -1), target).to(torch.int32)
            state['g_logp'] = -(0.5 + uniform(n)) / n
            state['g_entropy'] = -0.01 * uniform(n) / n
        return state

    p, h, kv, d, n, rows = (case[k] for k in ('parents', 'heads', 'kv', 'dim', 'edges', 'rows'))
    state = {'case': case, 'scale': 1.0 / math.sqrt(d), 'ids': None, 'indptr': None, 'offset': 0, 'v': None, 'inverse': None}
    state['q'] = normal(p, h, d).to(dtype)
    state['k'] = normal(rows, kv, d).to(dtype)
    if not case['shared']:
        state['v'] = normal(rows, kv, d).to(dtype)
    if not case['child']:                                   # popular parents first, the last ones often without neighbors
        parent = (p * uniform(n) ** 3).to(torch.int64).clamp_(max=p - 1)
        state['indptr'] = torch.cat([torch.zeros(1, dtype=torch.int64, device=dev),
                                     torch.bincount(parent, minlength=p).cumsum(0)])
    if case['ids']:
        state['offset'] = 1000
        row = (rows * uniform(n) ** 2).to(torch.int64).clamp_(max=rows - 1)
        none = uniform(n) < 0.01                            # a neighbor that is not there
        row = torch.where(none, torch.full_like(row, -1), row)
        state['ids'] = torch.where(none, row, row + 1000).to(torch.int32)
        if case['train']:
            # which edges read a row: the adjacency seen from the other side, kept with it
            order = torch.where(none, torch.full_like(row, rows), row)
            edges = torch.sort(order, stable=True)[1].to(torch.int32)
            ends = torch.bincount(order, minlength=rows + 1)[:rows].cumsum(0)
            state['inverse'] = (torch.cat([torch.zeros(1, dtype=torch.int64, device=dev), ends]), edges)
    if case['train']:
        state['g_out'] = normal(p, h, d).to(dtype)
    return state


# ---- one pass --------------------------------------------------------------------------------------------------------

def run(state):
    op = state['case']['op']
    if own:
        return {'attention': _own_attention, 'catalog': _own_catalog, 'dropout': _own_dropout}[op](state)
    return {'attention': _attention, 'catalog': _catalog, 'dropout': _dropout}[op](state)


def _own_attention(s):
    from graphsage_amd import kernels
    child = s['case']['child'] or None
    out, lse = kernels.neighbor_attention(s['q'], s['k'], s['v'], s['ids'], child, id_offset=s['offset'],
                                          scale=s['scale'], indptr=s['indptr'])
    if not s['case']['train']:
        return out, lse
    g_q, g_k, g_v = kernels.neighbor_attention_bwd(s['q'], s['k'], s['v'], s['ids'], child, out, lse, s['g_out'],
                                                   id_offset=s['offset'], scale=s['scale'], indptr=s['indptr'],
                                                   inverse=s['inverse'])
    return (out, lse, g_q, g_k) if g_v is None else (out, lse, g_q, g_k, g_v)


def _own_catalog(s):
    from graphsage_amd import kernels
    c = s['case']
    if not c['train']:
        r = kernels.catalog_log_probs(s['user'], s['item'], bias=s['bias'], scale=c['scale'], top_k=c['top'])
        return r.entropy, r.top_log_prob, r.top_ids
    r = kernels.catalog_log_probs(s['user'], s['item'], s['target'], s['bias'], c['scale'])
    g_user, g_item, g_bias = kernels.catalog_log_probs_bwd(s['user'], s['item'], s['target'], s['bias'], c['scale'], r.lse,
                                                           r.entropy, s['g_logp'], s['g_entropy'])
    return (r.log_prob, r.entropy, g_user, g_item) if g_bias is None else (r.log_prob, r.entropy, g_user, g_item, g_bias)


def _own_dropout(s):
    from graphsage_amd import kernels
    return kernels.dropout(s['x'], s['case']['rate'], s['seed'], s['offset'])


def _sums(x, ends, each=0):
    """Sums of x over runs of rows, in 64 bits: `each` rows a run, or runs that end where `ends` says (the first begins
    at ends[0]), as differences of a running sum, which in 64 bits loses nothing that 32 hold."""
    if each:
        return x.reshape((-1, each) + x.shape[1:]).sum(1, dtype=torch.float64)
    run = x.reshape(x.shape[0], -1).T.double().contiguous().cumsum(1)
    run = torch.cat([torch.zeros_like(run[:, :1]), run], 1)
    return (run[:, ends[1:]] - run[:, ends[:-1]]).T.reshape((-1,) + x.shape[1:])


def _attention(s):
    """out[p, h] = sum_e softmax_e(scale q[p, h] . k[row(e), h / (heads / kv)]) v[row(e), ...] over the edges e of parent
    p; an id outside the table is no neighbor; a parent without any gives zeros.  Gradients by the formula:
    ds = p (g_out . v - g_out . out).  Products in 32 bits; exponentials, which then need no shift, and sums over edges
    in 64."""
    c = s['case']
    p, h, kv, d, n, rows = (c[k] for k in ('parents', 'heads', 'kv', 'dim', 'edges', 'rows'))
    dev = s['q'].device
    edge = torch.arange(n, device=dev)
    if c['child']:
        ends, seg = None, edge // c['child']
    else:
        ends = s['indptr']
        seg = torch.repeat_interleave(torch.arange(p, device=dev), ends[1:] - ends[:-1], output_size=n)
    row = edge if s['ids'] is None else s['ids'].to(torch.int64) - s['offset']
    here = (row >= 0) & (row < rows)
    row = torch.where(here, row, torch.zeros_like(row))
    q = s['q'].float().reshape(p, kv, h // kv, d)
    keys = s['k'].float()[row].unsqueeze(2)                                        # [n, kv, 1, d]
    values = keys if s['v'] is None else s['v'].float()[row].unsqueeze(2)
    q_edge = q[seg]                                                                # [n, kv, h / kv, d]
    score = (q_edge * keys).sum(-1, keepdim=True) * s['scale']
    weight = torch.where(here[:, None, None, None], torch.exp(score.double()), torch.zeros_like(score, dtype=torch.float64))
    total = _sums(weight, ends, c['child'])
    lse = torch.log(total).float().reshape(p, h)
    total = torch.where(total > 0, total, torch.ones_like(total))
    prob = (weight / total[seg]).float()
    out = _sums(prob * values, ends, c['child']).float()
    result = out.reshape(p, h, d).to(s['q'].dtype)
    if not c['train']:
        return result, lse
    g = s['g_out'].float().reshape(p, kv, h // kv, d)
    delta = (g * result.float().reshape(p, kv, h // kv, d)).sum(-1, keepdim=True)
    g_edge = g[seg]
    ds = prob * ((g_edge * values).sum(-1, keepdim=True) - delta[seg]) * s['scale']
    g_q = _sums(ds * keys, ends, c['child']).reshape(p, h, d).to(s['q'].dtype)

    def of_rows(x):                                         # sums over the edges that read a row
        return (x if s['inverse'] is None else _sums(x[s['inverse'][1].to(torch.int64)], s['inverse'][0])).to(s['k'].dtype)

    to_key, to_value = (ds * q_edge).sum(2), (prob * g_edge).sum(2)
    if s['v'] is None:
        return result, lse, g_q, of_rows(to_key + to_value)
    return result, lse, g_q, of_rows(to_key), of_rows(to_value)


def _catalog(s):
    """z = scale user . item + bias over all items; log_prob = z[target] - logsumexp(z), entropy = -sum p log p (a
    target outside the catalog: 0), the best items by z (in 64 bits), the lowest index first where two are equal.
    Gradients by the formula: dz_j = g_logp ([j is the target] - p_j) - g_entropy p_j (log p_j + entropy)."""
    c = s['case']
    wide = torch.float32 if c['train'] else torch.float64         # ranks hang on the last bits of z
    user, item = s['user'].to(wide), s['item'].to(wide)
    z = user @ item.T * c['scale']
    if s['bias'] is not None:
        z = z + s['bias'].to(wide)
    most = z.amax(1, keepdim=True)
    lse = most + torch.log(torch.exp(z - most).sum(1, keepdim=True))
    log_p = z - lse
    p = torch.exp(log_p)
    p_log_p = p * torch.where(p > 0, log_p, torch.zeros_like(p))
    entropy = -p_log_p.sum(1)
    if not c['train']:
        best, at = torch.sort(log_p, dim=1, descending=True, stable=True)
        best, at = best[:, :c['top']], at[:, :c['top']]
        at = torch.where(best == -math.inf, torch.full_like(at, -1), at)
        return entropy.float(), best.float(), at.to(torch.int32)
    target = s['target'].to(torch.int64)
    there = target >= 0
    hit = (torch.arange(c['items'], device=z.device)[None, :] == target[:, None])
    log_prob = torch.where(there, log_p.gather(1, target.clamp(min=0)[:, None])[:, 0], torch.zeros_like(entropy))
    g_logp = torch.where(there, s['g_logp'], torch.zeros_like(s['g_logp']))[:, None]
    dz = g_logp * (hit.float() - p) - s['g_entropy'][:, None] * (p_log_p + p * entropy[:, None])
    g_user = (dz @ item * c['scale']).to(s['user'].dtype)
    g_item = (dz.T @ user * c['scale']).to(s['item'].dtype)
    if s['bias'] is None:
        return log_prob, entropy, g_user, g_item
    return log_prob, entropy, g_user, g_item, dz.sum(0)


def _philox(block, key):
    """Four words of Philox4x32-10 at counters (low half, high half of block, 0x50000000, 0), in whole torch numbers."""
    low = 0xFFFFFFFF
    c = [block & low, (block >> 32) & low, torch.full_like(block, 0x50000000), torch.zeros_like(block)]
    k0, k1 = key & low, (key >> 32) & low
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57           # products modulo 2^64
        c = [((b >> 32) & low) ^ c[1] ^ k0, b & low, ((a >> 32) & low) ^ c[3] ^ k1, a & low]
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return c


def _dropout(s):
    """Element i is kept where the 16-bit piece i % 8 of Philox block offset + i / 8 is not below floor(rate 2^16);
    what is kept is divided by the share that is kept."""
    x, threshold = s['x'], int(s['case']['rate'] * 65536)
    n = x.numel()
    block = torch.arange((n + 7) // 8, device=x.device) + s['offset']
    words = torch.stack(_philox(block, s['seed']), dim=1)
    pieces = torch.stack([words & 0xFFFF, words >> 16], dim=2).reshape(-1)[:n]
    scaled = x.float() * (65536.0 / (65536 - threshold))
    return torch.where(pieces >= threshold, scaled, torch.zeros_like(scaled)).to(x.dtype)


# ---- the same from the definitions, in 64 bits -------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {'attention': _exact_attention, 'catalog': _exact_catalog, 'dropout': _exact_dropout}[case['op']](s)


def _exact_attention(s):
    """Head by head: weights are plain exponentials over their sum (64 bits hold them), gradients are autograd's."""
    c = s['case']
    p, n, train = c['parents'], c['edges'], c['train']
    dev = s['q'].device
    if c['child']:
        ends = torch.arange(1, p + 1, device=dev) * c['child']
    else:
        ends = s['indptr'][1:]
    seg = torch.bucketize(torch.arange(n, device=dev), ends, right=True)
    row = torch.arange(n, device=dev) if s['ids'] is None else s['ids'].long() - s['offset']
    kept = torch.nonzero((row >= 0) & (row < c['rows']))[:, 0]
    seg, row = seg[kept], row[kept]
    ends = torch.searchsorted(kept, ends)                         # where a parent's kept edges end
    q, k = s['q'].double().requires_grad_(train), s['k'].double().requires_grad_(train)
    v = k if s['v'] is None else s['v'].double().requires_grad_(train)
    outs, lses = [], []
    for h in range(c['heads']):
        j = h // (c['heads'] // c['kv'])
        e = torch.exp(s['scale'] * (q[seg, h] * k[row, j]).sum(1))
        sums = torch.cumsum(torch.cat([e[:, None], e[:, None] * v[row, j]], 1), 0)
        sums = torch.cat([torch.zeros_like(sums[:1]), sums])[ends]
        sums = torch.diff(sums, dim=0, prepend=torch.zeros_like(sums[:1]))
        total, o = sums[:, 0], sums[:, 1:]
        outs.append(o / torch.where(total > 0, total, torch.ones_like(total))[:, None])      # without neighbors: zeros
        lses.append(torch.log(total))
    out, lse = torch.stack(outs, 1), torch.stack(lses, 1)
    if not train:
        return out, lse
    leaves = [q, k] if s['v'] is None else [q, k, v]
    return (out.detach(), lse.detach()) + torch.autograd.grad((out * s['g_out'].double()).sum(), leaves)


def _exact_catalog(s):
    c = s['case']
    user, item = s['user'].double().requires_grad_(), s['item'].double().requires_grad_()
    bias = torch.zeros(c['items'], dtype=torch.float64, device=user.device) if s['bias'] is None else s['bias'].double()
    on = torch.nonzero(bias > -math.inf)[:, 0]                    # items that are on offer
    free = bias[on].requires_grad_()
    with torch.set_grad_enabled(c['train']):
        z = c['scale'] * (user @ item[on].T) + free
        log_p = z - torch.logsumexp(z, 1, keepdim=True)
        entropy = -(torch.exp(log_p) * log_p).sum(1)
    if not c['train']:
        n, top = c['users'], c['top']
        values = torch.full((n, top), -math.inf, dtype=torch.float64, device=z.device)
        ids = torch.full((n, top), -1, dtype=torch.int32, device=z.device)
        left, at = log_p.detach().clone(), torch.arange(len(on), device=z.device)
        for r in range(min(top, len(on))):
            values[:, r] = left.amax(1)
            first = torch.where(left == values[:, r:r + 1], at, len(on)).amin(1)
            ids[:, r] = on[first].to(torch.int32)
            left.scatter_(1, first[:, None], -math.inf)
        return entropy, values, ids
    where = torch.searchsorted(on, s['target'].long().clamp(min=0))
    chosen = torch.where(s['target'] >= 0, log_p[torch.arange(len(where), device=z.device), where.clamp(max=len(on) - 1)], 0.0)
    total = (chosen * s['g_logp'].double()).sum() + (entropy * s['g_entropy'].double()).sum()
    g_user, g_item, g_free = torch.autograd.grad(total, [user, item, free])
    result = (chosen.detach(), entropy.detach(), g_user, g_item)
    return result if s['bias'] is None else result + (torch.zeros_like(bias).index_put((on,), g_free),)


def _exact_dropout(s):
    """On the host, in unsigned numbers of 64 bits."""
    n, u = s['x'].numel(), np.uint64
    threshold = math.floor(s['case']['rate'] * 65536)
    count = (n + 7) // 8
    counter = np.arange(count, dtype=u) + u(s['offset'])
    x0, x1, x2, x3 = counter & u(0xFFFFFFFF), counter >> u(32), np.full(count, 0x50000000, u), np.zeros(count, u)
    for r in range(10):
        k0 = u(((s['seed'] & 0xFFFFFFFF) + r * 0x9E3779B9) & 0xFFFFFFFF)
        k1 = u(((s['seed'] >> 32) + r * 0xBB67AE85) & 0xFFFFFFFF)
        m0, m1 = x0 * u(0xD2511F53), x2 * u(0xCD9E8D57)
        x0, x1, x2, x3 = (m1 >> u(32)) ^ x1 ^ k0, m1 & u(0xFFFFFFFF), (m0 >> u(32)) ^ x3 ^ k1, m0 & u(0xFFFFFFFF)
    halves = np.stack([x0, x1, x2, x3], 1).astype('<u4').view('<u2').reshape(-1)[:n]
    keep = torch.from_numpy(halves >= threshold).to(s['x'].device)
    return s['x'].double() * keep * (65536.0 / (65536 - threshold))
