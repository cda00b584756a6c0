"""Attention over neighbors and its gradients against the formulas in 64 bits -- needs a GPU.

Tolerances are bounds on the rounding, element by element.  With u = 2^-24 (fp32), a score is a sum of dim products and
is off by at most ds = (dim + 4) u scale sum |q k|; a probability then by a share r = 2 max ds + (n + 16) u (numerator,
denominator and the sum over n edges); a result of type t is rounded by at most eps_t / 2 of itself.  ``delta`` is taken
from the rounded output, which adds eps_t / 2 sum |g_out| |out| to every <g_out, v> - delta."""
import math

import pytest
import torch

from graphsage_amd import _lib, autograd, kernels

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _case(seed, dtype, parents, heads, kv, dim, rows, child=None, lengths=None, ids=True, offset=0, masked=0.1, shared=False,
          unaligned=False):
    g = torch.Generator(device='cuda').manual_seed(seed)

    def normal(*shape):
        n = math.prod(shape)
        if unaligned:                                 # contiguous, one element behind a 16-byte border
            return torch.randn(n + 1, generator=g, device='cuda').to(dtype)[1:].reshape(shape)
        return torch.randn(shape, generator=g, device='cuda').to(dtype)
    indptr = None
    if lengths is not None:
        indptr = torch.cat([torch.zeros(1, dtype=torch.int64), torch.as_tensor(lengths, dtype=torch.int64).cumsum(0)]).cuda()
        edges = int(indptr[-1])
    else:
        edges = parents * child
    child_ids = None
    if ids:
        row = torch.randint(0, max(rows, 1), (edges,), generator=g, device='cuda')
        gone = torch.rand(edges, generator=g, device='cuda') < masked
        child_ids = torch.where(gone, torch.full_like(row, -5), row + offset).to(torch.int32)
    q, k, go = normal(parents, heads, dim), normal(rows, kv, dim), normal(parents, heads, dim)
    v = None if shared else normal(rows, kv, dim)
    return dict(q=q, k=k, v=v, go=go, child_ids=child_ids, child=child, indptr=indptr, offset=offset, edges=edges)


def _reference(c, scale, out=None):
    """Everything in 64 bits, with the bounds: out, lse, g_q, g_k, g_v and a tolerance for each."""
    q, k, go = c['q'].double(), c['k'].double(), c['go'].double()
    v = k if c['v'] is None else c['v'].double()
    (p, h, d), (rows, kv, _), n = q.shape, k.shape, c['edges']
    dev, half = q.device, torch.finfo(c['q'].dtype).eps / 2
    if c['indptr'] is None:
        seg = torch.arange(p, device=dev).repeat_interleave(c['child'])
    else:
        seg = torch.arange(p, device=dev).repeat_interleave(c['indptr'].diff())
    row = torch.arange(n, device=dev) if c['child_ids'] is None else c['child_ids'].reshape(-1).long() - c['offset']
    ok = (row >= 0) & (row < rows)
    seg, row = seg[ok], row[ok]
    head = torch.arange(h, device=dev) // (h // kv)
    ke, ve, qe, ge = k[row][:, head], v[row][:, head], q[seg], go[seg]         # [n, h, d]
    s = (qe * ke).sum(-1) * scale

    def sums(x):
        return torch.zeros((p,) + x.shape[1:], dtype=torch.float64, device=dev).index_add_(0, seg, x)
    top = torch.full((p, h), -math.inf, dtype=torch.float64, device=dev).scatter_reduce_(0, seg[:, None].expand(-1, h), s, 'amax')
    w = torch.exp(s - top[seg])
    tot = sums(w)
    prob = w / tot[seg]
    lse = top + torch.log(tot)
    o = sums(prob[..., None] * ve)
    count = torch.zeros(p, device=dev, dtype=torch.float64).index_add_(0, seg, torch.ones_like(seg, dtype=torch.float64))
    ds = torch.zeros((p, h), dtype=torch.float64, device=dev).scatter_reduce_(
        0, seg[:, None].expand(-1, h), (d + 4) * U * scale * (qe * ke).abs().sum(-1), 'amax')
    r = 2 * ds + (count[:, None] + 16) * U
    spread = sums(prob[..., None] * ve.abs())
    tol_out = half * o.abs() + r[..., None] * spread + 1e-30
    tol_lse = ds + (count[:, None] + 16) * U + 4 * U * lse.abs().nan_to_num(posinf=0, neginf=0) + 1e-30
    # gradients
    delta = (go * o).sum(-1)
    gap = (ge * ve).sum(-1) - delta[seg]
    dscore = prob * gap * scale
    off = prob * scale * (r[seg] * gap.abs() + (d + 4) * U * ((ge * ve).abs().sum(-1) + (go * o).abs().sum(-1)[seg])
                          + (go.abs() * tol_out).sum(-1)[seg])
    g_q = sums(dscore[..., None] * ke)
    tol_q = half * g_q.abs() + sums((off + (count[seg][:, None] + 4) * U * dscore.abs())[..., None] * ke.abs()) + 1e-30
    reads = torch.zeros(max(rows, 1), device=dev, dtype=torch.float64).index_add_(0, row, torch.ones_like(row, dtype=torch.float64))[:rows] * (h // kv)

    def of_rows(x):
        return torch.zeros((rows, kv, d), dtype=torch.float64, device=dev).index_add_(0, row, x.reshape(-1, kv, h // kv, d).sum(2))
    g_k, g_v = of_rows(dscore[..., None] * qe), of_rows(prob[..., None] * ge)
    many = (reads[:, None, None] + 8) * U
    tol_k = of_rows(off[..., None] * qe.abs()) + many * of_rows(dscore.abs()[..., None] * qe.abs())
    tol_v = of_rows((r[seg] * prob)[..., None] * ge.abs()) + many * of_rows(prob[..., None] * ge.abs())
    if c['v'] is None:
        g_k, tol_k, g_v, tol_v = g_k + g_v, tol_k + tol_v, None, None
        tol_k = tol_k + half * g_k.abs() + 1e-30
    else:
        tol_k, tol_v = tol_k + half * g_k.abs() + 1e-30, tol_v + half * g_v.abs() + 1e-30
    return dict(out=(o, tol_out), lse=(lse, tol_lse), g_q=(g_q, tol_q), g_k=(g_k, tol_k), g_v=(g_v, tol_v))


def _near(name, got, want):
    want, tol = want
    if got.dtype == torch.float16:                    # results below the normal range of fp16 keep fewer bits
        tol = tol + 2.0 ** -25
    got = got.double()
    assert got.shape == want.shape, name
    finite = torch.isfinite(want)
    assert torch.equal(got[~finite], want[~finite]), name
    off = ((got - want).abs() / tol)[finite]
    assert off.numel() == 0 or float(off.max()) <= 1.0, "%s: %.3g times the bound" % (name, float(off.max()))


def _check(c, scale=None):
    d = c['q'].shape[-1]
    s = d ** -0.5 if scale is None else scale
    want = _reference(c, s)
    out, lse = kernels.neighbor_attention(c['q'], c['k'], c['v'], c['child_ids'], c['child'], c['offset'], scale, c['indptr'])
    _near('out', out, want['out'])
    _near('lse', lse, want['lse'])
    g_q, g_k, g_v = kernels.neighbor_attention_bwd(c['q'], c['k'], c['v'], c['child_ids'], c['child'], out, lse, c['go'], c['offset'],
                                                   scale, c['indptr'])
    _near('g_q', g_q, want['g_q'])
    _near('g_k', g_k, want['g_k'])
    assert (g_v is None) == (c['v'] is None)
    if g_v is not None:
        _near('g_v', g_v, want['g_v'])
    return out, lse, g_q, g_k, g_v


DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('dim', [1, 3, 8, 16, 24, 33, 64, 100, 128, 200, 256])
def test_widths(cuda, dtype, dim):
    for unaligned in (False, True):
        _check(_case(dim, dtype, 37, 2, 1, dim, 50, child=9, offset=100, unaligned=unaligned))
        _check(_case(dim, dtype, 11, 2, 2, dim, 40, lengths=[0, 3, 0, 0, 40, 1, 0, 150, 7, 0, 0], unaligned=unaligned, shared=True))


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('heads,kv', [(1, 1), (2, 1), (3, 1), (4, 2), (5, 1), (6, 6), (9, 3), (16, 2)])
def test_head_layouts(cuda, dtype, heads, kv):
    for shared in (False, True):
        _check(_case(heads * 10 + kv, dtype, 23, heads, kv, 32, 61, child=6, shared=shared))
        _check(_case(heads * 10 + kv, dtype, 5, heads, kv, 20, 300, lengths=[0, 100, 37, 0, 163], ids=False, shared=shared))


@pytest.mark.parametrize('child', [0, 1, 2, 7, 8, 9, 25, 32, 33, 64, 300])
@pytest.mark.parametrize('ids', [True, False])
def test_lengths_of_one_kind(cuda, child, ids):
    for parents in (1, 2, 65, 700):
        rows = 90 if ids else parents * child + 3     # dense: three rows behind the last group
        _check(_case(child, torch.float32, parents, 2, 1, 64, rows, child=child, ids=ids, shared=True))


@pytest.mark.parametrize('dtype', DTYPES)
def test_ragged_lengths_from_none_to_long(cuda, dtype):
    lengths = [0, 0, 5000, 1, 0, 8, 64, 7, 9, 0, 2000, 3] + [0] * 200 + [1] * 130 + [0, 17]
    _check(_case(3, dtype, len(lengths), 4, 2, 64, 1000, lengths=lengths))
    _check(_case(4, dtype, len(lengths), 2, 2, 33, 3, lengths=lengths, shared=True))    # three rows take all edges
    _check(_case(5, dtype, len(lengths), 1, 1, 128, sum(lengths), lengths=lengths, ids=False))


def test_many_short_parents_and_one_long_list(cuda):
    _check(_case(6, torch.float32, 40000, 1, 1, 16, 500, child=3, shared=True))
    _check(_case(7, torch.float32, 1, 4, 1, 64, 1000, child=20001, shared=True))
    _check(_case(8, torch.bfloat16, 1, 8, 2, 64, 30000, child=30000, ids=False))
    _check(_case(9, torch.float32, 3, 1, 1, 256, 700, lengths=[30000, 0, 9]))


def test_parents_whose_neighbors_are_all_masked(cuda):
    c = _case(10, torch.float32, 20, 2, 1, 32, 30, child=12, shared=True)
    ids = c['child_ids'].reshape(20, 12)
    ids[3], ids[19], ids[0] = -1, 30, 2 ** 31 - 1     # below, behind, far behind the table
    out, lse, g_q, g_k, _ = _check(c)
    for p in (3, 19, 0):
        assert not out[p].any() and bool((lse[p] == -math.inf).all()) and not g_q[p].any()
    c['child_ids'].fill_(-1)
    out, lse, g_q, g_k, _ = _check(c)
    assert not out.any() and not g_q.any() and not g_k.any()
    _check(_case(11, torch.float32, 4, 1, 1, 8, 0, child=5))                            # a table without rows
    _check(_case(12, torch.float32, 0, 1, 1, 8, 9, child=5))                            # no parents
    _check(_case(12, torch.float32, 3, 1, 1, 8, 9, lengths=[0, 0, 0]))
    none = _case(12, torch.float32, 0, 1, 1, 8, 9, lengths=[])                          # entries that belong to nobody
    none['child_ids'] = torch.arange(7, dtype=torch.int32, device='cuda')
    g_k = kernels.neighbor_attention_bwd(none['q'], none['k'], none['v'], none['child_ids'], None, none['q'],
                                         torch.zeros((0, 1), device='cuda'), none['go'], indptr=none['indptr'])[1]
    assert not g_k.any()


def test_rows_that_are_no_neighbors_may_hold_anything(cuda):
    for lengths in (None, [0, 300, 2, 98, 0]):
        c = _case(13, torch.float32, 40 if lengths is None else 5, 2, 1, 32, 60, child=None if lengths else 10, lengths=lengths, shared=True)
        want = _check(c)
        used = torch.zeros(60, dtype=torch.bool, device='cuda')
        row = c['child_ids'].reshape(-1).long()
        row[(row == 7) | (row == 8)] = -1
        c['child_ids'] = row.to(torch.int32)
        want = _check(c)
        used[row[row >= 0]] = True
        c['k'][7], c['k'][8] = math.nan, math.inf
        out, lse = kernels.neighbor_attention(c['q'], c['k'], None, c['child_ids'], c['child'], 0, None, c['indptr'])
        grads = kernels.neighbor_attention_bwd(c['q'], c['k'], None, c['child_ids'], c['child'], out, lse, c['go'], 0, None, c['indptr'])
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1]) and torch.equal(grads[0], want[2])
        assert torch.equal(grads[1][used], want[3][used]) and not grads[1][~used].any()


def test_scores_far_apart_and_far_from_zero(cuda):
    c = _case(14, torch.float32, 30, 1, 1, 16, 40, child=20, shared=True)
    for scale in (1e-6, 30.0):
        _check(c, scale)
    c['q'] *= 40
    _check(c, 1.0)


def test_dense_rows_behind_the_last_neighborhood_are_left_alone(cuda):
    c = _case(15, torch.float32, 4, 1, 1, 8, 30, lengths=[3, 0, 5, 6], ids=False, masked=0)
    c['indptr'] += 2                                  # rows 0, 1 and 16.. belong to nobody
    out, lse = kernels.neighbor_attention(c['q'], c['k'], c['v'], None, None, indptr=c['indptr'])
    g_k, g_v = torch.full_like(c['k'], 7.0), torch.full_like(c['k'], 7.0)
    kernels.neighbor_attention_bwd(c['q'], c['k'], c['v'], None, None, out, lse, c['go'], indptr=c['indptr'], g_k=g_k, g_v=g_v)
    outside = torch.ones(30, dtype=torch.bool, device='cuda')
    outside[2:16] = False
    for g in (g_k, g_v):
        assert bool((g[outside] == 7.0).all()) and not bool((g[~outside] == 7.0).any())
    c['k'], c['v'] = c['k'][2:16].contiguous(), c['v'][2:16].contiguous()
    c['indptr'] -= 2
    c['edges'] = 14
    want = _reference(c, 8 ** -0.5)                   # edges are dealt from another start: other bits, the same bounds
    _near('g_k', g_k[2:16], want['g_k'])
    _near('g_v', g_v[2:16], want['g_v'])


def test_a_table_longer_than_32_bits_of_elements(cuda):
    rows = (1 << 31) // 256 + 1000                    # 2.1e9 elements of 16 bits
    k = torch.zeros((rows, 1, 256), dtype=torch.bfloat16, device='cuda')
    g = torch.Generator(device='cuda').manual_seed(2)
    tail = torch.randn((900, 1, 256), generator=g, device='cuda').to(torch.bfloat16)
    k[-900:] = tail
    c = _case(16, torch.bfloat16, 9, 1, 1, 256, 900, child=20, shared=True, masked=0)
    small = kernels.neighbor_attention(c['q'], tail, None, c['child_ids'], 20)
    big = kernels.neighbor_attention(c['q'], k, None, c['child_ids'], 20, id_offset=-(rows - 900))
    assert torch.equal(small[0], big[0]) and torch.equal(small[1], big[1])


def test_results_repeat_and_do_not_depend_on_what_memory_held(cuda):
    lengths = [0, 3000, 5, 77, 0, 900]
    c = _case(17, torch.float32, 6, 2, 1, 40, 100, lengths=lengths)
    first = _check(c)
    junk = torch.full((1 << 24,), float('nan'), device='cuda')
    del junk                                          # the allocator hands this memory to the next workspaces
    again = _check(c)
    for a, b in zip(first, again):
        assert torch.equal(a, b)


def test_autograd_gives_the_gradients_of_differences(cuda):
    c = _case(18, torch.float32, 12, 2, 1, 6, 15, child=5)
    leaves = [c['q'].clone().requires_grad_(), c['k'].clone().requires_grad_(), c['v'].clone().requires_grad_()]
    out, _ = autograd.NeighborAttention.apply(*leaves, c['child_ids'], 5, 0, None, None, None)
    (out * c['go']).sum().backward()

    def loss(q, k, v):                                # the definition, in 64 bits
        x = dict(c, q=q, k=k, v=v)
        return float((_reference(x, 6 ** -0.5)['out'][0] * c['go'].double()).sum())
    base = [t.detach().double() for t in leaves]
    g = torch.Generator(device='cuda').manual_seed(1)
    for i in range(3):
        for _ in range(4):
            step = torch.randn(base[i].shape, generator=g, device='cuda', dtype=torch.float64)
            args = lambda t: [b + t * step if j == i else b for j, b in enumerate(base)]
            eps = 1e-5
            slope = (loss(*args(eps)) - loss(*args(-eps))) / (2 * eps)
            got = float((leaves[i].grad.double() * step).sum())
            # central differences are off by eps^2 times a third derivative (about 1e-8 here), fp32 by u per term
            assert abs(got - slope) <= 1e-5 * (leaves[i].grad.double() * step).abs().sum() + 1e-7


def test_autograd_leaves_out_what_needs_no_gradient(cuda):
    c = _case(19, torch.float32, 12, 2, 1, 8, 15, child=5, shared=True)
    q = c['q'].clone().requires_grad_()
    out, lse = autograd.NeighborAttention.apply(q, c['k'], None, c['child_ids'], 5, 0, None, None, None)
    assert not lse.requires_grad
    out.backward(c['go'])
    assert torch.equal(q.grad, _check(c)[2])
    k = c['k'].clone().requires_grad_()
    out, _ = autograd.NeighborAttention.apply(c['q'], k, None, c['child_ids'], 5, 0, None, None, None)
    out.backward(c['go'])
    assert torch.equal(k.grad, _check(c)[3])


def test_on_another_stream_and_in_a_replayed_graph(cuda):
    lengths = [0, 700, 5, 77, 0, 200]
    c = _case(20, torch.float32, 6, 2, 1, 64, 100, lengths=lengths, shared=True)
    want = _check(c)
    inverse = kernels.neighbor_inverse(c['child_ids'], 100)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out, lse = kernels.neighbor_attention(c['q'], c['k'], None, c['child_ids'], None, indptr=c['indptr'])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want[0])

    def body():
        o, s = kernels.neighbor_attention(c['q'], c['k'], None, c['child_ids'], None, indptr=c['indptr'])
        return (o, s) + kernels.neighbor_attention_bwd(c['q'], c['k'], None, c['child_ids'], None, o, s, c['go'],
                                                       indptr=c['indptr'], inverse=inverse)[:2]
    graphs, results = [], []
    for _ in range(2):                                # two graphs with workspaces of their own
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            results.append(body())
        graphs.append(g)
    for k in range(3):
        c['q'].add_(0.25)                             # new inputs in place
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = body()
        for res in results:
            for a, b in zip(res, want):
                assert torch.equal(a, b)
    with pytest.raises(_lib.GsageError, match='capture'):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            kernels.neighbor_inverse(c['child_ids'], 100)


def test_inverse_lists(cuda):
    ids = torch.tensor([5, 9, 5, -1, 12, 6, 5, 100, 4], dtype=torch.int32, device='cuda')
    indptr, edges = kernels.neighbor_inverse(ids, 6, 4)          # rows 0 .. 5 are ids 4 .. 9
    assert indptr.tolist() == [0, 1, 4, 5, 5, 5, 6] and edges.tolist() == [8, 0, 2, 6, 5, 1, 3, 4, 7]
    indptr, edges = kernels.neighbor_inverse(ids[:0], 3)
    assert indptr.tolist() == [0, 0, 0, 0] and edges.numel() == 0


def test_refusals(cuda):
    z = lambda *s, t=torch.float32: torch.zeros(s, dtype=t, device='cuda')
    q, k, ids = z(4, 2, 8), z(10, 1, 8), z(12, t=torch.int32)
    ok = kernels.neighbor_attention(q, k, None, ids, 3)
    for bad, err in [
            (lambda: kernels.neighbor_attention(q.cpu(), k, None, ids, 3), _lib.GsageError),
            (lambda: kernels.neighbor_attention(q.double(), k.double(), None, ids, 3), TypeError),
            (lambda: kernels.neighbor_attention(q, k.half(), None, ids, 3), TypeError),
            (lambda: kernels.neighbor_attention(q, k, k.half(), ids, 3), TypeError),
            (lambda: kernels.neighbor_attention(q[:, :, ::2], k[:, :, ::2], None, ids, 3), ValueError),
            (lambda: kernels.neighbor_attention(q[0], k, None, ids, 3), ValueError),
            (lambda: kernels.neighbor_attention(q, z(10, 1, 9), None, ids, 3), ValueError),
            (lambda: kernels.neighbor_attention(z(4, 3, 8), z(10, 2, 8), None, ids, 3), ValueError),
            (lambda: kernels.neighbor_attention(q, k, z(9, 1, 8), ids, 3), ValueError),
            (lambda: kernels.neighbor_attention(q, k, None, ids, 4), ValueError),
            (lambda: kernels.neighbor_attention(q, k, None, ids.long(), 3), TypeError),
            (lambda: kernels.neighbor_attention(q, k, None, None, 3), ValueError),
            (lambda: kernels.neighbor_attention(q, k, None, ids, None), ValueError),
            (lambda: kernels.neighbor_attention(q, k, None, ids, 3, indptr=z(5, t=torch.int64)), ValueError),
            (lambda: kernels.neighbor_attention(q, k, None, ids, None, indptr=z(4, t=torch.int64)), ValueError),
            (lambda: kernels.neighbor_attention(z(4, 2, 257), z(10, 1, 257), None, ids, 3), _lib.GsageError),
            (lambda: kernels.neighbor_attention(q, k, None, ids, 3, out=z(4, 2, 9)), ValueError),
            (lambda: kernels.neighbor_attention(q, k, None, ids, 3, lse=z(4, 3)), ValueError),
            (lambda: kernels.neighbor_attention_bwd(q, k, None, ids, 3, ok[0], ok[1], z(4, 2, 7)), ValueError),
            (lambda: kernels.neighbor_attention_bwd(q, k, None, ids, 3, ok[0], ok[1], q, inverse=(z(10, t=torch.int64), ids)), ValueError),
            (lambda: kernels.neighbor_attention_bwd(q, k, None, ids, 3, ok[0], ok[1], q,
                                                    inverse=(z(11, t=torch.int64), z(13, t=torch.int32))), ValueError)]:
        with pytest.raises(err):
            bad()


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('heads,kv,dim,shared', [(1, 1, 64, True), (2, 1, 33, False), (5, 1, 100, True), (6, 3, 8, False), (4, 4, 256, True),
                                                 (3, 1, 3, False), (1, 1, 1, True)])
def test_gradients_of_many_rows_that_few_read(cuda, dtype, heads, kv, dim, shared):
    """Lists of rows that are short on the mean: empty, of one entry, and a few read by so many that they are cut."""
    c = _case(21, dtype, 600, heads, kv, dim, 3000, child=11, masked=0.05, shared=shared, offset=7)
    ids = c['child_ids']
    ids[::3] = torch.where(ids[::3] >= 0, 7 + 1234, ids[::3])         # row 1234: 2000 entries
    ids[1::30] = 7 + 2999                                             # the last row: 220
    _check(c)
    lengths = torch.randint(0, 12, (500,), generator=torch.Generator().manual_seed(5)).tolist()
    _check(_case(22, dtype, 500, heads, kv, dim, 9000, lengths=lengths, shared=shared))


def test_edges_outside_the_lists_count_nowhere(cuda):
    """child_ids may hold more than the lists of indptr name, on either side."""
    for rows in (60, 4000):                                           # long and short lists of the rows
        c = _case(23, torch.float32, 40, 2, 1, 64, rows, lengths=[30, 0, 700] + [5] * 37)
        whole = _check(c)
        more = lambda n, s: torch.randint(0, rows, (n,), generator=torch.Generator(device='cuda').manual_seed(s), device='cuda').to(torch.int32)
        ids = torch.cat([more(333, 1), c['child_ids'], more(3000, 2)])
        indptr = c['indptr'] + 333
        out, lse = kernels.neighbor_attention(c['q'], c['k'], c['v'], ids, None, 0, None, indptr)
        junk = torch.zeros(64 << 20, dtype=torch.uint8, device='cuda')        # what a workspace may find: parent 0 everywhere
        del junk
        g_q, g_k, g_v = kernels.neighbor_attention_bwd(c['q'], c['k'], c['v'], ids, None, out, lse, c['go'], 0, None, indptr)
        want = _reference(c, 64 ** -0.5)
        for name, got in zip(('out', 'lse', 'g_q', 'g_k', 'g_v'), (out, lse, g_q, g_k, g_v)):
            _near(name, got, want[name])
        assert len(whole) == 5


@pytest.mark.parametrize('n', [1, 511, 513, 2000, 40000])
def test_every_row_of_a_table_gets_its_gradient(cuda, n):
    """Counts around the borders of how lists are shared out to be joined: all rows empty but the first and the last."""
    k = torch.randn(n, 1, 16, device='cuda')
    q = torch.randn(3, 1, 16, device='cuda')
    ids = torch.tensor([0, n - 1, 0, n - 1, -1, 0], dtype=torch.int32, device='cuda')
    out, lse = kernels.neighbor_attention(q, k, None, ids, 2)
    g_k = torch.full_like(k, 7.0)
    kernels.neighbor_attention_bwd(q, k, None, ids, 2, out, lse, torch.ones_like(q), g_k=g_k)
    c = dict(q=q, k=k, v=None, go=torch.ones_like(q), child_ids=ids, child=2, indptr=None, offset=0, edges=6)
    _near('g_k', g_k, _reference(c, 0.25)['g_k'])


@pytest.mark.parametrize('rows', [40, 4000])
def test_inverse_lists_that_are_part_of_larger_ones(cuda, rows):
    """Entries before the first row's list and behind the last one's are no row's, whatever they name."""
    c = _case(24, torch.float32, 300, 2, 1, 32, rows, child=6)
    out, lse = kernels.neighbor_attention(c['q'], c['k'], c['v'], c['child_ids'], 6)
    indptr, edges = kernels.neighbor_inverse(c['child_ids'], rows)
    n = int(indptr[-1])
    moved = torch.cat([edges[50:150], edges[:n], edges[:30]])
    args = (c['q'], c['k'], c['v'], c['child_ids'], 6, out, lse, c['go'])
    g_q, g_k, g_v = kernels.neighbor_attention_bwd(*args, inverse=(indptr + 100, moved))
    want = _reference(c, 32 ** -0.5)
    for name, got in (('g_q', g_q), ('g_k', g_k), ('g_v', g_v)):
        _near(name, got, want[name])


@pytest.mark.parametrize('heads,kv', [(1, 1), (2, 1), (4, 1), (6, 2)])
@pytest.mark.parametrize('child,dim,dtype', [(13, 64, torch.float32), (20, 3, torch.float32), (32, 16, torch.bfloat16), (25, 33, torch.float16),
                                             (21, 32, torch.float32)])
def test_many_lists_of_one_length(cuda, heads, kv, child, dim, dtype):
    """Enough lists that several share a wave, of lengths around where that begins and ends."""
    for ids in (True, False):
        _check(_case(25, dtype, 8195, heads, kv, dim, 900 if ids else 8195 * child, child=child, ids=ids, shared=dim != 33))
