"""Log probabilities, entropy and best items over a catalog, and their gradients, against the formulas in 64 bits --
needs a GPU.

Tolerances bound the rounding.  u = 2^-24.  A score is a sum of at most 6 * 256 exact piece products, each addition off by at
most 2 u of sum |user| |item|, what the pieces leave out below 4 u of it: ez = scale (6 width + 16) 2 u sum |user| |item| +
8 u |z|, width the padded width.  A sum of exponentials adds at most 256 terms one after the other in any lane at these
sizes: T = 256 u.  Gradients: an element of dz (the target's own term apart) is cut into bf16 pieces, piece i at most 2^-8i of it, and
products of pieces i and k of dz and the table's element count for i + k < n.  bf16 tables, n = 1: off by 2^-8 of the
product.  fp16, n = 2: 2^-16 of dz left, 2^-16 for the product left out, together below 2^-14.  fp32, n = 3: nothing
left, products 1-2, 2-1 and 2-2 left out, 2^-24 + 2^-24 + 2^-32, below 2^-22."""
import math

import pytest
import torch

from graphsage_amd import _lib, autograd, kernels

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
T = 256 * U
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _case(seed, dtype, users, items, dim, bias=True, off=0.1, targets=True, unaligned=False, norm=True):
    g = torch.Generator(device='cuda').manual_seed(seed)

    def table(*shape):
        x = torch.randn(shape, generator=g, device='cuda')
        if norm:
            x = x / x.norm(dim=1, keepdim=True).clamp(min=1e-3)
        if unaligned:
            y = torch.empty(x.numel() + 1, dtype=dtype, device='cuda')[1:].reshape(shape)
            return y.copy_(x)
        return x.to(dtype)
    user, item = table(users, dim), table(items, dim)
    b = None
    if bias:
        b = torch.randn(items, generator=g, device='cuda')
        b[torch.rand(items, generator=g, device='cuda') < off] = -math.inf
    t = None
    if targets:
        t = torch.randint(-1, max(items, 1) + 1, (users,), generator=g, device='cuda').to(torch.int32)   # some outside
        if users > 2:
            t[1] = t[0]                               # the same item twice
    return user, item, t, b


def _reference(user, item, t, b, scale, g_lp, g_e):
    users, dim = user.shape
    items = item.shape[0]
    u, e = user.double(), item.double()
    on = torch.ones(items, dtype=torch.bool, device='cuda') if b is None else b > -1e10
    e = torch.where(on[:, None], e, torch.zeros_like(e))
    z = scale * (u @ e.T)
    width = 32 if dim <= 32 else 64 if dim <= 64 else 128 if dim <= 128 else 256
    mass = scale * (u.abs() @ e.abs().T)
    if b is not None:
        z = torch.where(on, z + b.double(), torch.full_like(z, -math.inf))
    ez = ((6 * width + 16) * 2 * U * mass + 8 * U * z.nan_to_num(neginf=0).abs())
    ez = torch.where(on, ez, torch.zeros_like(ez)).amax(1) if items else torch.zeros(users, device='cuda', dtype=torch.float64)
    lse = torch.logsumexp(z, 1) if items else torch.full((users,), -math.inf, device='cuda', dtype=torch.float64)
    some = lse > -math.inf
    lp = torch.where(on & some[:, None], z - lse[:, None], torch.full_like(z, -math.inf))
    p = torch.exp(lp)
    plp = torch.where(p > 0, p * lp.nan_to_num(neginf=0), torch.zeros_like(p))
    entropy = -plp.sum(1)
    there = torch.zeros(users, dtype=torch.bool, device='cuda') if t is None else (t >= 0) & (t < items)
    index = torch.zeros(users, dtype=torch.long, device='cuda') if t is None else torch.where(there, t, torch.zeros_like(t)).long()
    picked = lp.gather(1, index[:, None])[:, 0] if items else torch.zeros_like(lse)
    log_prob = torch.where(there, picked, torch.zeros_like(lse))
    r = 2 * ez + T
    logs = math.log(max(items, 2))
    tol = {'lse': r + 8 * U * lse.abs().nan_to_num(posinf=0), 'log_prob': r + 8 * U * log_prob.abs().nan_to_num(posinf=0),
           'entropy': r * (2 * (entropy + logs) + 2) + 8 * U * logs}
    g = torch.zeros_like(lse) if g_lp is None else torch.where(there, g_lp.double(), torch.zeros_like(lse))
    ge = torch.zeros_like(lse) if g_e is None else g_e.double()
    hit = (torch.arange(items, device='cuda')[None] == index[:, None]) & there[:, None] & on[None] & some[:, None]
    lp0 = lp.nan_to_num(neginf=0)
    dz = g[:, None] * (hit.double() - p) - ge[:, None] * (plp + p * entropy[:, None])
    factor = (g + ge * entropy)[:, None].abs() + (ge[:, None] * lp0).abs()
    cut = {torch.float32: 2.0 ** -22, torch.float16: 2.0 ** -14, torch.bfloat16: 2.0 ** -8}[user.dtype]
    off = p * (r[:, None] * factor + ge.abs()[:, None] * (r + tol['entropy'])[:, None] + 8 * U * factor) + cut * (p * factor)
    # the sums run over at most 3000 rows here, products of pieces in fp32
    add = (6 * 3000) * U
    half = torch.finfo(user.dtype).eps / 2
    tiny = 2.0 ** -24 if user.dtype == torch.float16 else 1e-30
    g_user, g_item, g_bias = scale * dz @ e, scale * dz.T @ u, dz.sum(0)
    size = off + add * dz.abs()
    tol['g_user'] = scale * size @ e.abs() + half * g_user.abs() + tiny
    tol['g_item'] = scale * size.T @ u.abs() + half * g_item.abs() + tiny
    tol['g_bias'] = size.sum(0) + 1e-30
    return dict(lse=lse, entropy=entropy, log_prob=log_prob, g_user=g_user, g_item=g_item, g_bias=g_bias, z=z), tol


def _near(name, got, want, tol):
    got = got.double()
    assert got.shape == want[name].shape, name
    finite = torch.isfinite(want[name])
    assert torch.equal(got[~finite], want[name][~finite]), name
    off = ((got - want[name]).abs() / tol[name].clamp(min=1e-30))[finite]
    assert off.numel() == 0 or float(off.max()) <= 1.0, "%s: %.3g times the bound" % (name, float(off.max()))


def _check(user, item, t, b, scale=7.0, top=0):
    n = user.shape[0]
    g = torch.Generator(device='cuda').manual_seed(n)
    g_lp = -torch.rand(n, generator=g, device='cuda') if t is not None else None
    g_e = 0.3 * torch.randn(n, generator=g, device='cuda')
    want, tol = _reference(user, item, t, b, scale, g_lp, g_e)
    r = kernels.catalog_log_probs(user, item, t, b, scale, top)
    for name in ('lse', 'entropy') + (('log_prob',) if t is not None else ()):
        _near(name, getattr(r, name), want, tol)
    grads = kernels.catalog_log_probs_bwd(user, item, t, b, scale, r.lse, r.entropy, g_lp, g_e)
    _near('g_user', grads[0], want, tol)
    _near('g_item', grads[1], want, tol)
    assert (grads[2] is None) == (b is None)
    if b is not None:
        _near('g_bias', grads[2], want, tol)
        assert not grads[1][b < -1e10].any() and not grads[2][b < -1e10].any()
    if top:
        _top(r, user, item, b, scale, top, want, tol)
    return r, grads


def _top(r, user, item, b, scale, top, want, tol):
    z = want['z']
    k = min(top, z.shape[1])
    best, at = torch.sort(z, dim=1, descending=True, stable=True)
    at = torch.where(best == -math.inf, torch.full_like(at, -1), at)[:, :k]
    assert torch.equal(r.top_ids[:, :k].long(), at)
    assert bool((r.top_ids[:, k:] == -1).all()) and bool((r.top_log_prob[:, k:] == -math.inf).all())
    value = torch.where(at < 0, torch.full_like(best[:, :k], -math.inf), best[:, :k] - want['lse'][:, None])
    _near('v', r.top_log_prob[:, :k], {'v': value}, {'v': (tol['lse'][:, None] + 8 * U * value.abs().nan_to_num(posinf=0))})


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('dim', [1, 8, 19, 32, 33, 64, 100, 128, 200, 256])
def test_widths(cuda, dtype, dim):
    _check(*_case(dim, dtype, 70, 333, dim), top=5)
    _check(*_case(dim, dtype, 9, 1000, dim, bias=False, unaligned=True), top=20)


@pytest.mark.parametrize('users', [1, 2, 31, 32, 33, 64, 65, 129, 1000])
@pytest.mark.parametrize('items', [1, 2, 31, 32, 33, 500, 2999])
def test_sizes(cuda, users, items):
    _check(*_case(users * 7 + items, torch.float32, users, items, 32), top=10)
    _check(*_case(users * 7 + items, torch.bfloat16, users, items, 64, bias=False), top=64)


def test_one_item_leaves_no_choice(cuda):
    user, item, _, _ = _case(1, torch.float32, 50, 1, 40, norm=False)
    t = torch.zeros(50, dtype=torch.int32, device='cuda')
    r = kernels.catalog_log_probs(user, item, t, None, 30.0)
    assert not r.log_prob.any() and not r.entropy.any()
    # lse comes back rounded to fp32, half a unit of |z| (some hundreds here): p = exp(z - lse) is 1 within r, which
    # counts 8 u |z| for it, and the gradients, exactly 0, are off by as much of what they are sums of
    _check(user, item, t, None, scale=30.0, top=1)


def test_nothing_on_offer_and_empty_tables(cuda):
    for b in (-math.inf, torch.finfo(torch.float32).min):
        user, item, t, bias = _case(2, torch.float32, 40, 100, 32)
        bias.fill_(b)
        r, g = _check(user, item, t, bias, top=3)
        assert bool((r.lse == -math.inf).all()) and not r.entropy.any() and bool((r.top_ids == -1).all())
        assert not g[0].any() and not g[1].any() and not g[2].any()
    _check(*_case(3, torch.float32, 5, 0, 32, bias=False), top=3)
    user, item, t, bias = _case(3, torch.float32, 0, 9, 32)
    r = kernels.catalog_log_probs(user, item, t, bias, 1.0, 4)
    assert r.entropy.numel() == 0 and r.top_ids.shape == (0, 4)
    g = kernels.catalog_log_probs_bwd(user, item, t, bias, 1.0, r.lse, r.entropy, r.entropy, r.entropy)
    assert g[0].shape == (0, 32) and not g[1].any() and not g[2].any()


def test_what_is_not_on_offer_may_be_anything(cuda):
    user, item, t, bias = _case(4, torch.float32, 70, 200, 48)
    want, g_want = _check(user, item, t, bias, top=7)
    off = bias == -math.inf
    item[off] = math.nan
    item[torch.nonzero(off)[0]] = math.inf
    bias[off] = torch.finfo(torch.float32).min
    got, g_got = (kernels.catalog_log_probs(user, item, t, bias, 7.0, 7), None)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    g = torch.Generator(device='cuda').manual_seed(70)
    g_lp, g_e = -torch.rand(70, generator=g, device='cuda'), 0.3 * torch.randn(70, generator=g, device='cuda')
    g_got = kernels.catalog_log_probs_bwd(user, item, t, bias, 7.0, got.lse, got.entropy, g_lp, g_e)
    for a, b in zip(g_got, g_want):
        assert torch.equal(a, b)


@pytest.mark.parametrize('dtype', DTYPES)
def test_ties_go_to_the_lowest_index(cuda, dtype):
    user, item, t, bias = _case(5, dtype, 33, 3000, 24, bias=False)
    item[1000:2000] = item[:1000]                     # every item of the first thousand twice
    _check(user, item, t, None, top=64)
    item[:] = item[7].clone()                         # all the same: more candidates than the buffer holds
    _check(user, item, t, None, top=64)
    bias = torch.zeros(3000, device='cuda')
    bias[:13] = -math.inf
    r, _ = _check(user, item, t, bias, top=5)
    assert bool((r.top_ids == torch.arange(13, 18, device='cuda')).all())
    user.zero_()
    _check(user, item, t, None, top=9)


def test_scores_that_32_bits_cannot_tell_apart(cuda):
    g = torch.Generator(device='cuda').manual_seed(6)
    item = torch.randn((4000, 64), generator=g, device='cuda')
    item = (item[:1] + 1e-7 * item).contiguous()      # scores apart by a few units in the last place of fp32
    user = torch.randn((17, 64), generator=g, device='cuda')
    _check(user, item, None, None, scale=1.0, top=50)


def test_far_scores_large_norms_and_small_scales(cuda):
    user, item, t, bias = _case(7, torch.float32, 65, 600, 64, norm=False)
    _check(user, item, t, bias, scale=10.0, top=8)    # scores of a hundred and more
    _check(user, item, t, bias, scale=1e-4, top=8)
    bias[::3] -= 65504.0                              # the lowest value of another type: still on offer
    _check(user, item, t, bias, scale=1.0, top=8)


def test_users_in_slices(cuda):
    """The table of tile maxima is bounded, so users are ranked in slices; 256 at a time for 9 million items."""
    g = torch.Generator(device='cuda').manual_seed(8)
    item = torch.randn((9_000_000, 4), generator=g, device='cuda').to(torch.bfloat16)
    user = torch.randn((300, 4), generator=g, device='cuda').to(torch.bfloat16)
    r = kernels.catalog_log_probs(user, item, None, None, 1.0, 3)
    for n in (0, 255, 256, 299):
        z = item.double() @ user[n].double()
        best, at = torch.sort(z, descending=True, stable=True)
        assert r.top_ids[n].tolist() == at[:3].tolist()
        one = kernels.catalog_log_probs(user[n:n + 1].contiguous(), item, None, None, 1.0, 3)
        assert one.top_ids.tolist() == r.top_ids[n:n + 1].tolist()
        assert abs(float(r.lse[n]) - float(torch.logsumexp(z, 0))) < 1e-4


def test_a_nan_stays_with_its_user(cuda):
    user, item, t, bias = _case(9, torch.float32, 40, 300, 32)
    want = kernels.catalog_log_probs(user, item, t, bias, 5.0, 4)
    user[3, 5] = math.nan
    got = kernels.catalog_log_probs(user, item, t, bias, 5.0, 4)
    keep = torch.arange(40, device='cuda') != 3
    for a, b in zip(got, want):
        assert torch.equal(a[keep], b[keep])
    assert bool(got.entropy[3].isnan()) and bool(got.lse[3].isnan()) and bool((got.top_ids[3] == -1).all())


def test_results_repeat(cuda):
    case = _case(10, torch.float32, 500, 2000, 64)
    first = _check(*case, top=10)
    junk = torch.full((1 << 25,), float('nan'), device='cuda')
    del junk
    again = _check(*case, top=10)
    for a, b in zip(first[0] + first[1], again[0] + again[1]):
        assert torch.equal(a, b)


def test_gradients_of_differences(cuda):
    user, item, t, bias = _case(11, torch.float32, 6, 9, 5, off=0.0)
    leaves = [x.clone().requires_grad_() for x in (user, item, bias)]
    lp, entropy = autograd.CatalogLogProbs.apply(leaves[0], leaves[1], t, leaves[2], 3.0)
    g = torch.Generator(device='cuda').manual_seed(1)
    c1, c2 = torch.randn(6, generator=g, device='cuda'), torch.randn(6, generator=g, device='cuda')
    (c1 * lp + c2 * entropy).sum().backward()

    def value(u, e, b):
        lp = torch.log_softmax(3.0 * u @ e.T + b, 1)
        there = (t >= 0) & (t < 9)
        chosen = torch.where(there, lp.gather(1, torch.where(there, t, torch.zeros_like(t)).long()[:, None])[:, 0], torch.zeros_like(lp[:, 0]))
        return float((c1.double() * chosen - c2.double() * (lp.exp() * lp).sum(1)).sum())
    base = [x.detach().double() for x in leaves]
    for i in range(3):
        for _ in range(4):
            step = torch.randn(base[i].shape, generator=g, device='cuda', dtype=torch.float64)
            eps = 1e-5
            plus, minus = ([b + s * step if j == i else b for j, b in enumerate(base)] for s in (eps, -eps))
            slope = (value(*plus) - value(*minus)) / (2 * eps)
            terms = leaves[i].grad.double() * step
            # central differences are off by about eps^2 here, fp32 by some hundred u of the terms
            assert abs(float(terms.sum()) - slope) <= 1e-4 * float(terms.abs().sum()) + 1e-7


def test_only_what_is_wanted(cuda):
    user, item, t, bias = _case(12, torch.float32, 50, 80, 32)
    r, full = _check(user, item, t, bias)
    g = torch.Generator(device='cuda').manual_seed(50)
    g_lp, g_e = -torch.rand(50, generator=g, device='cuda'), 0.3 * torch.randn(50, generator=g, device='cuda')
    for i in range(3):
        got = kernels.catalog_log_probs_bwd(user, item, t, bias, 7.0, r.lse, r.entropy, g_lp, g_e, need_user=i == 0,
                                            need_item=i == 1, need_bias=i == 2)
        assert [x is None for x in got] == [j != i for j in range(3)] and torch.equal(got[i], full[i])
    _, none = _reference(user, item, t, bias, 7.0, None, None)
    got = kernels.catalog_log_probs_bwd(user, item, t, bias, 7.0, r.lse, r.entropy)
    assert not got[0].any() and not got[1].any() and not got[2].any()


def test_another_stream_and_replayed_graphs(cuda):
    user, item, t, bias = _case(13, torch.float32, 200, 900, 32)
    ones = torch.full((200,), -0.005, device='cuda')

    def body():
        r = kernels.catalog_log_probs(user, item, t, bias, 7.0, 6)
        return tuple(r) + kernels.catalog_log_probs_bwd(user, item, t, bias, 7.0, r.lse, r.entropy, ones, ones)
    want = body()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = body()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    graphs, results = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            results.append(body())
        graphs.append(g)
    for _ in range(3):
        user.mul_(0.9)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = body()
        for res in results:
            for a, b in zip(res, want):
                assert torch.equal(a, b)


def test_refusals(cuda):
    z = lambda *s, t=torch.float32: torch.zeros(s, dtype=t, device='cuda')
    u, e, t, b = z(4, 8), z(9, 8), z(4, t=torch.int32), z(9)
    f = kernels.catalog_log_probs
    for bad, err in [(lambda: f(u.cpu(), e), _lib.GsageError), (lambda: f(u.double(), e.double()), TypeError),
                     (lambda: f(u, e.half()), TypeError), (lambda: f(u, z(9, 7)), ValueError),
                     (lambda: f(u[:, ::2], e[:, ::2]), ValueError), (lambda: f(u, e, t.long()), TypeError),
                     (lambda: f(u, e, z(5, t=torch.int32)), ValueError), (lambda: f(u, e, t, z(8)), ValueError),
                     (lambda: f(u, e, t, b.half()), TypeError), (lambda: f(u, e, t, b, 0.0), ValueError),
                     (lambda: f(u, e, t, b, float('inf')), ValueError), (lambda: f(u, e, t, b, 1.0, -1), ValueError),
                     (lambda: f(u, e, t, b, 1.0, 65), _lib.GsageError), (lambda: f(z(4, 257), z(9, 257)), _lib.GsageError),
                     (lambda: kernels.catalog_log_probs_bwd(u, e, t, b, 1.0, None, None), ValueError),
                     (lambda: kernels.catalog_log_probs_bwd(u, e, t, b, 1.0, z(4), None, None, z(4)), ValueError),
                     (lambda: kernels.catalog_log_probs_bwd(u, e, t, b, 1.0, z(5), z(4)), ValueError)]:
        with pytest.raises(err):
            bad()


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('users', [1, 31, 32, 33, 63, 64, 65, 96, 97, 128, 129])
def test_counts_of_users_around_the_tiles_of_a_block(cuda, dtype, users):
    for items, dim, k in ((1, 5, 1), (130, 64, 20), (2100, 33, 5)):
        _check(*_case(users + items, dtype, users, items, dim), top=k)
