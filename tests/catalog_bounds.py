"""The catalog's gradients and log probabilities in 64 bits with bounds that stay sharp where a score is exact, and the
kernels' rounding restated on the CPU.

One of the two tables is zeros, so a score is the item's bias alone and what is left to round is known step by step
(u = 2^-24, natural logarithms):

* a bias b and an lse L in units of log 2, their difference and its exponential: p is off by at most
  e_p = u (4 (|b| + |L| + |log p|) + 8) p, and by what L itself is off;
* L: a sum of ``items`` exponentials, each off by 2 u, the logarithm, two roundings of the result:
  e_L = u (items + 8 + 2 |L|);
* a target's log p: its distance to the largest score, exactly 0 for that one, else 4 u (|b| + |largest b|), and the
  logarithm of the sum of what lies relative to the largest, u (items + 8), rounded: 4 u |log p|;
* the target's dz = g + p (A + B log p) is formed in fp32, so that what remains of it is off by e_p p |factor| and by the
  additions of a tile of 32 rows, and of the pieces of g, while the sum holds the one and not yet the other: those of
  min(rows, 32) rows at u (|g| + p |factor|) each;
* any other dz is cut into n bf16 pieces (n: 1 bf16, 2 fp16, 3 fp32): 2^-8, 2^-14, 2^-22 of it with the products that
  are left out, on top of e_p;
* a sum of ``rows`` terms adds the products of their pieces one after the other at the worst (rows with nothing in them add
  zeros, exactly): (6 rows + 8) u of the terms' sizes for fp32, (4 rows + 8) u for fp16, (rows + 8) u for bf16;
* the result is rounded to the tables' type.
"""
import math

import torch

U = 2.0 ** -24
CUT = {torch.float32: 2.0 ** -22, torch.float16: 2.0 ** -14, torch.bfloat16: 2.0 ** -8}
PRODUCTS = {torch.float32: 6, torch.float16: 4, torch.bfloat16: 1}
PIECES = {torch.float32: 3, torch.float16: 2, torch.bfloat16: 1}


def reference(user, item, target, bias, scale, g_log_prob, g_entropy):
    """(values, bounds) of lse, entropy, log_prob, g_user, g_item, g_bias; user or item is all zeros."""
    dtype, dev = user.dtype, user.device
    users, items = user.shape[0], item.shape[0]
    assert not user.any() or not item.any()
    u, e = user.double(), item.double()
    z = bias.double()[None].expand(users, items)
    lse = torch.logsumexp(z, 1)
    lp = z - lse[:, None]
    # log p of a term that leaves next to nothing to the others, without the cancellation
    order = torch.arange(items, device=dev)
    rest = torch.stack([torch.logsumexp(torch.cat([z[:, :j], z[:, j + 1:]], 1) - z[:, j:j + 1], 1) for j in range(items)], 1) \
        if items > 1 else torch.full_like(z, -math.inf)
    lp = torch.where(lp > -1, -torch.log1p(torch.exp(rest)), lp)
    left = torch.where(lp > -1, -torch.expm1(lp), 1 - torch.exp(lp))             # 1 - p
    p = torch.exp(lp)
    entropy = -(p * lp).sum(1)
    there = (target >= 0) & (target < items)
    hit = (order[None] == target[:, None]) & there[:, None]
    picked, top = (z * hit).sum(1), z.amax(1)
    log_prob = torch.where(there, (lp * hit).sum(1), torch.zeros_like(lse))
    g = torch.where(there, g_log_prob.double(), torch.zeros_like(lse))[:, None]
    ge = g_entropy.double()[:, None]
    dz = torch.where(hit, g * left, -g * p) - ge * p * (lp + entropy[:, None])

    e_lse = U * (items + 8 + 2 * lse.abs())[:, None]
    e_p = U * (4 * (z.abs() + lse.abs()[:, None] + lp.abs()) + 8) + e_lse
    factor = g.abs() + ge.abs() * (entropy[:, None] + lp.abs())
    logs = math.log(items) + 1
    e_entropy = U * (items + 8) * (2 * entropy + 2 * logs) + 8 * U * logs
    off = p * factor * (e_p + 4 * U) + ge.abs() * p * (e_p + e_entropy[:, None])
    off = off + torch.where(hit, torch.zeros_like(off), CUT[dtype] * p * factor)
    whole = torch.where(hit, g.abs() + p * factor, torch.zeros_like(off))
    half = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -24 if dtype == torch.float16 else 1e-37
    grad = lambda w, x: scale * torch.matmul(w, x)
    add = lambda rows: (PRODUCTS[dtype] * rows + 8) * U
    want = dict(lse=lse, entropy=entropy, log_prob=log_prob, g_user=grad(dz, e), g_item=grad(dz.T, u), g_bias=dz.sum(0))
    tol = dict(lse=e_lse[:, 0], entropy=e_entropy,
               log_prob=torch.where(there, U * (items + 8 + 4 * log_prob.abs()) + torch.where(picked < top, 4 * U * (picked.abs() + top.abs()),
                                    torch.zeros_like(top)), torch.zeros_like(top)))
    tol['g_user'] = grad(off + add(min(items, 32)) * whole + add(items) * dz.abs(), e.abs()) + half * want['g_user'].abs() + tiny
    by_user = off + add(min(users, 32)) * whole + add(users) * dz.abs()
    tol['g_item'] = grad(by_user.T, u.abs()) + half * want['g_item'].abs() + tiny
    tol['g_bias'] = by_user.sum(0) + 1e-37
    return want, tol


def worst(got, want, tol):
    """The largest error in units of its bound."""
    off = (got.double() - want).abs() / tol.clamp(min=1e-300)
    return float(torch.where((got.double() == want), torch.zeros_like(off), off).max()) if off.numel() else 0.0


def emulate(user, item, target, bias, scale, g_log_prob, g_entropy, whole_target=True, pieces=None):
    """(g_user, g_item) with the kernels' roundings: p, dz in fp32, dz and the tables in pieces, sums in 64 bits.
    ``whole_target`` false: g whole, but -g p in pieces like any other element; ``pieces``: fewer than the type has."""
    dtype = user.dtype
    n = PIECES[dtype] if pieces is None else pieces
    z = bias.float()[None].expand(user.shape[0], -1)
    lse = torch.logsumexp(z.double(), 1).float()
    lp = z - lse[:, None]
    p = torch.exp(lp.double()).float()
    entropy = -(p.double() * lp.double()).sum(1).float()
    there = (target >= 0) & (target < item.shape[0])
    g = torch.where(there, g_log_prob, torch.zeros_like(lse))[:, None]
    hit = (torch.arange(item.shape[0])[None] == target[:, None]) & there[:, None]
    ge = g_entropy[:, None]
    dz = p * (-(g + ge * entropy[:, None]) - ge * lp)
    whole = torch.where(hit, g + dz if whole_target else g.expand_as(dz), torch.zeros_like(dz)).double()
    if whole_target:
        dz = torch.where(hit, torch.zeros_like(dz), dz)

    def cut(x):
        x, out = x.float().clone(), []
        for _ in range(n):
            out.append(x.bfloat16().float())
            x = x - out[-1]
        return out

    def product(w, x):
        ws, xs = cut(w), cut(x.float())
        return sum(ws[i].double() @ xs[k].double() for i in range(n) for k in range(n) if i + k <= 2)
    g_user = scale * (product(dz, item) + whole @ item.double())
    g_item = scale * (product(dz.T.contiguous(), user) + whole.T @ user.double())
    return g_user.to(dtype), g_item.to(dtype)


def case(dtype, users, items, dim, gap, shift, seed, device, user_zero, same=False):
    """Users whose first half chooses item 0, which is ahead of the others by ``gap``; the others choose any item or none, or
    (``same``) that one too."""
    gen = torch.Generator().manual_seed(seed)
    user = torch.randn(users, dim, generator=gen).to(dtype)
    item = torch.randn(items, dim, generator=gen).to(dtype)
    (user if user_zero else item).zero_()
    bias = torch.rand(items, generator=gen) - gap + shift
    bias[0] = shift
    target = torch.randint(-1, items + 1, (users,), generator=gen).to(torch.int32)
    target[:users if same else (users + 1) // 2] = 0
    g_log_prob = -0.5 - torch.rand(users, generator=gen)
    g_entropy = 0.01 * torch.randn(users, generator=gen)
    return [x.to(device) for x in (user, item, target, bias)] + [2.5] + [x.to(device) for x in (g_log_prob, g_entropy)]


# ---- scores of fp32 tables: two elements a row, the others zeros ---------------------------------------------------------

def thin_tables(users, items, dim, seed, device):
    """fp32 rows whose first and last elements, in [1/2, 1), are all they have: a score is a sum of 12 products of pieces."""
    gen = torch.Generator().manual_seed(seed)
    tables = []
    for n in (users, items):
        x = torch.zeros(n, dim)
        x[:, 0] = 0.5 + 0.5 * torch.rand(n, generator=gen)
        x[:, -1] = 0.5 + 0.5 * torch.rand(n, generator=gen)
        tables.append(x.to(device))
    return tables


def thin_scores(user, item, scale):
    """(scores in 64 bits, their bound): 12 additions of products, the three products left out (2 u), the fused
    multiply-add with its constant and the conversion to units of log 2 (4 u) and back (2 u)."""
    z = scale * torch.matmul(user.double(), item.double().T.contiguous())
    return z, 20 * U * z.abs()                       # (all terms are positive: the sum of their sizes is the score)


def cut_scores(user, item, scale, pieces):
    """The scores of tables cut into fewer pieces than fp32 has."""
    cut = []
    for x in (user, item):
        left, total = x.clone(), torch.zeros_like(x)
        for _ in range(pieces):
            p = left.bfloat16().float()
            total, left = total + p, left - p
        cut.append(total.double())
    return scale * cut[0] @ cut[1].T
