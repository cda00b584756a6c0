"""torch.autograd glue: records which HIP kernel undoes which, nothing more.

Each Function calls one forward entry point of ``libgsage.so`` and, in
``backward``, the matching backward entry point.  Feature tables are constants
of the reference model (they are inputs, not variables, ``models.py:241``), so
the indexed gather-mean only propagates a gradient into the table when the
table itself requires one (trainable embeddings); then it is the float-atomic
scatter-add kernel.

A backward pass may be captured into a HIP graph.  Results of eager calls on the
same leaves have to be gone by then: torch's engine would wait for the stream
they ran on, which a capture does not survive.
"""
import torch

from . import kernels


class GatherRows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, feat, ids, id_offset):
        ctx.save_for_backward(ids)
        ctx.meta = (feat.shape, int(id_offset))
        return kernels.gather_rows(feat, ids, id_offset)

    @staticmethod
    def backward(ctx, g):
        if not ctx.needs_input_grad[0]:
            return None, None, None
        (ids,) = ctx.saved_tensors
        shape, off = ctx.meta
        g_feat = torch.zeros(shape, dtype=torch.float32, device=g.device)
        kernels.gather_mean_bwd(g.contiguous(), ids, 1, g_feat, off)
        return g_feat, None, None


class GatherMean(torch.autograd.Function):
    """mean over the n_child sampled children of each parent, rows taken from a
    feature table by node id."""

    @staticmethod
    def forward(ctx, feat, child_ids, n_parents, n_child, id_offset):
        ctx.save_for_backward(child_ids)
        ctx.meta = (feat.shape, int(n_child), int(id_offset))
        return kernels.gather_mean(feat, child_ids, n_parents, n_child, id_offset)

    @staticmethod
    def backward(ctx, g):
        if not ctx.needs_input_grad[0]:
            return None, None, None, None, None
        (child_ids,) = ctx.saved_tensors
        shape, n_child, off = ctx.meta
        g_feat = torch.zeros(shape, dtype=torch.float32, device=g.device)
        kernels.gather_mean_bwd(g.contiguous(), child_ids, n_child, g_feat, off)
        return g_feat, None, None, None, None


class GroupMean(torch.autograd.Function):
    """mean over axis 1 of a dense (n_parents, n_child, F) tensor."""

    @staticmethod
    def forward(ctx, x, n_parents, n_child):
        ctx.meta = (x.shape, int(n_parents), int(n_child))
        return kernels.gather_mean(x.reshape(n_parents * n_child, -1), None, n_parents, n_child)

    @staticmethod
    def backward(ctx, g):
        shape, n_parents, n_child = ctx.meta
        g_x = torch.empty((n_parents * n_child, g.shape[1]), dtype=torch.float32, device=g.device)
        kernels.gather_mean_bwd(g.contiguous(), None, n_child, g_x)
        return g_x.reshape(shape), None, None


class GatherMax(torch.autograd.Function):
    """max over the sampled children of each parent, rows taken from a feature
    table by node id; the table is an input of the model and gets no gradient."""

    @staticmethod
    def forward(ctx, feat, child_ids, n_parents, n_child, id_offset):
        if feat.requires_grad:
            raise NotImplementedError("the max aggregator has no gradient into a feature table")
        return kernels.gather_max(feat, child_ids, n_parents, n_child, id_offset)

    @staticmethod
    def backward(ctx, g):
        return None, None, None, None, None


class GroupMax(torch.autograd.Function):
    """max over axis 1 of a dense (n_parents, n_child, F) tensor; ties share the
    gradient evenly."""

    @staticmethod
    def forward(ctx, x, n_parents, n_child):
        x2 = x.reshape(n_parents * n_child, -1)
        out = kernels.gather_max(x2, None, n_parents, n_child)
        ctx.save_for_backward(x2, out)
        ctx.meta = (x.shape, int(n_child))
        return out

    @staticmethod
    def backward(ctx, g):
        x2, out = ctx.saved_tensors
        shape, n_child = ctx.meta
        return kernels.group_max_bwd(g.contiguous(), x2, out, n_child).reshape(shape), None, None


class SageProject(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x_self, x_mean, w_self, w_neigh, bias, act):
        out = kernels.sage_project(x_self, x_mean, w_self, w_neigh, bias, act)
        ctx.act = act
        ctx.has_bias = bias is not None
        ctx.save_for_backward(x_self, x_mean, w_self, w_neigh, out)
        return out

    @staticmethod
    def backward(ctx, g):
        x_self, x_mean, w_self, w_neigh, out = ctx.saved_tensors
        need = ctx.needs_input_grad
        g_ws, g_wn, g_b, g_xs, g_xm = kernels.sage_project_bwd(
            x_self, x_mean, w_self, w_neigh, ctx.act, out, g.contiguous(),
            need_x_self=need[0], need_x_mean=need[1], need_bias=ctx.has_bias)
        return g_xs, g_xm, g_ws, g_wn, g_b, None


class L2Normalize(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        ctx.save_for_backward(x)
        return kernels.l2_normalize(x)

    @staticmethod
    def backward(ctx, g):
        (x,) = ctx.saved_tensors
        return kernels.l2_normalize_bwd(x, g.contiguous())


class _Refuse(torch.autograd.Function):
    @staticmethod
    def forward(ctx, what, *grads):
        ctx.what = what
        return tuple(None if g is None else g.view_as(g) for g in grads)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("the gradients of %s cannot be differentiated again" % ctx.what)


def _once(backward):
    """A backward pass whose results depend on the saved inputs but have no derivatives of their own: where a graph of it is
    asked for, whoever differentiates them gets an error (torch's own mark for this lets them pass as constants when the gradient
    that came in is one)."""
    def once(ctx, *grads):
        with torch.no_grad():
            out = backward(ctx, *grads)
        if not torch.is_grad_enabled():
            return out
        return _Refuse.apply(type(ctx).__name__.replace('Backward', ''),
                             *(None if g is None else g.detach().requires_grad_() for g in out))
    return once


class Dropout(torch.autograd.Function):
    """``kernels.dropout``; the backward pass draws the mask again.  A seed that lives in GPU memory is copied, so that
    the gradient goes by the mask that was drawn even if the caller has changed the seed since."""

    @staticmethod
    def forward(ctx, x, rate, seed, offset):
        if isinstance(seed, torch.Tensor):
            seed = seed.clone()
        ctx.mask = (rate, seed, offset)
        return kernels.dropout(x, rate, seed, offset)

    @staticmethod
    def backward(ctx, g):
        # (the map is linear: where the gradient is to be differentiated again, it is this function once more)
        again = Dropout.apply if torch.is_grad_enabled() and g.requires_grad else kernels.dropout
        return again(g.contiguous(), *ctx.mask), None, None, None


class NeighborAttention(torch.autograd.Function):
    """``kernels.neighbor_attention``: (out, lse); gradients through ``out`` only.  With child_ids, the gradient of
    the tables takes ``inverse`` (``kernels.neighbor_inverse``; built in the backward pass when it is None).  The gradients
    cannot be differentiated again (an error says so)."""

    @staticmethod
    def forward(ctx, q, k, v, child_ids, n_child, id_offset, scale, indptr, inverse):
        out, lse = kernels.neighbor_attention(q, k, v, child_ids, n_child, id_offset, scale, indptr)
        ctx.save_for_backward(q, k, v, child_ids, out, lse, indptr)
        ctx.meta = (n_child, int(id_offset), scale, inverse)
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @_once
    def backward(ctx, g, _):
        q, k, v, child_ids, out, lse, indptr = ctx.saved_tensors
        n_child, id_offset, scale, inverse = ctx.meta
        need = ctx.needs_input_grad
        g_q, g_k, g_v = kernels.neighbor_attention_bwd(
            q, k, v, child_ids, n_child, out, lse, g.contiguous(), id_offset, scale, indptr, inverse,
            need_q=need[0], need_rows=need[1] or need[2])
        return (g_q, g_k if need[1] else None, g_v if need[2] else None) + (None,) * 6


class CatalogLogProbs(torch.autograd.Function):
    """``kernels.catalog_log_probs``: (log_prob, entropy) of users over a catalog, with gradients to users, items and
    bias, which cannot be differentiated again (an error says so)."""

    @staticmethod
    def forward(ctx, user, item, targets, bias, scale):
        r = kernels.catalog_log_probs(user, item, targets, bias, scale)
        ctx.save_for_backward(user, item, targets, bias, r.lse, r.entropy)
        ctx.scale = scale
        return r.log_prob, r.entropy

    @staticmethod
    @_once
    def backward(ctx, g_log_prob, g_entropy):
        user, item, targets, bias, lse, entropy = ctx.saved_tensors
        need = ctx.needs_input_grad
        g = [None if x is None else x.contiguous() for x in (g_log_prob, g_entropy)]
        g_user, g_item, g_bias = kernels.catalog_log_probs_bwd(user, item, targets, bias, ctx.scale, lse, entropy, *g,
                                                               need_user=need[0], need_item=need[1], need_bias=need[3])
        return g_user, g_item, None, g_bias, None
