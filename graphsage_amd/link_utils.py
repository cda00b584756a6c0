"""Link prediction heads, after the reference's ``link_utils.py``.

``link_classification(edge_embedding_method="concat")`` -- what the training
script uses (``train_movielens.py:179``): concatenate the two node embeddings,
``Dense(1, sigmoid)``, reshape to ``(B, 1)`` (``link_utils.py:167-168,244-247,
312-317``) -- is the head with kernels of its own (``train.LinkHead``: fused
forward + MSE + gradients, part of the static training plan).

The other operators of ``LinkEmbedding.call`` (``link_utils.py:154-176``: ip/dot,
mul/hadamard, l1, l2, avg), other output widths and activations, and the clipped
regression head (``link_regression``, ``LeakyClippedLinear``) are plain torch
modules here; a model with one of them trains through autograd.

``link_ranking`` (not in the reference) gives ``CatalogHead``: links are learned as a choice among the items of the batch
(softmax loss) and users are answered with the best items of a whole catalog.
"""
import math
import warnings

import torch

from . import autograd as _ag
from . import kernels
from .train import LinkHead

__all__ = ['LinkEmbedding', 'EdgeHead', 'CatalogHead', 'link_inference', 'link_classification', 'link_regression',
           'link_ranking']

_ACTIVATIONS = {
    'linear': lambda x: x, None: lambda x: x,
    'sigmoid': torch.sigmoid, 'relu': torch.relu, 'tanh': torch.tanh,
    'softmax': lambda x: torch.softmax(x, dim=-1),
}


def _activation(name):
    try:
        return _ACTIVATIONS[name]
    except KeyError:
        raise ValueError("unknown activation %r" % (name,))


class LinkEmbedding:
    """Combines the two node embeddings of a link (``link_utils.py:104-180``):
    a list of two (N, M) tensors, or one tensor with a dimension of size 2 at
    ``axis``."""

    def __init__(self, method="ip", axis=-2, activation="linear"):
        self.method = method.lower()
        self.axis = axis
        self.activation = _activation(activation)

    def __call__(self, x):
        if isinstance(x, (list, tuple)):
            if len(x) != 2:
                raise ValueError("Expecting a list of length 2 for link embedding")
            x0, x1 = x
        elif isinstance(x, torch.Tensor):
            if int(x.shape[self.axis]) != 2:
                raise ValueError("Expecting a tensor of shape 2 along specified axis for link embedding")
            x0, x1 = torch.unbind(x, dim=self.axis)
        else:
            raise TypeError("Expected a list, tuple, or Tensor as input")
        if self.method in ("ip", "dot"):
            out = (x0 * x1).sum(dim=-1, keepdim=True)
        elif self.method == "l1":
            out = (x0 - x1).abs()
        elif self.method == "l2":
            out = (x0 - x1) ** 2
        elif self.method in ("mul", "hadamard"):
            out = x0 * x1
        elif self.method == "concat":
            out = torch.cat([x0, x1], dim=-1)
        elif self.method == "avg":
            out = (x0 + x1) / 2
        else:
            raise NotImplementedError
        return self.activation(out)

    def width(self, emb_dim):
        return {'ip': 1, 'dot': 1, 'concat': 2 * emb_dim}.get(self.method, emb_dim)


class EdgeHead:
    """``link_inference``'s edge function (``link_utils.py:236-256``): link
    embedding, then ``Dense(output_dim, output_act)`` (inner product: only the
    activation), reshape to ``(B, output_dim)``, optionally the leaky clip."""

    def __init__(self, emb_dim, device, output_dim=1, output_act="linear", method="ip", clip_limits=None, seed=None):
        self.embed = LinkEmbedding(method=method, activation="linear")
        self.output_dim = output_dim
        self.act = _activation(output_act)
        self.clip_limits = clip_limits
        self.kernel = self.bias = None
        if self.embed.method not in ("ip", "dot"):
            gen = torch.Generator(device='cpu')
            gen.manual_seed(int(seed)) if seed is not None else gen.seed()
            fan_in = self.embed.width(emb_dim)
            limit = math.sqrt(6.0 / (fan_in + output_dim))                    # Keras glorot_uniform
            k = (torch.rand(fan_in, output_dim, generator=gen, dtype=torch.float64) * 2 - 1) * limit
            self.kernel = k.to(torch.float32).to(device).requires_grad_(True)
            self.bias = torch.zeros(output_dim, dtype=torch.float32, device=device, requires_grad=True)

    def parameters(self):
        return [] if self.kernel is None else [self.kernel, self.bias]

    def __call__(self, x_out):
        le = self.embed(x_out)
        out = self.act(le) if self.kernel is None else self.act(le @ self.kernel + self.bias)
        out = out.reshape(-1, self.output_dim)
        if self.clip_limits:
            low, high = self.clip_limits                                       # LeakyClippedLinear, alpha = 0.1
            out = torch.where(out < low, low + 0.1 * (out - low), torch.where(out > high, high + 0.1 * (out - high), out))
        return out


def link_inference(output_dim=1, output_act="linear", edge_embedding_method="ip", clip_limits=None,
                   name="link_inference"):
    if edge_embedding_method in ("ip", "dot") and output_dim != 1:
        warnings.warn("For inner product link method the output_dim will be ignored as it is fixed to be 1.", stacklevel=2)
        output_dim = 1
    LinkEmbedding(method=edge_embedding_method)([torch.zeros(1, 1), torch.zeros(1, 1)])   # unknown methods raise here
    _activation(output_act)

    def edge_function(x_out, seed=None):
        """``x_out`` is what ``GraphSAGE.in_out_tensors()`` returns second (the
        built model); the head takes its embedding width and device from it."""
        model = x_out.build()
        emb_dim, device = model.dims[-1]['user'], model.parameters()[0].device
        if edge_embedding_method == "concat" and output_dim == 1 and output_act == "sigmoid" and not clip_limits:
            return LinkHead(emb_dim, device, seed=seed)                       # the head with its own kernels
        return EdgeHead(emb_dim, device, output_dim, output_act, edge_embedding_method, clip_limits, seed=seed)

    print("{}: using '{}' method to combine node embeddings into edge embeddings".format(name, edge_embedding_method))
    return edge_function


def link_classification(output_dim=1, output_act="sigmoid", edge_embedding_method="ip"):
    return link_inference(output_dim=output_dim, output_act=output_act,
                          edge_embedding_method=edge_embedding_method, name="link_classification")


def link_regression(output_dim=1, clip_limits=None, edge_embedding_method="ip"):
    return link_inference(output_dim=output_dim, output_act="linear", edge_embedding_method=edge_embedding_method,
                          clip_limits=clip_limits, name="link_regression")


def _first_places(ids):
    """For every entry the first place in which its value stands (nothing waits for the device)."""
    n = ids.numel()
    value, at = torch.sort(ids, stable=True)
    place = torch.arange(n, device=ids.device)
    new = torch.ones(n, dtype=torch.bool, device=ids.device)
    new[1:] = value[1:] != value[:-1]
    run = torch.cummax(torch.where(new, place, torch.zeros_like(place)), 0)[0] if n else place
    return torch.empty_like(place).scatter_(0, at, at[run])


class CatalogHead:
    """Scores ``scale * <user, item>`` as logits over a catalog of items.

    ``loss((user_emb, item_emb), targets)``: every positive link (target > 0.5) is a choice of its item among the items of
    the batch; minus the mean log probability of these choices, minus ``entropy_weight`` times the mean entropy of all
    users' choices (``gs_catalog_fwd`` / ``gs_catalog_bwd``: the logits never pass through memory).  ``item_bias`` corrects for
    how the batch's items are drawn (minus the logarithm of their frequencies): one value per item of the batch in the call, or
    one per item of the catalog (its row in the graph's item table) in the constructor; the call is then told which the
    batch's are (``items``, as ``Trainer`` does).
    An item that occurs several times in the batch is as many choices, so that a user's own item is a wrong one, too, in every
    other place; with ``distinct_items`` (and ``items``) it is one choice, for which its first place in the batch stands.
    Under several ranks each rank's batch is a choice of its own, and their gradients are averaged.
    ``recommend(user_emb, item_emb, k)``: the k best of all items for every user.
    Called like the other heads it scores the batch's own pairs, ``sigmoid(scale * <user, item>)``, (B, 1)."""

    def __init__(self, scale=10.0, entropy_weight=0.0, item_bias=None, distinct_items=False):
        self.scale = float(scale)
        if not 0.0 < self.scale < float('inf'):
            raise ValueError("scale must be positive and finite (got %r)" % (scale,))
        self.entropy_weight = float(entropy_weight)
        self.item_bias = None if item_bias is None else torch.as_tensor(item_bias, dtype=torch.float32).reshape(-1)
        self.distinct_items = bool(distinct_items)

    @property
    def needs_items(self):
        """Whether ``loss`` has to be told the items' rows in the catalog."""
        return self.item_bias is not None or self.distinct_items

    def parameters(self):
        return []

    def __call__(self, x_out):
        user_emb, item_emb = x_out
        return torch.sigmoid(self.scale * (user_emb * item_emb).sum(dim=-1, keepdim=True))

    def loss(self, x_out, targets, item_bias=None, items=None):
        """(loss, the pairs' scores (B, 1)).  ``items``: the rows of the batch's items in the catalog, whole numbers on the
        embeddings' device."""
        user_emb, item_emb = (x.contiguous() for x in x_out)
        n, dev = user_emb.shape[0], user_emb.device
        positive = torch.as_tensor(targets, dtype=torch.float32, device=dev).reshape(-1) > 0.5
        if positive.numel() != n or item_emb.shape[0] != n:
            raise ValueError("one target and one item per user are needed (%d users, %d items, %d targets)" %
                             (n, item_emb.shape[0], positive.numel()))
        if self.needs_items and items is None:
            raise ValueError("item_bias and distinct_items of the head need the batch's items")
        if items is not None and items.numel() != n:
            raise ValueError("%d items for %d links" % (items.numel(), n))
        if item_bias is None and self.item_bias is not None:
            item_bias = self._bias_of(items.reshape(-1))
        own = torch.arange(n, dtype=torch.int32, device=dev)
        if self.distinct_items:
            first = _first_places(items.reshape(-1))
            repeated = first != own
            own = first.to(torch.int32)
            item_bias = torch.zeros(n, device=dev) if item_bias is None else item_bias
            item_bias = torch.where(repeated, torch.full_like(item_bias, -math.inf), item_bias)
        log_prob, entropy = _ag.CatalogLogProbs.apply(user_emb, item_emb, torch.where(positive, own, -1).to(torch.int32), item_bias,
                                                      self.scale)
        loss = -log_prob.sum() / positive.sum().clamp(min=1) - self.entropy_weight * entropy.mean()
        with torch.no_grad():
            pred = self((user_emb, item_emb))
        return loss, pred

    def _bias_of(self, items):
        if self.item_bias.device != items.device:
            self.item_bias = self.item_bias.to(items.device)
        n = self.item_bias.numel()
        if n == 0:
            raise ValueError("the head's item_bias is empty")
        inside = (items >= 0) & (items < n)                   # (an item that the catalog does not have: NaN, not another's)
        bias = self.item_bias[torch.where(inside, items, torch.zeros_like(items)).long()]
        return torch.where(inside, bias, torch.full_like(bias, math.nan))

    @torch.no_grad()
    def recommend(self, user_emb, item_emb, k, item_bias=None):
        """(item indices int32 (N, k), their log probabilities (N, k)), best first; an item whose bias is -inf is never
        among them (``kernels.catalog_log_probs``)."""
        r = kernels.catalog_log_probs(user_emb.contiguous(), item_emb.contiguous(), bias=item_bias, scale=self.scale, top_k=k)
        return r.top_ids, r.top_log_prob


def link_ranking(scale=10.0, entropy_weight=0.0, item_bias=None, distinct_items=False):
    """The edge function of ``CatalogHead``, taken like those of ``link_inference``."""
    head = CatalogHead(scale, entropy_weight, item_bias, distinct_items)

    def edge_function(x_out, seed=None):
        x_out.build()
        return head

    return edge_function
