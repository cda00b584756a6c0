"""Two-type GraphSAGE layer stack for user-item link batches.

Constructor and call convention of the reference's ``GraphSAGE``
(``models.py:14-245``): ``GraphSAGE(layer_sizes, generator, agg_option, bias,
dropout, normalize)``, ``model(xin)`` on the batch the generator produced gives
``[user_embedding, item_embedding]``, each ``(B, layer_sizes[-1])``.

Layer wiring (``models.py:48-90,134-190``), stated directly instead of through
the reference's generic tree walk: with L hops the batch has slots
``s = 2*h + side`` (``h`` = hop, ``side`` = which head the walk started from);
layer ``l`` keeps slots ``0 .. 2*(L-l)-1``; slot ``s`` aggregates itself (head)
with slot ``s + 2`` (its sampled neighbors, ``n_samples[h]`` per head node); one
weight set exists per (layer, node type of the head slot) and is shared by all
slots of that type in the layer; activations are relu except linear on the last
layer; the surviving two slots are reshaped to ``(B, H)`` and l2-normalised.

Two execution paths produce the same numbers:

* dense -- ``xin`` is a list of ``(B, n, F)`` tensors (the reference's input
  format): every layer is neighbor mean + projection on materialised tensors;
* fused -- ``xin`` is the generator's ``BatchFeatures``: layer 0 reads the
  deepest slots straight from the feature tables through their sampled ids
  (``gs_gather_mean_fwd``), so the largest tensors of the batch, ``(B, n0*n1, F)``,
  are never written or read back.

Two arguments beyond the reference's: ``agg_option='attention'`` with ``heads`` (``Aggregator``), and ``dropout_seed``.
Without it dropout draws from torch's generator and torch keeps the masks; with it every mask is a function of the seed
and of how much has been drawn before (``gs_dropout``), drawn again in the backward pass and never stored.
What has been drawn is counted on the host, call by call: a step that is captured into a graph replays its masks unless the
seed is an int64 tensor in GPU memory that the caller changes in between, and a forward pass that the backward pass runs
again (``torch.utils.checkpoint``) would draw others, which is refused.  There, and wherever a call has to be repeatable,
``model(batch, dropout_offset=n)`` says where its masks begin: the n-th block of eight elements under the seed, whatever was
drawn before (``step << 24`` keeps steps of up to 2^27 elements apart).
A seed is one sequence of masks for every process that has it.  The ranks of a ``Trainer`` begin 2^48 blocks apart
(``dropout_base``), so that they drop other positions; processes that train otherwise take seeds of their own.
"""
import itertools as it
import operator as op
import threading

from . import autograd as _ag
from ._lib import GsageError
from .utils import Aggregator

__all__ = ['GraphSAGE']


_drawing = threading.Lock()                                  # threads that share a model draw one after the other


class GraphSAGE:
    def __init__(self, layer_sizes, generator=None, agg_option='mean', bias=True, dropout=0.0,
                 normalize="l2", seed=None, heads=1, dropout_seed=None):
        self._aggregator = Aggregator
        self.agg_option = agg_option
        self.normalize = normalize
        if generator is not None:
            self._get_sizes_from_generator(generator)
        else:
            raise ValueError("Generator must be inserted")
        self.n_layers = len(self.n_samples)
        if len(layer_sizes) != self.n_layers:
            raise ValueError("one layer size per hop is needed (%d hops, %d sizes)" %
                             (self.n_layers, len(layer_sizes)))
        self.bias = bias
        self.dropout = dropout
        self.heads = heads
        self.dropout_seed = dropout_seed
        self._dropout_drawn = 0                              # blocks of eight elements drawn under the seed so far
        self.dropout_base = 0                                # the block this process begins with
        self.training = True
        n_slots = len(self.subtree_schema)

        # slots alive at the input of each layer, with their neighbor slot
        self.neigh_trees = [self.subtree_schema[:2 * (self.n_layers - layer)] for layer in range(self.n_layers)]
        self._depths = [s // 2 for s in range(n_slots)]
        types = sorted({t for t, _ in self.subtree_schema}, reverse=True)      # ['user', 'item']
        self.dims = [dict(self.input_dims)] + [{t: int(size) for t in types} for size in layer_sizes]
        self.activations = ["relu"] * (self.n_layers - 1) + ["linear"]
        self._aggs = [
            {
                node_type: self._aggregator(
                    output_dim, has_bias=self.bias, activation_function=self.activations[layer],
                    agg_option=self.agg_option, heads=self.heads,
                    seed=None if seed is None else seed * 1000 + layer * 10 + ti)
                for ti, (node_type, output_dim) in enumerate(self.dims[layer + 1].items())
            }
            for layer in range(self.n_layers)
        ]

    def __repr__(self):
        return "<GraphSAGE model with {} layers>".format(self.n_layers)

    def _get_sizes_from_generator(self, generator):
        self.input_dims = generator.graph.node_feature_sizes
        self.n_samples = generator.num_samples
        self.subtree_schema = generator.type_adjacency_list

    # ---- parameters ---------------------------------------------------------
    def build(self, device=None):
        """Creates every aggregator's weights (Keras does this on first call)."""
        for layer in range(self.n_layers):
            for node_type, agg in self._aggs[layer].items():
                if agg.built:
                    continue
                other = [t for t in self.dims[layer] if t != node_type][0]
                agg.build([(None, 1, self.dims[layer][node_type]),
                           (None, 1, 1, self.dims[layer][other])], device=device)
        return self

    def parameters(self):
        return [p for layer in self._aggs for agg in layer.values() for p in agg.parameters()]

    def named_parameters(self):
        out = {}
        for layer, aggs in enumerate(self._aggs):
            for node_type, agg in aggs.items():
                out['l%d.%s.w_self' % (layer, node_type)] = agg.w_self
                out['l%d.%s.w_neigh' % (layer, node_type)] = agg.w_neigh
                if agg.bias is not None:
                    out['l%d.%s.bias' % (layer, node_type)] = agg.bias
                if agg.w_query is not None:
                    out['l%d.%s.w_query' % (layer, node_type)] = agg.w_query
        return out

    def train(self, mode=True):
        self.training = mode
        return self

    def eval(self):
        return self.train(False)

    # ---- forward ------------------------------------------------------------------
    def _dropper(self, offset=None):
        """Dropout as one call of the model applies it; ``offset``: the block its first mask begins with."""
        if offset is not None and self.dropout_seed is None:
            raise ValueError("dropout_offset needs a model with a dropout_seed")
        if not (self.dropout and self.training):
            return lambda x: x
        import torch
        if self.dropout_seed is None:
            return lambda x: torch.nn.functional.dropout(x, p=self.dropout, training=True)
        drawn = None if offset is None else int(offset)
        if drawn is not None and drawn < 0:
            raise ValueError("dropout_offset must not be negative")

        def drop(x):
            nonlocal drawn
            blocks = (x.numel() + 7) // 8
            if drawn is not None:
                first, drawn = drawn, drawn + blocks
            else:
                if torch._C._current_graph_task_id() != -1:
                    raise GsageError("a forward pass run again by the backward pass would draw other masks than the first one: "
                                     "call the model with dropout_offset")
                with _drawing:
                    first = self._dropout_drawn
                    self._dropout_drawn += blocks
            return _ag.Dropout.apply(x.contiguous(), self.dropout, self.dropout_seed, self.dropout_base + first)
        return drop

    def _finish(self, h):
        out = [x.reshape(x.shape[0], x.shape[2]) for x in h if x.shape[1] == 1]
        if self.normalize == "l2":
            out = [_ag.L2Normalize.apply(x.contiguous()) for x in out]
        return out[0] if len(out) == 1 else out

    def _dense_layer(self, h, layer, drop):
        out = []
        for i, (node_type, neigh_indices) in enumerate(self.neigh_trees[layer]):
            j = neigh_indices[0]
            heads = h[i].shape[1]
            n = self.n_samples[self._depths[i]]
            f_neigh = self.dims[layer][self.subtree_schema[j][0]]
            x_neigh = drop(h[j].reshape(h[j].shape[0], heads, n, f_neigh))
            out.append(self._aggs[layer][node_type]([drop(h[i]), x_neigh]))
        return out

    def _fused_first_layer(self, batch):
        alive = self.neigh_trees[0]
        b = batch.head_size
        x_self = []
        for i, (node_type, _) in enumerate(alive):
            feat, off = batch.table(node_type)
            x_self.append(_ag.GatherRows.apply(feat, batch.ids[i].reshape(-1), off))
        out = []
        for i, (node_type, neigh_indices) in enumerate(alive):
            j = neigh_indices[0]
            m = x_self[i].shape[0]
            n = self.n_samples[self._depths[i]]
            agg = self._aggs[0][node_type]
            if self.agg_option == 'attention':
                if j < len(alive):
                    x_mean = agg.attend(x_self[i], x_self[j], None, n)
                else:
                    feat, off = batch.table(self.subtree_schema[j][0])
                    x_mean = agg.attend(x_self[i], feat, batch.ids[j].reshape(-1), n, off)
                out.append(agg.project(x_self[i], x_mean).reshape(b, m // b, agg.output_dim))
                continue
            group, gather = ((_ag.GroupMax, _ag.GatherMax) if self.agg_option == 'max'
                             else (_ag.GroupMean, _ag.GatherMean))
            if j < len(alive):            # neighbor slot is itself gathered: mean (max) of those rows
                x_mean = group.apply(x_self[j].reshape(m, n, -1), m, n)
            else:                          # deepest slot: rows are reduced as they are fetched
                feat, off = batch.table(self.subtree_schema[j][0])
                x_mean = gather.apply(feat, batch.ids[j].reshape(-1), m, n, off)
            out.append(agg.project(x_self[i], x_mean).reshape(b, m // b, agg.output_dim))
        return out

    def __call__(self, xin, dropout_offset=None):
        self.build()
        drop = self._dropper(dropout_offset)
        self.layer_tensors = []
        from .generator import BatchFeatures
        if isinstance(xin, BatchFeatures) and not (self.dropout and self.training):
            h = self._fused_first_layer(xin)
            self.layer_tensors.append(h)
            first = 1
        else:
            h = [xin[i] for i in range(len(self.subtree_schema))]
            first = 0
        for layer in range(first, self.n_layers):
            h = self._dense_layer(h, layer, drop)
            self.layer_tensors.append(h)
        return self._finish(h)

    # ---- shapes -------------------------------------------------------------------
    def _input_shapes(self):
        """(nodes per head, feature size) of every slot."""
        sizes = list(it.accumulate([1] + list(self.n_samples), op.mul))
        return [(sizes[self._depths[s]], self.input_dims[t]) for s, (t, _) in enumerate(self.subtree_schema)]

    def in_out_tensors(self):
        """The reference returns Keras placeholders and the symbolic output
        (``models.py:229-245``); without a graph-building framework the
        equivalent is the list of per-slot input shapes and the model itself as
        the function from a batch to ``[user_embedding, item_embedding]``."""
        return self._input_shapes(), self
