"""Ranks that share a ``dropout_seed`` drop other positions: two gloo processes on the CPU, the kernel replaced by a formula of
seed and block."""
import os
import socket

import numpy as np
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

import graphsage_amd as ga
from graphsage_amd import kernels
from graphsage_amd.train import LinkHead, Trainer


def _model(seed):
    edges = np.array([[0, 1, 2, 3, 4, 3], [3, 4, 3, 0, 1, 2]])
    g = ga.Graph({'user': np.zeros((3, 2)), 'item': np.zeros((2, 2))}, {'user': [0, 1, 2], 'item': [3, 4]}, edges)
    gen = ga.GraphSAGEGenerator(g, 2, [2, 2], head_node_types=['user', 'item'], seed=3)
    return ga.GraphSAGE([4, 4], gen, dropout=0.5, dropout_seed=seed, seed=1).build(device='cpu')


def _worker(rank, world, port, out_dir):
    os.environ['MASTER_ADDR'] = '127.0.0.1'
    os.environ['MASTER_PORT'] = str(port)
    dist.init_process_group('gloo', rank=rank, world_size=world)
    try:
        begins = []
        kernels.dropout = lambda x, rate, seed, offset: begins.append(offset) or x
        model = _model(7)
        Trainer(model, head=LinkHead(4, 'cpu', seed=1), engine='autograd')
        x = torch.ones(4, 25)
        drop = model._dropper()
        drop(x), drop(x), model._dropper(1000)(x)
        plain = _model(None)
        Trainer(plain, head=LinkHead(4, 'cpu', seed=1), engine='autograd')
        assert plain.dropout_base == 0
        torch.save(torch.tensor(begins), os.path.join(out_dir, 'r%d.pt' % rank))
    finally:
        dist.destroy_process_group()


def test_ranks_draw_from_stretches_that_do_not_meet(tmp_path):
    s = socket.socket()
    s.bind(('127.0.0.1', 0))
    port = s.getsockname()[1]
    s.close()
    mp.spawn(_worker, args=(2, port, str(tmp_path)), nprocs=2, join=True)
    begins = [torch.load(tmp_path / ('r%d.pt' % r), weights_only=True).tolist() for r in range(2)]
    assert begins[0] == [0, 13, 1000]
    assert begins[1] == [(1 << 48) + b for b in begins[0]]


def test_one_process_begins_at_the_first_block():
    model = _model(7)
    Trainer(model, head=LinkHead(4, 'cpu', seed=1), engine='autograd')
    assert model.dropout_base == 0
