"""Attention over neighbors on both sides of the borders between its forms, against the formulas in 64 bits -- needs a
GPU.  Bounds and cases are those of test_gpu_attention.py."""
import pytest
import torch

from test_gpu_attention import _case, _check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('heads', [1, 4])
@pytest.mark.parametrize('dim,dtype,lanes', [(16, torch.float32, 4), (32, torch.float32, 8), (64, torch.bfloat16, 8), (64, torch.float32, 16),
                                             (128, torch.float16, 16), (100, torch.float32, 32), (200, torch.float32, 64)])
def test_lists_around_a_wave_for_every_simd(cuda, heads, dim, dtype, lanes):
    full = 1024 * 64 // lanes
    for lists, child in ((full - 1, 13), (full, 13), (full, 32), (full, 33), (full + 1, 20)):
        if lists * child * heads * dim > 40_000_000:
            continue
        _check(_case(lists + child, dtype, lists, heads, 1, dim, 900, child=child, shared=True))


@pytest.mark.parametrize('ids', [True, False])
@pytest.mark.parametrize('child', [12, 13])
def test_few_lists_around_the_length_taken_always(cuda, ids, child):
    for lists in (1, 3, 100):
        _check(_case(child + lists, torch.float32, lists, 2, 1, 48, 70 if ids else lists * child, child=child, ids=ids, masked=0.2 if ids else 0))


@pytest.mark.parametrize('heads,mean', [(1, 8), (2, 6), (3, 4), (4, 4)])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_rows_around_the_mean_taken_by_runs(cuda, heads, mean, dtype):
    parents, child = 1200, 10
    for rows in (parents * child // mean, parents * child // mean - 1, parents * child // mean + 1):
        for shared, dim in ((True, 64), (False, 19)):
            _check(_case(rows + heads, dtype, parents, heads, 1, dim, rows, child=child, shared=shared))
