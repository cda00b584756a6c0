"""First places of repeated items, on the CPU."""
import pytest
import torch

from graphsage_amd.link_utils import CatalogHead, _first_places


@pytest.mark.parametrize('ids', [[], [5], [3, 3, 3], [4, 1, 4, 2, 1, 1, 9], list(range(40, 0, -1)), [-1, 7, -1, 7]])
def test_first_places(ids):
    got = _first_places(torch.tensor(ids, dtype=torch.int32))
    assert got.tolist() == [ids.index(x) for x in ids]


def test_what_the_head_needs():
    assert not CatalogHead().needs_items
    assert CatalogHead(item_bias=[0.0, 1.0]).needs_items and CatalogHead(distinct_items=True).needs_items
