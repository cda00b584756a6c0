"""Counter-based dropout against the generator restated on the CPU -- needs a GPU.  Masks are compared exactly, kept values
within half a step of their type (x * scale is one product in fp32, rounded once more for 16-bit types: together at most
eps_t / 2 + 2^-24 of the value)."""
import numpy as np
import pytest
import torch

from graphsage_amd import _lib, autograd, kernels
from oracle import philox

pytestmark = pytest.mark.gpu


def _pieces(n, seed, offset):
    block = np.arange((n + 7) // 8, dtype=np.uint64) + np.uint64(offset)
    words = philox.philox4x32_10(block & np.uint64(0xFFFFFFFF), block >> np.uint64(32), 0x50000000, 0,
                                 seed & 0xFFFFFFFF, seed >> 32)
    words = np.stack(words, 1).astype(np.uint32)
    return np.stack([words & 0xFFFF, words >> 16], 2).reshape(-1)[:n]


def _check(x, rate, seed, offset, got):
    t = int(rate * 65536)
    keep = torch.from_numpy(_pieces(x.numel(), seed, offset) >= t).reshape(x.shape).to(x.device)
    assert not got[~keep].any()
    want = x.double() * (65536.0 / (65536 - t))
    off = (got.double() - want).abs()[keep]
    tol = (want.abs() * (torch.finfo(x.dtype).eps / 2 + 2.0 ** -24) * 1.001)[keep]
    if x.dtype == torch.float16:
        tol = tol + 2.0 ** -25                        # below the normal range
    assert bool((off <= tol).all())
    return keep


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('n', [1, 2, 7, 8, 9, 15, 16, 17, 255, 2049, 100003])
def test_mask_and_values(cuda, dtype, n):
    g = torch.Generator(device='cuda').manual_seed(n)
    x = torch.randn(n + 1, generator=g, device='cuda').to(dtype)
    for view in (x[:n], x[1:]):                       # on a 16-byte border and one element behind it
        for rate, seed, offset in [(0.3, 12345, 0), (0.5, (1 << 63) + 77, 5), (0.0, 3, 1), (0.999, 9, (1 << 40))]:
            got = kernels.dropout(view, rate, seed, offset)
            assert got.dtype == dtype and got.shape == view.shape
            _check(view, rate, seed, offset, got)


def test_a_rate_of_zero_copies_and_shapes_are_kept(cuda):
    x = torch.randn(3, 5, 7, device='cuda')
    assert torch.equal(kernels.dropout(x, 0.0, 1), x)
    assert kernels.dropout(x[:0], 0.4, 1).shape == (0, 5, 7)


def test_blocks_continue_under_an_offset_that_passes_32_bits(cuda):
    x = torch.ones(8 * 100, device='cuda')
    whole = kernels.dropout(x, 0.5, 42, (1 << 32) - 50)
    assert torch.equal(whole[400:], kernels.dropout(x[400:], 0.5, 42, 1 << 32))
    _check(x, 0.5, 42, (1 << 32) - 50, whole)


def test_more_elements_than_32_bits_count(cuda):
    n = (1 << 32) + 8 * 3 + 5
    x = torch.ones(n, dtype=torch.bfloat16, device='cuda')
    kernels.dropout(x, 0.5, 7, 0, out=x)
    for lo in (0, (1 << 31) - 64, (1 << 32) - 64):
        part = x[lo:lo + 93]
        _check(torch.ones_like(part), 0.5, 7, lo // 8, part)
    kept = sum(int((x[i:i + (1 << 30)] != 0).sum()) for i in range(0, n, 1 << 30))
    assert abs(kept / n - 0.5) < 5 * 0.5 / n ** 0.5   # five standard deviations


def test_what_is_dropped_may_be_anything(cuda):
    x = torch.full((4096,), float('nan'), device='cuda')
    got = kernels.dropout(x, 0.5, 3)
    keep = torch.from_numpy(_pieces(4096, 3, 0) >= 32768).cuda()
    assert not got[~keep].any() and bool(got[keep].isnan().all())


def test_seed_in_memory_other_streams_and_replayed_graphs(cuda):
    x = torch.randn(1000, device='cuda')
    seed = torch.tensor([-5], dtype=torch.int64, device='cuda')
    want = kernels.dropout(x, 0.4, (1 << 64) - 5, 11)
    assert torch.equal(kernels.dropout(x, 0.4, seed, 11), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = kernels.dropout(x, 0.4, seed, 11)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = kernels.dropout(x, 0.4, seed, 11)
    for value in (3, 4, 3):
        seed.fill_(value)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, kernels.dropout(x, 0.4, value, 11))


def test_in_place_and_gradient(cuda):
    x = torch.randn(777, device='cuda')
    want = kernels.dropout(x, 0.25, 6, 2)
    leaf = x.clone().requires_grad_()
    y = autograd.Dropout.apply(leaf, 0.25, 6, 2)
    assert torch.equal(y, want)
    g = torch.randn(777, device='cuda')
    y.backward(g)
    assert torch.equal(leaf.grad, kernels.dropout(g, 0.25, 6, 2))
    seed = torch.tensor([6], dtype=torch.int64, device='cuda')
    leaf.grad = None
    y = autograd.Dropout.apply(leaf, 0.25, seed, 2)
    seed.fill_(9)                                     # the gradient goes by the mask that was drawn
    y.backward(g)
    assert torch.equal(leaf.grad, kernels.dropout(g, 0.25, 6, 2))
    assert kernels.dropout(x, 0.25, 6, 2, out=x) is x and torch.equal(x, want)


def test_refusals(cuda):
    x = torch.zeros(64, device='cuda')
    for bad, err in [(lambda: kernels.dropout(x.cpu(), 0.1, 1), _lib.GsageError),
                     (lambda: kernels.dropout(x.double(), 0.1, 1), TypeError),
                     (lambda: kernels.dropout(x[::2], 0.1, 1), ValueError),
                     (lambda: kernels.dropout(x, 1.0, 1), ValueError),
                     (lambda: kernels.dropout(x, -0.1, 1), ValueError),
                     (lambda: kernels.dropout(x, float('nan'), 1), ValueError),
                     (lambda: kernels.dropout(x, 0.1, 1, out=x[:8]), ValueError),
                     (lambda: kernels.dropout(x, 0.1, 1, out=x.half()), TypeError),
                     (lambda: kernels.dropout(x[:32], 0.1, 1, out=x[8:40]), _lib.GsageError),
                     (lambda: kernels.dropout(x, 0.1, torch.zeros(1, device='cuda')), TypeError),
                     (lambda: kernels.dropout(x, 0.1, torch.zeros(2, dtype=torch.int64, device='cuda')), ValueError)]:
        with pytest.raises(err):
            bad()
