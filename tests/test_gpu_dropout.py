"""Counter-based dropout against Philox4x32-10 in numpy: the same elements dropped, survivors within
one rounding."""
from __future__ import annotations

import math

import pytest
import torch

import training_reference as R

pytestmark = pytest.mark.gpu

STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TYPES = list(STEP)


def _rng(seed, position, device):
    return torch.tensor([seed, position], dtype=torch.int64, device=device)


def _expect(x, p, seed, position, residual=None):
    keep, scale = R.dropout_keep(x.numel(), p, seed, position)
    y = torch.where(keep.view(x.shape), x.cpu().double() * scale, torch.zeros((), dtype=torch.float64))
    return y if residual is None else y + residual.cpu().double(), keep.view(x.shape)


def _close(got, ref, size, dtype):
    # the product (and the sum) in fp32, then one rounding; fp16 results below 2^-14 have an absolute step
    bound = STEP[dtype] * ref.abs() + 2 * 2.0 ** -23 * size + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    assert float(((got.cpu().double() - ref).abs() - bound).max()) <= 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 7, 8, 9, 255, 2048, 2049, 769 * 33])
@pytest.mark.parametrize("with_residual", [False, True])
def test_against_the_generator(pe, cuda_device, dtype, n, with_residual):
    from flash_modernbert_b200 import ops

    gen = torch.Generator().manual_seed(n)
    x = torch.randn(n, generator=gen).to(dtype)
    residual = torch.randn(n, generator=gen).to(dtype) if with_residual else None
    for p, seed, position in ((0.1, 0, 0), (0.5, 2 ** 62 + 12345, 2 ** 32 - 3), (0.9, -7, 2 ** 63 - 2)):
        got = ops.dropout(x.to(cuda_device), p, _rng(seed, position, cuda_device),
                          residual=None if residual is None else residual.to(cuda_device))
        ref, _ = _expect(x, p, seed % 2 ** 64, position, residual)
        size = x.double().abs() / (1 - p) + (0 if residual is None else residual.double().abs())
        assert got.dtype == dtype and got.shape == x.shape
        _close(got, ref, size, dtype)


def test_known_answer(pe, cuda_device):
    """The published first block of Philox4x32-10 for counter 0 and key 0."""
    import numpy as np

    from flash_modernbert_b200 import ops

    words = [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert R.philox(np.zeros(1, dtype=np.uint64), 0)[0].tolist() == words
    fields = [f for w in words for f in (w & 0xFFFF, w >> 16)]
    for p in (0.2, 0.5, 0.8):
        got = ops.dropout(torch.ones(8, device=cuda_device), p, _rng(0, 0, cuda_device)) != 0
        assert got.tolist() == [f >= math.floor(p * 65536 + 0.5) for f in fields]


@pytest.mark.parametrize("dtype", TYPES)
def test_extremes(pe, cuda_device, dtype):
    """p = 0 keeps, p = 1 drops all; a dropped NaN or infinity leaves no trace; empty tensors pass."""
    from flash_modernbert_b200 import ops

    rng = _rng(3, 5, cuda_device)
    x = torch.randn(1001, device=cuda_device).to(dtype)
    assert torch.equal(ops.dropout(x, 0.0, rng), x)
    assert torch.equal(ops.dropout(torch.full_like(x, math.nan), 1.0, rng, residual=x), x)
    bad = torch.full_like(x, math.inf)
    keep = R.dropout_keep(1001, 0.5, 3, 5)[0]
    assert torch.equal(torch.isinf(ops.dropout(bad, 0.5, rng)).cpu(), keep)
    assert ops.dropout(x[:0], 0.5, rng).shape == (0,)


def test_layout_does_not_matter(pe, cuda_device):
    from flash_modernbert_b200 import ops

    rng = _rng(11, 2 ** 40, cuda_device)
    x = torch.randn(65, 70, device=cuda_device).to(torch.bfloat16)
    y = ops.dropout(x, 0.3, rng, residual=x)
    assert torch.equal(ops.dropout(x.t().contiguous().t(), 0.3, rng, residual=x), y)
    off = torch.empty(x.numel() + 1, dtype=x.dtype, device=cuda_device)[1:].view_as(x).copy_(x)
    assert off.data_ptr() % 16 != 0
    assert torch.equal(ops.dropout(off, 0.3, rng, residual=x), y)
    assert torch.equal(ops.dropout(x, 0.3, rng, residual=off), y)


def test_share_of_dropped(pe, cuda_device):
    """2^22 draws: the share dropped is within five standard deviations, and blocks do not repeat."""
    from flash_modernbert_b200 import ops

    n = 1 << 22
    x = torch.ones(n, device=cuda_device)
    for p in (0.1, 0.5):
        dropped = ops.dropout(x, p, _rng(77, 0, cuda_device)) == 0
        assert abs(float(dropped.double().mean()) - p) < 5 * math.sqrt(p * (1 - p) / n) + 2.0 ** -17
        both = float((dropped & dropped.roll(8)).double().mean())
        assert abs(both - p * p) < 5 * math.sqrt(p * p / n) + 2.0 ** -16


def test_gradient_uses_the_forward_numbers(pe, cuda_device):
    """Through autograd, even after the program has moved its generator on; the residual passes through."""
    from flash_modernbert_b200 import ops

    for dtype in TYPES:
        rng = _rng(5, 100, cuda_device)
        x = torch.randn(37, 21, device=cuda_device).to(dtype).requires_grad_(True)
        r = torch.randn(37, 21, device=cuda_device).to(dtype).requires_grad_(True)
        y = ops.dropout(x, 0.4, rng, residual=r)
        rng[1] += ops.dropout_positions(x.numel())
        dy = torch.randn(37, 21, device=cuda_device).to(dtype)
        y.backward(dy)
        ref, keep = _expect(dy, 0.4, 5, 100)
        _close(x.grad, ref, dy.cpu().double().abs() / 0.6, dtype)
        assert torch.equal(r.grad, dy)
        assert torch.equal(ops.dropout_backward(dy, 0.4, _rng(5, 100, cuda_device)), x.grad)
        again = ops.dropout(x.detach(), 0.4, rng)
        assert not torch.equal(again == 0, x.grad == 0)


def test_gradient_against_differences(pe, cuda_device):
    from flash_modernbert_b200 import ops

    rng = _rng(9, 9, cuda_device)
    x = torch.randn(500, device=cuda_device, requires_grad=True)
    dy = torch.randn(500, device=cuda_device)
    (g,) = torch.autograd.grad(ops.dropout(x, 0.25, rng), x, dy)
    v = torch.randn(500, device=cuda_device)
    with torch.no_grad():
        up, down = ((ops.dropout(x + s * v, 0.25, rng).double() * dy.double()).sum() for s in (1.0, -1.0))
    # the map is linear: the difference is exact but for fp32 roundings of 500 terms of size 10 or less
    assert abs(float((up - down) / 2 - (g.double() * v.double()).sum())) < 500 * 10 * 2.0 ** -23


def test_captured_call_reads_the_generator_at_replay(pe, cuda_device):
    from flash_modernbert_b200 import ops

    rng = _rng(21, 0, cuda_device)
    x = torch.ones(4096, device=cuda_device)
    ops.dropout(x, 0.5, rng)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.dropout(x, 0.5, rng)
        rng[1] += ops.dropout_positions(x.numel())
    for step in range(3):
        graph.replay()
        assert torch.equal((y != 0).cpu(), R.dropout_keep(4096, 0.5, 21, 512 * step)[0])
