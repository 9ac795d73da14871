"""Token log-probabilities, entropy and top alternatives with their gradient against log-softmax in
64 bits."""
from __future__ import annotations

import math

import pytest
import torch

import training_reference as R

pytestmark = pytest.mark.gpu

STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TYPES = list(STEP)
# Sums of up to 2^18 exponentials in fp32, each good to 2^-21, joined pairwise: 2^-18 relative for
# the sum covers it, hence 2^-18 absolute for its logarithm; the difference x - lse adds half a step
# of fp32 of its size.
TOL = 2.0 ** -18


def _inputs(rows, vocab, dtype, device, seed=0, scale=3.0):
    gen = torch.Generator(device=device).manual_seed(seed)
    logits = (torch.randn(rows, vocab, generator=gen, device=device) * scale).to(dtype)
    targets = torch.randint(0, vocab, (rows,), generator=gen, device=device)
    return logits, targets


def _check_forward(r, logits, targets, top_k, ignore_index=-100):
    lp, ent, lse, ids, top = R.logprobs(logits, targets, top_k, ignore_index)
    size = 2.0 ** -23 * (logits.double().masked_fill(logits == -math.inf, 0).abs().amax(-1) + lse.abs())
    assert float(((r.logprobs.double() - lp).abs() - TOL - size).max()) <= 0
    assert float(((r.lse.double() - lse).abs() - TOL - size).max()) <= 0
    # the entropy is log s - w / s, both relative to the row's maximum
    assert float(((r.entropy.double() - ent).abs() - 4 * TOL * (1 + ent)).max()) <= 0
    if top_k:
        assert torch.equal(r.top_ids, ids)
        assert float(((r.top_logprobs.double() - top).abs() - TOL - size.unsqueeze(-1)).nan_to_num(0.0).max()) <= 0
    else:
        assert r.top_ids is None and r.top_logprobs is None


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,top_k", [(1, 1, 1), (2, 2, 2), (5, 31, 0), (3, 32, 32), (7, 501, 5), (4, 4095, 20),
                                              (300, 1000, 3), (1, 50368, 20), (3, 50368, 1), (40, 30011, 32),
                                              (160, 8193, 7), (2, 256001, 20)])
def test_forward(pe, cuda_device, dtype, rows, vocab, top_k):
    from flash_modernbert_b200 import ops

    logits, targets = _inputs(rows, vocab, dtype, cuda_device, seed=rows + vocab)
    _check_forward(ops.token_logprobs(logits, targets, top_k=top_k), logits, targets, top_k)
    ops.check_status(cuda_device)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [50, 5000, 50368])
@pytest.mark.parametrize("order", ["equal", "ascending", "descending", "few"])
def test_ties_and_orders(pe, cuda_device, dtype, vocab, order):
    """Rows of equal values, sorted rows and rows of three values: exact ids, the lowest index first."""
    from flash_modernbert_b200 import ops

    base = torch.arange(vocab, device=cuda_device, dtype=torch.float64)
    values = {"equal": torch.full_like(base, -1.5), "ascending": base / vocab * 8, "descending": -base / vocab * 8,
              "few": (base * 7919) % 3}[order]
    logits = values.to(dtype).expand(3, vocab).contiguous()
    targets = torch.tensor([0, vocab // 2, vocab - 1], device=cuda_device)
    for k in (1, 20, 32):
        _check_forward(ops.token_logprobs(logits, targets, top_k=k), logits, targets, k)


@pytest.mark.parametrize("dtype", TYPES)
def test_masked_logits(pe, cuda_device, dtype):
    """-inf and the type's lowest value as masks, a single survivor, a row of nothing but the lowest
    value; NaN, +inf and rows of -inf give NaN like log-softmax and leave their neighbours alone."""
    from flash_modernbert_b200 import ops

    vocab = 9000
    logits, targets = _inputs(9, vocab, dtype, cuda_device, seed=3)
    low = torch.finfo(dtype).min
    logits[1, ::2] = -math.inf
    logits[2, ::2] = low
    logits[3] = -math.inf
    logits[3, 4321] = 2.0
    targets[3] = 4321
    logits[4] = low
    logits[5, 17] = math.nan
    logits[6, 8999] = math.inf
    logits[7] = -math.inf
    targets[1], targets[2] = 7, 7
    r = ops.token_logprobs(logits, targets, top_k=4)
    good = [0, 1, 2, 3, 4, 8]
    part = type(r)(*(t[good] for t in r))
    assert abs(float(r.logprobs[4]) + math.log(vocab)) <= TOL  # log s does not drown in the row's size
    _check_forward(part, logits[good], targets[good], 4)
    assert float(r.logprobs[3]) == 0.0 and float(r.entropy[3]) == 0.0
    for row in (5, 6, 7):
        assert math.isnan(float(r.logprobs[row])) and math.isnan(float(r.entropy[row]))
    assert r.top_ids[5, 0] == 17 and r.top_ids[6, 0] == 8999 and r.top_ids[7].tolist() == [0, 1, 2, 3]
    g = torch.ones(9, device=cuda_device)
    grad = ops.token_logprobs_backward(logits, targets, r, g, g)
    ref = R.logprobs_gradient(logits, targets, g, g, torch.zeros_like(g))
    assert float((grad[good].double() - ref[good]).abs().max()) <= (STEP[dtype] + 2.0 ** -12) * float(ref[good].abs().max())
    assert bool((grad[1, ::2] == 0).all()) and bool((grad[2, ::2] == 0).all())
    assert torch.isnan(grad[5]).all()


def _gradient_bound(ref, logits, dtype):
    # p is good to 2^-18 relative (above) plus the fp32 exponent's own error, 2^-23 of |x - lse| log2 e;
    # then one rounding, with an absolute floor where the type runs out of exponent
    span = float(logits.double().masked_fill(logits == -math.inf, 0).abs().max()) * 2
    floor = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -126}[dtype]
    return STEP[dtype] * ref.abs() + floor, 2.0 ** -17 + span * 2.0 ** -22


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 31), (6, 502), (5, 8191), (2, 50368), (1, 256001)])
def test_gradient(pe, cuda_device, dtype, rows, vocab):
    from flash_modernbert_b200 import ops

    logits, targets = _inputs(rows, vocab, dtype, cuda_device, seed=vocab)
    gen = torch.Generator(device=cuda_device).manual_seed(1)
    g, h, z = (torch.randn(rows, generator=gen, device=cuda_device) for _ in range(3))
    r = ops.token_logprobs(logits, targets)
    got = ops.token_logprobs_backward(logits, targets, r, g, h, d_lse=z)
    ref = R.logprobs_gradient(logits, targets, g, h, z)
    bound, rel = _gradient_bound(ref, logits, dtype)
    p = torch.exp(torch.log_softmax(logits.double(), -1))
    terms = p * (g.abs() + z.abs() + h.abs() * 40).double().unsqueeze(-1)  # |log p + H| < 40 here
    assert float(((got.double() - ref).abs() - bound - rel * terms * (1 + STEP[dtype])
                  - 2.0 ** -23 * g.abs().double().unsqueeze(-1)).max()) <= 0
    # through autograd, one loss of all three
    leaf = logits.clone().requires_grad_(True)
    a = ops.token_logprobs(leaf, targets, top_k=1)
    (a.logprobs * g + a.entropy * h + a.lse * z).sum().backward()
    assert torch.equal(leaf.grad, got)
    assert not a.top_logprobs.requires_grad
    # written over the logits
    copy = logits.clone()
    assert ops.token_logprobs_backward(copy, targets, r, g, h, d_lse=z, inplace=True) is copy
    assert torch.equal(copy, got)


def test_gradient_against_differences(pe, cuda_device):
    from flash_modernbert_b200 import ops

    logits, targets = _inputs(4, 700, torch.float32, cuda_device, seed=5)
    g, h = torch.randn(4, device=cuda_device), torch.randn(4, device=cuda_device)
    leaf = logits.clone().requires_grad_(True)
    r = ops.token_logprobs(leaf, targets)
    (d,) = torch.autograd.grad((r.logprobs * g + r.entropy * h).sum(), leaf)
    v = torch.randn(logits.shape, device=cuda_device, dtype=torch.float64)
    step = 1e-5

    def value(x):
        lp, ent, *_ = R.logprobs(x, targets)
        return float((lp * g.double() + ent * h.double()).sum())

    difference = (value(logits.double() + step * v) - value(logits.double() - step * v)) / (2 * step)
    assert abs(difference - float((d.double() * v).sum())) < 1e-4 * (1 + abs(difference))


def test_ignored_and_bad_targets(pe, cuda_device):
    from flash_modernbert_b200 import _lib, ops

    logits, targets = _inputs(6, 4000, torch.bfloat16, cuda_device, seed=6)
    targets[1], targets[4] = -100, 3
    g = torch.ones(6, device=cuda_device)
    for ignore in (-100, 3):
        t = targets if ignore == -100 else targets.clamp(min=0)
        r = ops.token_logprobs(logits, t, top_k=2, ignore_index=ignore)
        ops.check_status(cuda_device)
        _check_forward(r, logits, t, 2, ignore)
        d = ops.token_logprobs_backward(logits, t, r, g, ignore_index=ignore)
        assert bool((d[t == ignore] == 0).all()) and bool((d[t != ignore] != 0).any(-1).all())
    for bad in (4000, -1, 2 ** 40):
        t = targets.clone()
        t[0] = bad
        r = ops.token_logprobs(logits, t)
        with pytest.raises(_lib.NativeLibraryError, match="304"):
            ops.check_status(cuda_device)
        assert float(r.logprobs[0]) == 0.0
        assert not ops.token_logprobs_backward(logits, t, r, g)[0].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab,width,start", [(1001, 1008, 0), (1000, 1003, 3), (4097, 4100, 1)])
def test_strided_logits(pe, cuda_device, dtype, vocab, width, start):
    """The slice of a padded vocabulary is read in place, whatever its alignment; what lies beyond it
    is neither read into a row nor written."""
    from flash_modernbert_b200 import ops

    wide = torch.full((9, width), math.nan, dtype=dtype, device=cuda_device)
    view = wide[:, start:start + vocab]
    logits, targets = _inputs(9, vocab, dtype, cuda_device, seed=7)
    view.copy_(logits)
    r, s = ops.token_logprobs(view, targets, top_k=6), ops.token_logprobs(logits, targets, top_k=6)
    _check_forward(r, logits, targets, 6)
    assert torch.equal(r.top_ids, s.top_ids)
    g = torch.ones(9, device=cuda_device)
    d = ops.token_logprobs_backward(logits, targets, s, g)
    assert torch.equal(ops.token_logprobs_backward(view, targets, s, g), d)
    ops.token_logprobs_backward(view, targets, s, g, inplace=True)
    assert torch.equal(view, d)
    outside = torch.ones(width, dtype=torch.bool)
    outside[start:start + vocab] = False
    assert torch.isnan(wide[:, outside.to(cuda_device)]).all()


def test_shapes_and_empty(pe, cuda_device):
    from flash_modernbert_b200 import ops

    logits, targets = _inputs(12, 300, torch.float32, cuda_device, seed=8)
    flat = ops.token_logprobs(logits, targets, top_k=3)
    r = ops.token_logprobs(logits.view(3, 4, 300), targets.view(3, 4), top_k=3)
    assert r.logprobs.shape == (3, 4) and r.top_ids.shape == (3, 4, 3)
    assert torch.equal(r.top_ids.view(12, 3), flat.top_ids) and torch.equal(r.logprobs.view(12), flat.logprobs)
    one = ops.token_logprobs(logits[0], targets[0])
    assert one.logprobs.shape == () and torch.equal(one.logprobs, flat.logprobs[0])
    none = ops.token_logprobs(logits[:0], targets[:0], top_k=3)
    assert none.logprobs.shape == (0,) and none.top_ids.shape == (0, 3)
    assert ops.token_logprobs_backward(logits[:0], targets[:0], none, none.lse).shape == (0, 300)


def test_far_logits(pe, cuda_device):
    """Logits far from zero keep their differences: statistics are relative to the maximum."""
    from flash_modernbert_b200 import ops

    logits, targets = _inputs(3, 5000, torch.float32, cuda_device, seed=9)
    logits = logits + torch.tensor([[8192.0], [-8192.0], [0.0]], device=cuda_device)
    _check_forward(ops.token_logprobs(logits, targets, top_k=5), logits, targets, 5)


def test_captured_and_replayed(pe, cuda_device):
    from flash_modernbert_b200 import ops

    logits, targets = _inputs(5, 9001, torch.bfloat16, cuda_device, seed=10)
    g = torch.ones(5, device=cuda_device)

    def step():
        r = ops.token_logprobs(logits, targets, top_k=5)
        return r, ops.token_logprobs_backward(logits, targets, r, g)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r, d = step()
    for seed in (11, 12):
        a, b = _inputs(5, 9001, torch.bfloat16, cuda_device, seed=seed)
        logits.copy_(a)
        targets.copy_(b)
        graph.replay()
        _check_forward(r, a, b, 5)
        e, f = step()
        assert torch.equal(f, d) and torch.equal(e.logprobs, r.logprobs)
