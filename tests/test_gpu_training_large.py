"""The training operators past 2^31 elements: the far end of a large call against the same rows alone."""
from __future__ import annotations

import pytest
import torch

import training_reference as R

pytestmark = pytest.mark.gpu


def test_dropout_beyond_32_bits(pe, cuda_device):
    from flash_modernbert_b200 import ops

    n, tail, position = 2 ** 31 + 1003, 1011, 77
    x = torch.ones(n, dtype=torch.bfloat16, device=cuda_device)
    rng = torch.tensor([5, position], dtype=torch.int64, device=cuda_device)
    y = ops.dropout(x, 0.3, rng)
    begin = n - tail  # a multiple of eight: where a block of the generator starts
    assert begin % 8 == 0
    keep, scale = R.dropout_keep(tail, 0.3, 5, position + begin // 8)
    assert torch.equal(y[begin:].cpu(), torch.where(keep, torch.full((tail,), scale), torch.zeros(tail)).bfloat16())


def test_logprobs_beyond_32_bits(pe, cuda_device):
    from flash_modernbert_b200 import ops

    vocab, rows = 50368, 2 ** 31 // 50368 + 9
    logits = torch.zeros(rows, vocab, dtype=torch.bfloat16, device=cuda_device)
    logits[-8:] = torch.randn(8, vocab, device=cuda_device)
    targets = torch.randint(0, vocab, (rows,), device=cuda_device)
    r = ops.token_logprobs(logits, targets, top_k=3)
    chosen, entropy, _, ids, _ = R.logprobs(logits[-8:], targets[-8:], top_k=3)
    # fp32 sums over the vocabulary: 2^-18 relative in the sum, 2^-22 of |x| and log s in the difference
    assert float((r.logprobs[-8:].double() - chosen).abs().max()) <= 2.0 ** -17
    assert float((r.entropy[-8:].double() - entropy).abs().max()) <= 2.0 ** -15
    assert torch.equal(r.top_ids[-8:], ids)
    ones = torch.ones(rows, device=cuda_device)
    grad = ops.token_logprobs_backward(logits, targets, r, ones, inplace=True)
    ops.check_status(cuda_device)
    again = torch.zeros(8, vocab, dtype=torch.bfloat16, device=cuda_device)
    assert int(torch.count_nonzero(grad[-9])) == vocab  # the uniform row: -1 / vocab everywhere but at the target
    assert bool(torch.isfinite(grad[-8:]).all()) and not torch.equal(grad[-8:], again)
    at = grad[-8:].gather(1, targets[-8:].unsqueeze(1)).squeeze(1).double()
    assert float((at - (1 - torch.exp(chosen))).abs().max()) <= R.EPS


@pytest.mark.parametrize("hw", [8, None])
def test_attention_beyond_32_bits(pe, cuda_device, hw):
    from flash_modernbert_b200 import ops

    n_heads, length, last = 12, 100, [100, 37, 90]
    lengths = [length] * (2 ** 31 // (3 * n_heads * 64) // length + 1) + last
    total = sum(lengths)
    assert (total - sum(last)) * 3 * n_heads * 64 >= 2 ** 31
    gen = torch.Generator(device=cuda_device).manual_seed(0)
    qkv = torch.empty(total, 3 * n_heads * 64, dtype=torch.bfloat16, device=cuda_device).normal_(generator=gen)
    dout = torch.empty(total, n_heads * 64, dtype=torch.bfloat16, device=cuda_device).normal_(generator=gen) * 0.1
    cu = torch.zeros(len(lengths) + 1, dtype=torch.int32)
    cu[1:] = torch.tensor(lengths).cumsum(0)
    cu = cu.to(cuda_device)
    out, lse = ops.attention_varlen_qkv_lse(qkv, cu, length, n_heads, hw)
    grad = ops.attention_varlen_qkv_backward(dout, qkv, out, lse, cu, length, n_heads, hw)
    ops.check_status(cuda_device)
    for sl in (slice(total - sum(last), total), slice(0, length)):
        here = last if sl.start else [length]
        ref, bound = R.attention(qkv[sl], dout[sl], here, n_heads, hw)
        for a, b, e in zip((out[sl], lse[:, sl], grad[sl]), ref, bound):
            assert float(((a.double() - b).abs() - e).max()) <= 0


def test_windows_and_lengths_of_any_size_are_taken(pe, cuda_device):
    from flash_modernbert_b200 import ops

    qkv = torch.randn(90, 3 * 64, device=cuda_device).bfloat16()
    dout = torch.randn(90, 64, device=cuda_device).bfloat16()
    cu = torch.tensor([0, 90], dtype=torch.int32, device=cuda_device)
    results = []
    for hw, longest in ((2 ** 20, 90), (2 ** 40, 2 ** 40)):
        out, lse = ops.attention_varlen_qkv_lse(qkv, cu, longest, 1, hw)
        results.append((out, lse, ops.attention_varlen_qkv_backward(dout, qkv, out, lse, cu, longest, 1, hw)))
    assert all(torch.equal(a, b) for a, b in zip(*results))
