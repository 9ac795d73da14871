"""Token log-probabilities of many rows at once, which are worked on by other thread counts than few rows."""
from __future__ import annotations

import math

import pytest
import torch

from test_gpu_token_logprobs import TYPES, _check_forward, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,top_k", [(1000, 1, 1), (1000, 8, 5), (1000, 40, 32), (900, 200, 5), (887, 1000, 20),
                                              (889, 1000, 20), (960, 3001, 0), (960, 3001, 32), (900, 33000, 5),
                                              (900, 65536, 32), (900, 65537, 3)])
def test_forward(pe, cuda_device, dtype, rows, vocab, top_k):
    from flash_modernbert_b200 import ops

    logits, targets = _inputs(rows, vocab, dtype, cuda_device, seed=rows + vocab)
    _check_forward(ops.token_logprobs(logits, targets, top_k=top_k), logits, targets, top_k)
    ops.check_status(cuda_device)


@pytest.mark.parametrize("vocab", [33, 700, 20000])
@pytest.mark.parametrize("order", ["equal", "ascending", "descending", "few"])
def test_ties_and_orders(pe, cuda_device, vocab, order):
    from flash_modernbert_b200 import ops

    rows = 1000
    line = {"equal": torch.zeros(vocab), "ascending": torch.linspace(-4, 4, vocab), "descending": torch.linspace(4, -4, vocab),
            "few": torch.randint(0, 3, (vocab,), generator=torch.Generator().manual_seed(1)).float()}[order]
    logits = line.to(cuda_device, torch.float16).expand(rows, vocab).contiguous()
    targets = torch.arange(rows, device=cuda_device) % vocab
    _check_forward(ops.token_logprobs(logits, targets, top_k=9), logits, targets, 9)


def test_masked_rows(pe, cuda_device):
    """Rows of which few logits are left, at either end of the row or anywhere, and strided rows."""
    from flash_modernbert_b200 import ops

    rows, vocab = 1000, 5003
    wide, targets = _inputs(rows, vocab + 5, torch.bfloat16, cuda_device, seed=4)
    logits = wide[:, 3:vocab + 3]
    gen = torch.Generator(device=cuda_device).manual_seed(2)
    keep = torch.rand(rows, vocab, generator=gen, device=cuda_device) < 0.002
    keep[:, :4] |= (torch.arange(rows, device=cuda_device) % 3 == 0)[:, None]
    keep[:, -4:] |= (torch.arange(rows, device=cuda_device) % 3 == 1)[:, None]
    keep[:, vocab // 2: vocab // 2 + 4] |= (torch.arange(rows, device=cuda_device) % 3 == 2)[:, None]
    logits.masked_fill_(~keep, -math.inf)
    first = keep.to(torch.int64).argmax(-1)
    _check_forward(ops.token_logprobs(logits, first, top_k=4), logits, first, 4)
