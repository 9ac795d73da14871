"""`rope_qk`, the rotation into a new tensor, against the one in place: equal bits."""
from __future__ import annotations

import pytest
import torch


@pytest.mark.gpu
@pytest.mark.parametrize("total,n_heads", [(0, 2), (1, 1), (7, 3), (300, 12), (1001, 28)])
def test_same_bits_as_in_place(pe, cuda_device, total, n_heads):
    from flash_modernbert_b200 import ops

    gen = torch.Generator(device=cuda_device).manual_seed(total)
    wide = torch.randn(total, 3 * n_heads * 64 + 8, generator=gen, device=cuda_device).bfloat16()
    table = ops.rope_table(10000.0, 50, cuda_device)
    pos = torch.randint(0, 50, (total,), generator=gen, device=cuda_device)
    for qkv in (wide[:, :-8].contiguous(), wide[:, 4:-4]):  # the second neither contiguous nor aligned
        before = qkv.clone()
        got = ops.rope_qk(qkv, pos, table, n_heads)
        assert torch.equal(qkv, before) and got.is_contiguous()
        want = before.contiguous()
        assert torch.equal(got, ops.rope_qk_inplace(want, pos, table, n_heads) if total else want)
    ops.check_status(cuda_device)


@pytest.mark.gpu
def test_refusals_and_bad_positions(pe, cuda_device):
    from flash_modernbert_b200 import _lib, ops
    from flash_modernbert_b200.errors import PackedEncodersError

    qkv = torch.randn(4, 192, device=cuda_device).bfloat16()
    table = ops.rope_table(10000.0, 8, cuda_device)
    pos = torch.arange(4, device=cuda_device)
    for bad in (lambda: ops.rope_qk(qkv.float(), pos, table, 1), lambda: ops.rope_qk(qkv, pos, table, 2),
                lambda: ops.rope_qk(qkv, pos.int(), table, 1), lambda: ops.rope_qk(qkv, pos[:3], table, 1),
                lambda: ops.rope_qk(qkv, pos, None, 1), lambda: ops.rope_qk(qkv, None, None, 1),
                lambda: ops.rope_qk(qkv, pos, table[:, :32], 1)):
        with pytest.raises((ValueError, PackedEncodersError)):
            bad()
    ops.check_status(cuda_device)
    got = ops.rope_qk(qkv, torch.tensor([0, 1, 8, -1], device=cuda_device), table, 1)
    with pytest.raises(_lib.NativeLibraryError, match="302"):
        ops.check_status(cuda_device)
    want = ops.rope_qk(qkv, torch.tensor([0, 1, 0, 0], device=cuda_device), table, 1)
    assert torch.equal(got, want)


def test_library_argument_errors(pe):
    from flash_modernbert_b200 import _lib

    lib = _lib.load()
    p, q = 4096, 8192
    assert lib.pe_rope_qk(None, None, None, 1, 0, 1, None, None, None) == 0
    for args in ((p, p, p, 1, 5, 1, p), (p, p, p, 0, 5, 1, q), (p, p, p, 1, 5, 0, q), (p, p, p, 1, -1, 1, q),
                 (p + 2, p, p, 1, 5, 1, q), (p, None, p, 1, 5, 1, q), (p, p, p, 1, 1 << 40, 1 << 20, q)):
        assert lib.pe_rope_qk(*args, None, None) != 0
