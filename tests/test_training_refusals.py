"""What the training operators refuse, on the host: no device work is reached."""
from __future__ import annotations

import ctypes

import pytest
import torch


def test_cpu_tensors_are_refused(pe):
    from flash_modernbert_b200 import ops

    qkv = torch.zeros(4, 192, dtype=torch.bfloat16)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    lse = torch.zeros(1, 4)
    with pytest.raises(pe.PackedEncodersError, match="CUDA"):
        ops.attention_varlen_qkv_lse(qkv, cu, 4, 1, None)
    with pytest.raises(pe.PackedEncodersError, match="CUDA"):
        ops.attention_varlen_qkv_train(qkv, cu, 4, 1, None)
    with pytest.raises(pe.PackedEncodersError, match="CUDA"):
        ops.attention_varlen_qkv_backward(qkv[:, :64], qkv, qkv[:, :64], lse, cu, 4, 1, None)
    rng = torch.zeros(2, dtype=torch.int64)
    for f in (lambda: ops.dropout(torch.zeros(4), 0.5, rng), lambda: ops.dropout_backward(torch.zeros(4), 0.5, rng)):
        with pytest.raises(pe.PackedEncodersError, match="CUDA"):
            f()
    with pytest.raises(pe.PackedEncodersError, match="CUDA"):
        ops.token_logprobs(torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(pe.PackedEncodersError, match="CUDA"):
        ops.token_logprobs(torch.zeros(2, 5, requires_grad=True), torch.zeros(2, dtype=torch.int64))


def test_library_argument_errors(pe):
    """Codes come back before anything is enqueued: null pointers, sizes, types, workspaces."""
    from flash_modernbert_b200 import _lib

    lib = _lib.load()
    p = 1 << 20  # an address that is never followed
    assert lib.pe_attn_varlen_lse(p, p, 1, 4, 1, -1, 4, p, None, p, 1 << 20, None, None) == _lib.PE_ERR_ARG
    assert lib.pe_attn_varlen_lse(p, p, 1, 4, 1, -1, 4, p + 2, p, p, 1 << 20, None, None) == _lib.PE_ERR_ARG
    assert lib.pe_attn_backward_workspace_bytes(-1, 1) == 0 and lib.pe_attn_backward_workspace_bytes(4, 0) == 0
    assert lib.pe_attn_backward_workspace_bytes(1000, 12) >= 1000 * 8 + 2 * 4 * 12 * 1000

    def backward(T=4, nh=1, n=1, pos=None, table=None, rows=0, ws=p, size=1 << 30, dqkv=p):
        return lib.pe_attn_varlen_backward(p, p, p, p, p, n, T, nh, -1, pos, table, rows, dqkv, ws, size, None, None)

    assert backward(dqkv=None) == _lib.PE_ERR_ARG and "null" in _lib.last_error()
    assert backward(n=0) == _lib.PE_ERR_ARG and backward(nh=0) == _lib.PE_ERR_ARG and backward(T=-1) == _lib.PE_ERR_ARG
    assert backward(T=1 << 31) == _lib.PE_ERR_ARG
    assert backward(T=(1 << 31) - 1024, nh=1024) == _lib.PE_ERR_ARG
    assert backward(pos=p) == _lib.PE_ERR_ARG and backward(table=p, rows=5) == _lib.PE_ERR_ARG
    assert backward(pos=p, table=p, rows=0) == _lib.PE_ERR_ARG
    assert backward(ws=p + 8) == _lib.PE_ERR_ARG
    assert backward(size=16) == _lib.PE_ERR_WORKSPACE and "workspace" in _lib.last_error()
    assert backward(T=0, size=1 << 20) == _lib.PE_OK

    def dropout(x=p, dtype=0, n=8, prob=0.5, rng=p, y=p):
        return lib.pe_dropout(x, None, dtype, n, prob, rng, None, y, None)

    assert dropout(x=None) == _lib.PE_ERR_ARG and dropout(y=None) == _lib.PE_ERR_ARG
    assert dropout(rng=None) == _lib.PE_ERR_ARG and dropout(dtype=3) == _lib.PE_ERR_ARG
    for prob in (-0.1, 1.1, float("nan")):
        assert dropout(prob=prob) == _lib.PE_ERR_ARG
    assert dropout(n=-1) == _lib.PE_ERR_ARG and dropout(x=p + 1) == _lib.PE_ERR_ARG
    assert dropout(n=0, x=None, y=None) == _lib.PE_OK

    def logprobs(logits=p, dtype=0, rows=2, vocab=10, ld=10, k=0, ids=None):
        return lib.pe_token_logprobs(logits, dtype, rows, vocab, ld, p, -100, k, p, p, p, p, ids, ids, None, None)

    assert logprobs(logits=None) == _lib.PE_ERR_ARG and logprobs(dtype=7) == _lib.PE_ERR_ARG
    assert logprobs(ld=9) == _lib.PE_ERR_ARG and logprobs(vocab=0) == _lib.PE_ERR_ARG
    assert logprobs(k=11, ids=p) == _lib.PE_ERR_ARG and logprobs(k=33, vocab=100, ld=100, ids=p) == _lib.PE_ERR_ARG
    assert logprobs(k=3) == _lib.PE_ERR_ARG and logprobs(logits=p + 1) == _lib.PE_ERR_ARG
    assert logprobs(rows=0) == _lib.PE_OK
    args = (p, 0, 2, 10, 10, p, -100, p, p, p, None, None, None)
    assert lib.pe_token_logprobs_backward(*args, None, 10, None) == _lib.PE_ERR_ARG
    assert lib.pe_token_logprobs_backward(*args, p, 9, None) == _lib.PE_ERR_ARG


@pytest.mark.gpu
def test_tensor_argument_errors(pe, cuda_device):
    from flash_modernbert_b200 import ops

    qkv = torch.zeros(4, 192, dtype=torch.bfloat16, device=cuda_device)
    cu = torch.tensor([0, 4], dtype=torch.int32, device=cuda_device)
    out, lse = ops.attention_varlen_qkv_lse(qkv, cu, 4, 1, None)
    for bad in (dict(n_heads=2), dict(half_window=-1), dict(max_seqlen=0), dict(cu_seqlens=cu.long()),
                dict(cu_seqlens=cu[:1])):
        kw = dict(cu_seqlens=cu, max_seqlen=4, n_heads=1, half_window=None) | bad
        with pytest.raises(ValueError):
            ops.attention_varlen_qkv_lse(qkv, **kw)
        with pytest.raises(ValueError):
            ops.attention_varlen_qkv_backward(out, qkv, out, lse, **kw)
    with pytest.raises(pe.PackedEncodersError):
        ops.attention_varlen_qkv_lse(qkv.float(), cu, 4, 1, None)
    with pytest.raises(ValueError, match="dout"):
        ops.attention_varlen_qkv_backward(out[:3], qkv, out, lse, cu, 4, 1, None)
    with pytest.raises(ValueError, match="lse"):
        ops.attention_varlen_qkv_backward(out, qkv, out, lse.double(), cu, 4, 1, None)
    table = ops.rope_table(1e4, 8, cuda_device)
    with pytest.raises(ValueError, match="together"):
        ops.attention_varlen_qkv_train(qkv, cu, 4, 1, None, table=table)
    with pytest.raises(ValueError, match="position_ids"):
        ops.attention_varlen_qkv_train(qkv, cu, 4, 1, None, table=table, position_ids=torch.arange(3, device=cuda_device))
    x = torch.zeros(4, device=cuda_device)
    rng = torch.zeros(2, dtype=torch.int64, device=cuda_device)
    for p in (-0.1, 1.5, float("nan")):
        with pytest.raises(ValueError, match="within"):
            ops.dropout(x, p, rng)
    with pytest.raises(ValueError, match="rng"):
        ops.dropout(x, 0.5, rng[:1])
    with pytest.raises(ValueError, match="rng"):
        ops.dropout(x, 0.5, rng.int())
    with pytest.raises(ValueError, match="residual"):
        ops.dropout(x, 0.5, rng, residual=x[:2])
    with pytest.raises(pe.PackedEncodersError):
        ops.dropout(x.double(), 0.5, rng)
    logits, targets = torch.zeros(2, 5, device=cuda_device), torch.zeros(2, dtype=torch.int64, device=cuda_device)
    for k in (-1, 6):
        with pytest.raises(ValueError, match="top_k"):
            ops.token_logprobs(logits, targets, top_k=k)
    with pytest.raises(ValueError, match="targets"):
        ops.token_logprobs(logits, targets[:1])
    with pytest.raises(ValueError, match="targets"):
        ops.token_logprobs(logits, targets.int())
    with pytest.raises(ValueError, match="vocab"):
        ops.token_logprobs(logits[:, :0], targets)
    r = ops.token_logprobs(logits, targets)
    with pytest.raises(ValueError, match="d_logprobs"):
        ops.token_logprobs_backward(logits, targets, r, r.lse.double())
    strided = torch.zeros(5, 2, device=cuda_device).t()
    with pytest.raises(pe.PackedEncodersError, match="written over"):
        ops.token_logprobs_backward(strided, targets, r, r.lse, inplace=True)
