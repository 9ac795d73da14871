"""Single-op entry points on torch tensors, one C-ABI call each.

Names and argument meaning follow the inference branches of packed_encoders/ops.py
(`fused_layer_norm` 191-208, `fused_add_layer_norm` 303-314, `_linear` 290-300,
`fused_geglu` 275-280, `geglu_mlp` 317-319, `flash_attention_qkv_bshd` 485-532), so
the parity tests read like the reference's. `packed_forward` does not go through
these wrappers (it is one C call); they exist for callers that compose their own
pipeline and for per-kernel tests. All tensors must be CUDA bf16 and contiguous.
"""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch import Tensor

from . import _lib
from .errors import PackedEncodersError


def _bf16_cuda(t: Tensor, name: str) -> Tensor:
    if not t.is_cuda or t.dtype != torch.bfloat16:
        raise PackedEncodersError(f"{name} must be a CUDA bf16 tensor, got {t.dtype} on {t.device}")
    return t if t.is_contiguous() else t.contiguous()


def _index_cuda(t: Tensor, name: str, dtype: torch.dtype, like: Tensor) -> Tensor:
    """An index operand (`cu_seqlens`, `position_ids`, token ids): the library reads it as raw
    `dtype` data on the device of `like`, so anything else is refused here instead of being
    misread there (an int64 `cu_seqlens` would give wrong boundaries, a CPU tensor a host
    address inside a kernel)."""
    if not isinstance(t, Tensor) or not t.is_cuda:
        raise PackedEncodersError(f"{name} must be a CUDA tensor (this package has no CPU path)")
    if t.dtype != dtype:
        raise ValueError(f"{name} must have dtype {dtype}, got {t.dtype}")
    if t.device != like.device:
        raise PackedEncodersError(f"{name} is on {t.device}, the data it indexes on {like.device}")
    return t if t.is_contiguous() else t.contiguous()


class _Call:
    """Device guard + stream + status word for one library call."""

    __slots__ = ("lib", "index", "guard", "stream")

    def __init__(self, ref: Tensor):
        self.lib = _lib.load()
        self.index = ref.device.index
        # switching to the device that is current already costs more than the launch of a small kernel
        self.guard = None if torch.cuda.current_device() == self.index else torch.cuda.device(self.index)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()
        self.stream = _lib.device_stream_ptr(self.index)
        return self

    def __exit__(self, *exc):
        return None if self.guard is None else self.guard.__exit__(*exc)


_status_words: dict[int, Tensor] = {}


def status_word(device: torch.device) -> Tensor:
    idx = device.index if device.index is not None else torch.cuda.current_device()
    if idx not in _status_words:
        _status_words[idx] = torch.zeros(1, dtype=torch.int32, device=torch.device("cuda", idx))
    return _status_words[idx]


def check_status(device: torch.device) -> None:
    """Synchronise and raise if any kernel launched through this module reported a fault."""
    word = status_word(device)
    code = int(word.item())
    if code != 0:
        word.zero_()
        raise _lib.NativeLibraryError(f"a CUDA kernel reported status {code}")


def fused_layer_norm(x: Tensor, weight: Tensor, eps: float) -> Tensor:
    x = _bf16_cuda(x, "x")
    flat = x.reshape(-1, x.shape[-1])
    y = torch.empty_like(flat)
    with _Call(x) as c:
        _lib.check(c.lib.pe_add_ln(flat.data_ptr(), None, _bf16_cuda(weight, "weight").data_ptr(),
                                   float(eps), flat.shape[0], flat.shape[1], None, y.data_ptr(),
                                   c.stream), "pe_add_ln")
    return y.view(x.shape)


def fused_add_layer_norm(x: Tensor, residual: Tensor, weight: Tensor, eps: float) -> tuple[Tensor, Tensor]:
    """`x_new = x + residual` (rounded to bf16), `y = LN(x_new)`; returns `(x_new, y)`."""
    x = _bf16_cuda(x, "x")
    residual = _bf16_cuda(residual, "residual")
    flat = x.reshape(-1, x.shape[-1])
    x_new = torch.empty_like(flat)
    y = torch.empty_like(flat)
    with _Call(x) as c:
        _lib.check(c.lib.pe_add_ln(flat.data_ptr(), residual.reshape(flat.shape).data_ptr(),
                                   _bf16_cuda(weight, "weight").data_ptr(), float(eps),
                                   flat.shape[0], flat.shape[1], x_new.data_ptr(), y.data_ptr(),
                                   c.stream), "pe_add_ln")
    return x_new.view(x.shape), y.view(x.shape)


def embed_layer_norm(ids: Tensor, table: Tensor, weight: Tensor, eps: float) -> Tensor:
    """`LN(table[ids])`: the embedding prologue of packed_encoders/forward.py:472-476."""
    table = _bf16_cuda(table, "table")
    ids = _index_cuda(ids, "ids", torch.int64, table)
    out = torch.empty(ids.numel(), table.shape[1], dtype=torch.bfloat16, device=table.device)
    with _Call(table) as c:
        _lib.check(c.lib.pe_embed_ln(ids.data_ptr(), table.data_ptr(),
                                     _bf16_cuda(weight, "weight").data_ptr(), float(eps),
                                     ids.numel(), table.shape[1], table.shape[0], out.data_ptr(),
                                     status_word(table.device).data_ptr(), c.stream), "pe_embed_ln")
    return out.view(*ids.shape, table.shape[1])


def _linear(x: Tensor, weight: Tensor) -> Tensor:
    """`x @ weight.T`, weight `[out, in]` as `nn.Linear` stores it; no bias."""
    x = _bf16_cuda(x, "x")
    weight = _bf16_cuda(weight, "weight")
    flat = x.reshape(-1, x.shape[-1])
    out = torch.empty(flat.shape[0], weight.shape[0], dtype=torch.bfloat16, device=x.device)
    with _Call(x) as c:
        _lib.check(c.lib.pe_gemm_bf16_tn(flat.data_ptr(), weight.data_ptr(), out.data_ptr(),
                                         flat.shape[0], weight.shape[0], weight.shape[1],
                                         status_word(x.device).data_ptr(), c.stream),
                   "pe_gemm_bf16_tn")
    return out.view(*x.shape[:-1], weight.shape[0])


def fused_geglu(proj: Tensor) -> Tensor:
    proj = _bf16_cuda(proj, "proj")
    flat = proj.reshape(-1, proj.shape[-1])
    inter = flat.shape[1] // 2
    out = torch.empty(flat.shape[0], inter, dtype=torch.bfloat16, device=proj.device)
    with _Call(proj) as c:
        _lib.check(c.lib.pe_geglu(flat.data_ptr(), flat.shape[0], inter, out.data_ptr(), c.stream),
                   "pe_geglu")
    return out.view(*proj.shape[:-1], inter)


def linear_geglu(x: Tensor, wi: Tensor) -> Tensor:
    """`fused_geglu(_linear(x, wi))` as one kernel (the projection never reaches memory)."""
    x = _bf16_cuda(x, "x")
    wi = _bf16_cuda(wi, "wi")
    flat = x.reshape(-1, x.shape[-1])
    inter = wi.shape[0] // 2
    out = torch.empty(flat.shape[0], inter, dtype=torch.bfloat16, device=x.device)
    with _Call(x) as c:
        _lib.check(c.lib.pe_gemm_geglu_bf16(flat.data_ptr(), wi.data_ptr(), out.data_ptr(),
                                            flat.shape[0], inter, wi.shape[1],
                                            status_word(x.device).data_ptr(), c.stream),
                   "pe_gemm_geglu_bf16")
    return out.view(*x.shape[:-1], inter)


def geglu_mlp(x: Tensor, wi: Tensor, wo: Tensor) -> Tensor:
    return _linear(linear_geglu(x, wi), wo)


def rope_table(theta: float, max_positions: int, device) -> Tensor:
    """bf16 `[max_positions, 64]`: cos of the 32 frequencies, then sin."""
    table = torch.empty(max_positions, 64, dtype=torch.bfloat16, device=device)
    with _Call(table) as c:
        _lib.check(c.lib.pe_rope_table(float(theta), max_positions, table.data_ptr(), c.stream),
                   "pe_rope_table")
    return table


def rope_qk_inplace(qkv: Tensor, position_ids: Tensor, table: Tensor, n_heads: int) -> Tensor:
    """Rotate the q and k thirds of the fused `qkv [T, 3*n_heads*64]` in place."""
    if not qkv.is_contiguous():
        raise PackedEncodersError("qkv must be contiguous for the in-place rotation")
    qkv = _bf16_cuda(qkv, "qkv")
    pos = _index_cuda(position_ids, "position_ids", torch.int64, qkv)
    with _Call(qkv) as c:
        _lib.check(c.lib.pe_rope_qk_inplace(qkv.data_ptr(), pos.data_ptr(),
                                            _bf16_cuda(table, "table").data_ptr(), table.shape[0],
                                            qkv.shape[0], n_heads,
                                            status_word(qkv.device).data_ptr(), c.stream),
                   "pe_rope_qk_inplace")
    return qkv


def linear_qkv_rope(x: Tensor, wqkv: Tensor, position_ids: Tensor, table: Tensor, n_heads: int) -> Tensor:
    """`rope_qk_inplace(_linear(x, wqkv), ...)` as one kernel: the rotation runs in the GEMM epilogue."""
    x = _bf16_cuda(x, "x")
    wqkv = _bf16_cuda(wqkv, "wqkv")
    flat = x.reshape(-1, x.shape[-1])
    pos = _index_cuda(position_ids, "position_ids", torch.int64, x)
    out = torch.empty(flat.shape[0], 3 * n_heads * 64, dtype=torch.bfloat16, device=x.device)
    with _Call(x) as c:
        _lib.check(c.lib.pe_gemm_qkv_rope_bf16(flat.data_ptr(), wqkv.data_ptr(), out.data_ptr(),
                                               flat.shape[0], n_heads, wqkv.shape[1],
                                               pos.data_ptr(),
                                               _bf16_cuda(table, "table").data_ptr(), table.shape[0],
                                               status_word(x.device).data_ptr(), c.stream),
                   "pe_gemm_qkv_rope_bf16")
    return out


def linear_residual(x: Tensor, weight: Tensor, residual: Tensor, *, inplace: bool = False) -> Tensor:
    """`residual + _linear(x, weight)` with the projection rounded to bf16 before the add, as one
    kernel. `inplace=True` writes the sum over `residual`."""
    x = _bf16_cuda(x, "x")
    weight = _bf16_cuda(weight, "weight")
    residual = _bf16_cuda(residual, "residual")
    flat = x.reshape(-1, x.shape[-1])
    res = residual.reshape(flat.shape[0], weight.shape[0])
    out = res if inplace else torch.empty_like(res)
    with _Call(x) as c:
        _lib.check(c.lib.pe_gemm_residual_bf16(flat.data_ptr(), weight.data_ptr(), res.data_ptr(),
                                               out.data_ptr(), flat.shape[0], weight.shape[0],
                                               weight.shape[1], status_word(x.device).data_ptr(),
                                               c.stream), "pe_gemm_residual_bf16")
    return out.view(residual.shape)


def attention_varlen_qkv(qkv: Tensor, cu_seqlens: Tensor, max_seqlen: int, n_heads: int,
                         half_window: int | None) -> Tensor:
    """Varlen attention on the fused, already-rotated `qkv [T, 3*n_heads*64]`;
    `half_window=None` is full attention. Returns `[T, n_heads*64]`."""
    qkv = _bf16_cuda(qkv, "qkv")
    cu = _index_cuda(cu_seqlens, "cu_seqlens", torch.int32, qkv)
    total = qkv.shape[0]
    n_seqs = cu.numel() - 1
    out = torch.empty(total, n_heads * 64, dtype=torch.bfloat16, device=qkv.device)
    with _Call(qkv) as c:
        ws_bytes = int(c.lib.pe_attn_workspace_bytes(total, n_seqs))
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=qkv.device)
        _lib.check(c.lib.pe_attn_varlen(qkv.data_ptr(), cu.data_ptr(), n_seqs,
                                        total, n_heads, -1 if half_window is None else half_window,
                                        int(max_seqlen), out.data_ptr(), ws.data_ptr(), ws_bytes,
                                        status_word(qkv.device).data_ptr(), c.stream),
                   "pe_attn_varlen")
    return out


def attention_varlen_qkv_static(qkv: Tensor, cu_seqlens: Tensor, max_seqlen: int, n_heads: int,
                                half_window: int | None) -> Tensor:
    """`attention_varlen_qkv` through the entry point that brings its own scratch: for callers
    that cannot allocate device memory (a host process whose allocator owns the whole GPU, a
    request path with a frozen memory budget). At most 4096 sequences and 1,048,576 tokens;
    calls share one built-in table, so keep them on one stream. Only the output tensor is
    created here, by the caller's own allocator."""
    qkv = _bf16_cuda(qkv, "qkv")
    cu = _index_cuda(cu_seqlens, "cu_seqlens", torch.int32, qkv)
    total = qkv.shape[0]
    out = torch.empty(total, n_heads * 64, dtype=torch.bfloat16, device=qkv.device)
    with _Call(qkv) as c:
        _lib.check(c.lib.pe_attn_varlen_static(qkv.data_ptr(), cu.data_ptr(),
                                               cu.numel() - 1, total, n_heads,
                                               -1 if half_window is None else half_window,
                                               int(max_seqlen), out.data_ptr(),
                                               status_word(qkv.device).data_ptr(), c.stream),
                   "pe_attn_varlen_static")
    return out


def pool_packed(hidden: Tensor, cu_seqlens: Tensor, mode: str = "mean", normalize: bool = True) -> Tensor:
    """Sentence embeddings from the packed last hidden state, as the reference's callers compute
    them right after `packed_forward` (benchmarks/showcases/inference.py:193-206): per sequence
    the fp32 mean of its token rows (`mode="mean"`) or its first token (`mode="cls"`),
    optionally L2-normalised like `F.normalize`, rounded to bf16 last. `[T, H]` -> `[N, H]`."""
    if mode not in ("mean", "cls"):
        raise ValueError(f"pool_packed: mode must be 'mean' or 'cls', got {mode!r}")
    hidden = _bf16_cuda(hidden, "hidden")
    total, width = hidden.shape
    cu = _index_cuda(cu_seqlens, "cu_seqlens", torch.int32, hidden)
    n_seqs = cu.numel() - 1
    out = torch.empty(n_seqs, width, dtype=torch.bfloat16, device=hidden.device)
    with _Call(hidden) as c:
        ws_bytes = int(c.lib.pe_pool_workspace_bytes(total, n_seqs, width)) if mode == "mean" else 0
        ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=hidden.device)
        _lib.check(c.lib.pe_pool_packed(hidden.data_ptr(), cu.data_ptr(), n_seqs, total, width,
                                        1 if mode == "mean" else 0, 1 if normalize else 0,
                                        out.data_ptr(), ws.data_ptr(), ws_bytes, c.stream),
                   "pe_pool_packed")
    return out


def project_normalize(hidden: Tensor, weight: Tensor) -> Tensor:
    """Token-level projection head: `F.normalize(F.linear(hidden, weight), p=2, dim=-1)` in one
    kernel, as the reference's ColBERT indexing path computes it after `packed_forward`
    (benchmarks/helpers/packed_index.py:182-186). `weight` is `[out_features <= 256, H]`."""
    hidden = _bf16_cuda(hidden, "hidden")
    weight = _bf16_cuda(weight, "weight")
    flat = hidden.reshape(-1, hidden.shape[-1])
    if weight.shape[0] > 256:
        raise ValueError("project_normalize: at most 256 output features (one tile holds whole rows)")
    out = torch.empty(flat.shape[0], weight.shape[0], dtype=torch.bfloat16, device=hidden.device)
    with _Call(hidden) as c:
        _lib.check(c.lib.pe_gemm_l2norm_bf16(flat.data_ptr(), weight.data_ptr(), out.data_ptr(),
                                             flat.shape[0], weight.shape[0], weight.shape[1],
                                             status_word(hidden.device).data_ptr(), c.stream),
                   "pe_gemm_l2norm_bf16")
    return out.view(*hidden.shape[:-1], weight.shape[0])


# ---------------------------------------------------------------------------
# Training operators: attention with its gradient, dropout, token log-probabilities
# ---------------------------------------------------------------------------


def _attention_args(qkv: Tensor, cu_seqlens: Tensor, n_heads: int, half_window: int | None) -> tuple[Tensor, Tensor]:
    qkv = _bf16_cuda(qkv, "qkv")
    if n_heads <= 0 or qkv.dim() != 2 or qkv.shape[1] != 3 * n_heads * 64:
        raise ValueError(f"qkv must be [T, 3 * {n_heads} * 64], got {tuple(qkv.shape)}")
    if half_window is not None and half_window < 0:
        raise ValueError(f"half_window must be None (full attention) or at least 0, got {half_window}")
    cu = _index_cuda(cu_seqlens, "cu_seqlens", torch.int32, qkv)
    if cu.dim() != 1 or cu.shape[0] < 2:
        raise ValueError("cu_seqlens must be [N+1] with N >= 1")
    return _aligned(qkv), cu


def _window(half_window: int | None, total: int) -> int:
    """As the library takes it: -1 for none, and not much wider than any sequence can need (full
    attention's kernel walks the whole band, also where it leaves the sequence)."""
    return -1 if half_window is None else min(int(half_window), max(total, 4096))


def _aligned(t: Tensor) -> Tensor:
    """The kernels move 16 bytes at a time: a view that starts elsewhere is copied."""
    return t if t.data_ptr() % 16 == 0 else t.clone()


def attention_varlen_qkv_lse(qkv: Tensor, cu_seqlens: Tensor, max_seqlen: int, n_heads: int,
                             half_window: int | None) -> tuple[Tensor, Tensor]:
    """`attention_varlen_qkv` that also returns `lse` fp32 `[n_heads, T]`, the natural logarithm of
    every query's sum of exponentials, which `attention_varlen_qkv_backward` recomputes the
    probabilities from. Rows outside every sequence get 0 and `-inf`."""
    qkv, cu = _attention_args(qkv, cu_seqlens, n_heads, half_window)
    if int(max_seqlen) <= 0:
        raise ValueError("max_seqlen must be positive")
    total = qkv.shape[0]
    n_seqs = cu.numel() - 1
    out = torch.empty(total, n_heads * 64, dtype=torch.bfloat16, device=qkv.device)
    lse = torch.empty(n_heads, total, dtype=torch.float32, device=qkv.device)
    if total == 0:
        return out, lse
    # grids are sized by it; the floor is far above where it chooses a kernel
    longest = min(int(max_seqlen), max(total, 65536))
    with _Call(qkv) as c:
        ws_bytes = int(c.lib.pe_attn_workspace_bytes(total, n_seqs))
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=qkv.device)
        _lib.check(c.lib.pe_attn_varlen_lse(qkv.data_ptr(), cu.data_ptr(), n_seqs, total, n_heads,
                                            _window(half_window, total), longest,
                                            out.data_ptr(), lse.data_ptr(), ws.data_ptr(), ws_bytes,
                                            status_word(qkv.device).data_ptr(), c.stream),
                   "pe_attn_varlen_lse")
    return out, lse


def _rotation_args(position_ids: Tensor | None, table: Tensor | None, qkv: Tensor) -> tuple[Tensor | None, Tensor | None]:
    if (position_ids is None) != (table is None):
        raise ValueError("position_ids and table come together")
    if table is None:
        return None, None
    pos = _index_cuda(position_ids, "position_ids", torch.int64, qkv)
    table = _bf16_cuda(table, "table")
    if table.device != qkv.device:
        raise PackedEncodersError(f"table is on {table.device}, qkv on {qkv.device}")
    if pos.shape != qkv.shape[:1] or table.dim() != 2 or table.shape[1] != 64 or table.shape[0] == 0:
        raise ValueError("position_ids must be [T] and table [max_positions, 64]")
    return pos, _aligned(table)


def attention_varlen_qkv_backward(dout: Tensor, qkv: Tensor, out: Tensor, lse: Tensor, cu_seqlens: Tensor,
                                  max_seqlen: int, n_heads: int, half_window: int | None, *,
                                  position_ids: Tensor | None = None, table: Tensor | None = None) -> Tensor:
    """Gradient of `attention_varlen_qkv` with respect to the (already rotated) `qkv`, from the
    gradient `dout` of its output and what `attention_varlen_qkv_lse` returned. With
    `position_ids` and `table`, the rotation that q and k went through, the gradient is that of the
    qkv before the rotation. Same bits on every call; rows outside every sequence get zeros."""
    qkv, cu = _attention_args(qkv, cu_seqlens, n_heads, half_window)
    total = qkv.shape[0]
    pos, table = _rotation_args(position_ids, table, qkv)
    dout, out = _bf16_cuda(dout, "dout"), _bf16_cuda(out, "out")
    for name, t in (("dout", dout), ("out", out)):
        if t.shape != (total, n_heads * 64) or t.device != qkv.device:
            raise ValueError(f"{name} must be [{total}, {n_heads * 64}] on {qkv.device}, got {tuple(t.shape)} on {t.device}")
    if lse.dtype != torch.float32 or lse.shape != (n_heads, total) or lse.device != qkv.device:
        raise ValueError(f"lse must be fp32 [{n_heads}, {total}] on {qkv.device}")
    if int(max_seqlen) <= 0:
        raise ValueError("max_seqlen must be positive")
    dout, out, lse = _aligned(dout), _aligned(out), lse.contiguous()
    dqkv = torch.empty_like(qkv)
    if total == 0:
        return dqkv
    with _Call(qkv) as c:
        ws_bytes = int(c.lib.pe_attn_backward_workspace_bytes(total, n_heads))
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=qkv.device)
        _lib.check(c.lib.pe_attn_varlen_backward(
            dout.data_ptr(), qkv.data_ptr(), out.data_ptr(), lse.data_ptr(), cu.data_ptr(), cu.numel() - 1, total,
            n_heads, _window(half_window, total), _lib.ptr(pos), _lib.ptr(table),
            0 if table is None else table.shape[0], dqkv.data_ptr(), ws.data_ptr(), ws_bytes,
            status_word(qkv.device).data_ptr(), c.stream), "pe_attn_varlen_backward")
    return dqkv


def rope_qk(qkv: Tensor, position_ids: Tensor, table: Tensor, n_heads: int) -> Tensor:
    """`rope_qk_inplace` into a new tensor: one pass that reads `qkv` and writes it with q and k rotated."""
    qkv = _bf16_cuda(qkv, "qkv")
    if n_heads <= 0 or qkv.dim() != 2 or qkv.shape[1] != 3 * n_heads * 64:
        raise ValueError(f"qkv must be [T, 3 * {n_heads} * 64], got {tuple(qkv.shape)}")
    pos, table = _rotation_args(position_ids, table, qkv)
    if table is None:
        raise ValueError("rope_qk needs position_ids and table")
    qkv = _aligned(qkv)
    out = torch.empty_like(qkv)
    with _Call(qkv) as c:
        _lib.check(c.lib.pe_rope_qk(qkv.data_ptr(), pos.data_ptr(), table.data_ptr(), table.shape[0], qkv.shape[0],
                                    n_heads, out.data_ptr(), status_word(qkv.device).data_ptr(), c.stream), "pe_rope_qk")
    return out


class _AttentionVarlen(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, cu_seqlens, max_seqlen, n_heads, half_window, position_ids, table):
        if table is not None:
            qkv = rope_qk(qkv.detach(), position_ids, table, n_heads)
        out, lse = attention_varlen_qkv_lse(qkv, cu_seqlens, max_seqlen, n_heads, half_window)
        ctx.save_for_backward(qkv, out, lse, cu_seqlens, position_ids, table)
        ctx.sizes = (max_seqlen, n_heads, half_window)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        qkv, out, lse, cu_seqlens, position_ids, table = ctx.saved_tensors
        dqkv = attention_varlen_qkv_backward(dout, qkv, out, lse, cu_seqlens, *ctx.sizes, position_ids=position_ids,
                                             table=table)
        return dqkv, None, None, None, None, None, None


def attention_varlen_qkv_train(qkv: Tensor, cu_seqlens: Tensor, max_seqlen: int, n_heads: int,
                               half_window: int | None, *, position_ids: Tensor | None = None,
                               table: Tensor | None = None) -> Tensor:
    """`attention_varlen_qkv` for autograd: the result has a gradient with respect to `qkv`. With
    `position_ids` and `table` (see `rope_table`) `qkv` is taken before the rotation of q and k,
    which then happens inside on a copy, and the gradient is turned back in the same kernel that
    computes it. Keeps the (rotated) qkv, the output and 4 bytes per token and head for the
    backward pass."""
    qkv, _ = _attention_args(qkv, cu_seqlens, n_heads, half_window)
    _rotation_args(position_ids, table, qkv)
    return _AttentionVarlen.apply(qkv, cu_seqlens, int(max_seqlen), n_heads, half_window, position_ids, table)


_ELEMENT_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def _element_cuda(t: Tensor, name: str) -> Tensor:
    if not isinstance(t, Tensor) or not t.is_cuda or t.dtype not in _ELEMENT_TYPES:
        kind = f"{t.dtype} on {t.device}" if isinstance(t, Tensor) else type(t).__name__
        raise PackedEncodersError(f"{name} must be a CUDA bf16, fp16 or fp32 tensor, got {kind}")
    return t


def dropout_positions(numel: int) -> int:
    """How far a `dropout` call over `numel` elements moves along the generator: add it to `rng[1]`
    before the next call, or calls share their random numbers."""
    return (numel + 7) // 8


def _dropout_call(x: Tensor, p: float, rng: Tensor, residual: Tensor | None, keep_rng: bool):
    x = _element_cuda(x, "x").contiguous()
    if not 0.0 <= float(p) <= 1.0:
        raise ValueError(f"dropout: p must be within [0, 1], got {p}")
    rng = _index_cuda(rng, "rng", torch.int64, x)
    if rng.shape != (2,):
        raise ValueError(f"rng must hold two numbers, seed and position, got {tuple(rng.shape)}")
    if residual is not None:
        if _element_cuda(residual, "residual").dtype != x.dtype or residual.shape != x.shape or residual.device != x.device:
            raise ValueError("residual must have the type, shape and device of x")
        residual = residual.contiguous()
    y = torch.empty_like(x)
    used = torch.empty(2, dtype=torch.int64, device=x.device) if keep_rng else None
    with _Call(x) as c:
        _lib.check(c.lib.pe_dropout(x.data_ptr(), _lib.ptr(residual), _ELEMENT_TYPES[x.dtype], x.numel(), float(p),
                                    rng.data_ptr(), _lib.ptr(used), y.data_ptr(), c.stream), "pe_dropout")
    return y, used


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, rng, residual):
        y, used = _dropout_call(x, p, rng, residual, True)
        ctx.p = p
        ctx.has_residual = residual is not None
        ctx.save_for_backward(used)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        (used,) = ctx.saved_tensors
        dx = dropout_backward(dy, ctx.p, used) if ctx.needs_input_grad[0] else None
        return dx, None, None, dy if ctx.has_residual else None


def dropout(x: Tensor, p: float, rng: Tensor, *, residual: Tensor | None = None) -> Tensor:
    """`x` with each element dropped with probability `p` and the others divided by `1 - p`, plus
    `residual` if given, in one pass. The mask is not stored: it is a function of `rng`, an int64
    CUDA tensor `[seed, position]`, and the element's number in the (contiguous) order of `x`, so
    equal `rng` gives equal masks whatever the layout, and a captured call reads the values that
    `rng` holds at replay. `p` counts in steps of 2^-16. Differentiable in `x` and `residual`; the
    gradient uses the numbers of its own forward even if `rng` has moved on since."""
    if torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad)):
        return _Dropout.apply(x, float(p), rng, residual)
    return _dropout_call(x, p, rng, residual, False)[0]


def dropout_backward(dy: Tensor, p: float, rng: Tensor) -> Tensor:
    """Gradient of `dropout` with respect to `x`: the same elements dropped, the others scaled."""
    return _dropout_call(dy, p, rng, None, False)[0]


class TokenLogprobs(NamedTuple):
    """Result of `token_logprobs`; every field has the shape of `targets` (the last two with one
    more dimension of `top_k`; `None` without it)."""

    logprobs: Tensor       # fp32: log p(target), 0 where ignored
    entropy: Tensor        # fp32: -sum p log p, in nats
    lse: Tensor            # fp32: log sum exp of the logits
    lse_rest: Tensor       # fp32: what the rounding of lse left; log p = (x - lse) - lse_rest
    top_ids: Tensor | None       # int64, largest logit first, equal ones by lowest index
    top_logprobs: Tensor | None  # fp32


def _logit_rows(logits: Tensor, name: str) -> tuple[Tensor, int]:
    """`[rows, vocab]` view and its row stride; only the last dimension has to be contiguous."""
    _element_cuda(logits, name)
    if logits.dim() < 1 or logits.shape[-1] == 0:
        raise ValueError(f"{name} must be [..., vocab] with a vocabulary, got {tuple(logits.shape)}")
    rows = logits if logits.dim() == 2 else logits.reshape(-1, logits.shape[-1])
    if rows.stride(1) != 1 or (rows.shape[0] > 1 and rows.stride(0) < rows.shape[1]):
        rows = rows.contiguous()
    return rows, rows.stride(0) if rows.shape[0] > 1 else rows.shape[1]


def _targets_for(targets: Tensor, logits: Tensor) -> Tensor:
    targets = _index_cuda(targets, "targets", torch.int64, logits)
    if targets.shape != logits.shape[:-1]:
        raise ValueError(f"targets must be {tuple(logits.shape[:-1])}, got {tuple(targets.shape)}")
    return targets.reshape(-1)


def _logprobs_call(logits: Tensor, targets: Tensor, top_k: int, ignore_index: int, separate: bool) -> TokenLogprobs:
    rows, ld = _logit_rows(logits, "logits")
    flat = _targets_for(targets, logits)
    vocab, lead = rows.shape[1], logits.shape[:-1]
    if not 0 <= top_k <= min(32, vocab):
        raise ValueError(f"top_k must be within 0..{min(32, vocab)}, got {top_k}")
    n, dev = rows.shape[0], logits.device
    if separate:  # outputs of an autograd function that the caller may change in place
        stats = [torch.empty(n, dtype=torch.float32, device=dev) for _ in range(4)]
    else:
        stats = torch.empty(4, n, dtype=torch.float32, device=dev).unbind(0)
    ids = torch.empty(n, top_k, dtype=torch.int64, device=dev) if top_k else None
    top = torch.empty(n, top_k, dtype=torch.float32, device=dev) if top_k else None
    with _Call(logits) as c:
        _lib.check(c.lib.pe_token_logprobs(rows.data_ptr(), _ELEMENT_TYPES[rows.dtype], n, vocab, ld, flat.data_ptr(),
                                           int(ignore_index), top_k, stats[0].data_ptr(), stats[1].data_ptr(),
                                           stats[2].data_ptr(), stats[3].data_ptr(), _lib.ptr(ids), _lib.ptr(top),
                                           status_word(dev).data_ptr(), c.stream), "pe_token_logprobs")
    if len(lead) != 1:
        stats = [s.view(lead) for s in stats]
        ids, top = ((t.view(*lead, top_k) if top_k else None) for t in (ids, top))
    return TokenLogprobs(*stats, ids, top)


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, top_k, ignore_index):
        r = _logprobs_call(logits, targets, top_k, ignore_index, True)
        ctx.save_for_backward(logits, targets, r.lse, r.lse_rest, r.entropy)
        ctx.ignore_index = ignore_index
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(r.lse_rest, *((r.top_ids, r.top_logprobs) if top_k else ()))
        return tuple(r)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_logprobs, d_entropy, d_lse, _rest, _ids, _top):
        logits, targets, lse, lse_rest, entropy = ctx.saved_tensors
        if d_logprobs is None and d_entropy is None and d_lse is None:
            return None, None, None, None
        forward = TokenLogprobs(None, entropy, lse, lse_rest, None, None)
        return token_logprobs_backward(logits, targets, forward, d_logprobs, d_entropy, d_lse=d_lse,
                                       ignore_index=ctx.ignore_index), None, None, None


def token_logprobs(logits: Tensor, targets: Tensor, *, top_k: int = 0, ignore_index: int = -100) -> TokenLogprobs:
    """Log-probabilities of `targets` (int64, `logits.shape[:-1]`) under `logits` `[..., vocab]` (bf16,
    fp16 or fp32; rows may be strided, as in a padded vocabulary's slice), with the entropy and
    the `top_k` (at most 32) most likely tokens, in one pass over the logits in fp32. The mean of
    `-logprobs` over the rows that are not ignored is the cross-entropy loss. `-inf` logits have
    probability 0. Differentiable through `logprobs`, `entropy` and `lse`, not through the top."""
    if torch.is_grad_enabled() and isinstance(logits, Tensor) and logits.requires_grad:
        return TokenLogprobs(*_TokenLogprobs.apply(logits, targets, int(top_k), int(ignore_index)))
    return _logprobs_call(logits, targets, int(top_k), int(ignore_index), False)


def token_logprobs_backward(logits: Tensor, targets: Tensor, forward: TokenLogprobs, d_logprobs: Tensor | None,
                            d_entropy: Tensor | None = None, *, d_lse: Tensor | None = None,
                            ignore_index: int = -100, inplace: bool = False) -> Tensor:
    """Gradient of `token_logprobs` with respect to `logits`, from what it returned (`forward`) and the
    gradients of `logprobs`, `entropy` and `lse` (`None`: zero). `inplace=True` writes it over `logits`, which saves the largest
    buffer of a training step."""
    rows, ld = _logit_rows(logits, "logits")
    flat = _targets_for(targets, logits)
    n, vocab = rows.shape
    per_row = []
    for name, t in (("lse", forward.lse), ("lse_rest", forward.lse_rest), ("entropy", forward.entropy), ("d_logprobs", d_logprobs), ("d_entropy", d_entropy),
                    ("d_lse", d_lse)):
        if t is not None:
            if t.dtype != torch.float32 or t.shape != targets.shape or t.device != logits.device:
                raise ValueError(f"{name} must be fp32 {tuple(targets.shape)} on {logits.device}")
            t = t.reshape(-1).contiguous()
        per_row.append(t)
    if inplace:
        if rows.data_ptr() != logits.data_ptr():
            raise PackedEncodersError("logits must be rows of a contiguous vocabulary to be written over")
        out, ld_out = rows, ld
    else:
        out = torch.empty(n, vocab, dtype=logits.dtype, device=logits.device)
        ld_out = vocab
    with _Call(logits) as c:
        _lib.check(c.lib.pe_token_logprobs_backward(
            rows.data_ptr(), _ELEMENT_TYPES[rows.dtype], n, vocab, ld, flat.data_ptr(), int(ignore_index),
            *(_lib.ptr(t) for t in per_row), out.data_ptr(), ld_out, c.stream), "pe_token_logprobs_backward")
    return logits if inplace else out.view(logits.shape)
