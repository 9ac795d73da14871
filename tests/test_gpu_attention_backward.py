"""Packed attention with its gradient (`attention_varlen_qkv_lse`, `attention_varlen_qkv_backward`,
`attention_varlen_qkv_train`) against the 64-bit definition, element by element within the bound that
the roundings to bf16 give."""
from __future__ import annotations

import math

import pytest
import torch

import training_reference as R

pytestmark = pytest.mark.gpu


def _case(lengths, n_heads, device, seed=0, scale=1.0, tail=0):
    gen = torch.Generator().manual_seed(seed)
    total = sum(lengths) + tail
    qkv = torch.randn(total, 3, n_heads, 64, generator=gen)
    qkv[:, 0] *= scale
    dout = torch.randn(total, n_heads * 64, generator=gen) * 0.1
    cu = torch.zeros(len(lengths) + 1, dtype=torch.int32)
    cu[1:] = torch.tensor(lengths).cumsum(0)
    return (qkv.reshape(total, -1).to(device, torch.bfloat16), dout.to(device, torch.bfloat16), cu.to(device))


def _both(qkv, dout, cu, longest, n_heads, hw):
    from flash_modernbert_b200 import ops

    out, lse = ops.attention_varlen_qkv_lse(qkv, cu, longest, n_heads, hw)
    dqkv = ops.attention_varlen_qkv_backward(dout, qkv, out, lse, cu, longest, n_heads, hw)
    ops.check_status(qkv.device)
    return out, lse, dqkv


def _within(got, ref, bound, what):
    for name, a, b, e in zip(("out", "lse", "dqkv"), got, ref, bound):
        same = a.double() == b  # rows outside every sequence: -inf, exact zeros
        excess = torch.where(same, torch.zeros_like(b), (a.double() - b).abs() - e)
        assert not torch.isnan(excess).any() and float(excess.max()) <= 0.0, (what, name, float(excess.max()))


def _check(lengths, n_heads, hw, device, **kw):
    qkv, dout, cu = _case(lengths, n_heads, device, **kw)
    got = _both(qkv, dout, cu, max(lengths + [1]), n_heads, hw)
    ref, bound = R.attention(qkv, dout, lengths, n_heads, hw)
    _within(got, ref, bound, (lengths, n_heads, hw, kw))


@pytest.mark.parametrize("hw", [None, 64])
@pytest.mark.parametrize("lengths", [[1], [2], [64], [65], [127], [128], [129], [255], [256], [257]])
def test_one_sequence(pe, cuda_device, lengths, hw):
    _check(lengths, 2, hw, cuda_device, seed=1)


@pytest.mark.parametrize("n_heads", [1, 3, 12])
@pytest.mark.parametrize("hw", [None, 0, 1, 5, 64, 200, 100000])
def test_ragged_batch(pe, cuda_device, n_heads, hw):
    """Many sequences to a tile, one sequence over many tiles, empty slots in between."""
    _check([3, 0, 30, 1, 1, 48, 200, 0, 0, 17, 128, 128, 65, 700, 5, 0], n_heads, hw, cuda_device, seed=2)


@pytest.mark.parametrize("hw", [None, 64])
def test_queries_only(pe, cuda_device, hw):
    _check([8 + (7 * i) % 41 for i in range(70)], 4, hw, cuda_device, seed=3)


@pytest.mark.parametrize("hw", [None, 64, 300])
def test_long_sequence(pe, cuda_device, hw):
    _check([4100, 3], 2, hw, cuda_device, seed=4)


@pytest.mark.parametrize("hw", [None, 64])
def test_many_tiles_per_block(pe, cuda_device, hw):
    """Every thread block works through dozens of tiles of one, two or many columns in turn."""
    lengths = [(37 * i) % 300 + 1 for i in range(150)] + [8 + i % 40 for i in range(150)] + [2500]
    _check(lengths, 12, hw, cuda_device, seed=16)


@pytest.mark.parametrize("hw", [None, 1500])
def test_deep_column_walks(pe, cuda_device, hw):
    """Blocks that walk hundreds of column tiles per item, several items each, row tiles of two sequences."""
    _check([6000, 2100, 1], 4, hw, cuda_device, seed=17)


@pytest.mark.parametrize("scale", [0.01, 4.0, 16.0])
def test_flat_and_peaked_scores(pe, cuda_device, scale):
    _check([300, 40], 2, None, cuda_device, seed=5, scale=scale)


@pytest.mark.parametrize("hw", [None, 64])
def test_rows_of_no_sequence(pe, cuda_device, hw):
    """Rows behind the last sequence get zeros (and -inf in lse); whatever they hold when the gradient
    is taken, NaN included, reaches no other row."""
    from flash_modernbert_b200 import ops

    lengths = [100, 61, 200]
    qkv, dout, cu = _case(lengths, 2, cuda_device, seed=6, tail=150)
    got = _both(qkv, dout, cu, 200, 2, hw)
    ref, bound = R.attention(qkv, dout, lengths, 2, hw)
    _within(got, ref, bound, hw)
    out, lse, dqkv = got
    total = sum(lengths)
    dirty = [t.clone() for t in (dout, qkv, out)]
    for t in dirty:
        t[total:] = math.nan
    dirty_lse = lse.clone()
    dirty_lse[:, total:] = math.nan
    again = ops.attention_varlen_qkv_backward(*dirty, dirty_lse, cu, 200, 2, hw)
    assert torch.equal(again[:total], dqkv[:total])
    assert torch.equal(again[total:], torch.zeros_like(again[total:]))


def test_all_slots_empty(pe, cuda_device):
    qkv, dout, _ = _case([5], 2, cuda_device)
    cu = torch.zeros(4, dtype=torch.int32, device=cuda_device)
    out, lse, dqkv = _both(qkv, dout, cu, 5, 2, None)
    assert not out.any() and not dqkv.any() and bool((lse == -math.inf).all())
    none = qkv[:0], dout[:0], cu
    out, lse, dqkv = _both(*none, 5, 2, None)
    assert out.shape == (0, 128) and lse.shape == (2, 0) and dqkv.shape == (0, 384)


def test_output_is_that_of_the_inference_operator(pe, cuda_device):
    from flash_modernbert_b200 import ops

    for lengths, hw in (([30, 12, 64], None), ([300, 20, 129], None), ([300, 20, 129], 64), ([300, 20, 129], 9)):
        qkv, dout, cu = _case(lengths, 3, cuda_device, seed=7)
        out, _, _ = _both(qkv, dout, cu, max(lengths), 3, hw)
        assert torch.equal(out, ops.attention_varlen_qkv(qkv, cu, max(lengths), 3, hw))


def test_same_bits_alone_in_a_batch_and_again(pe, cuda_device):
    """Calls are deterministic, on any stream, two at a time."""
    lengths = [40, 300, 9, 513]
    qkv, dout, cu = _case(lengths, 12, cuda_device, seed=8)
    first = _both(qkv, dout, cu, 513, 12, 64)
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    results = []
    torch.cuda.synchronize()
    for s in side:
        with torch.cuda.stream(s):
            from flash_modernbert_b200 import ops

            out, lse = ops.attention_varlen_qkv_lse(qkv, cu, 513, 12, 64)
            results.append((out, lse, ops.attention_varlen_qkv_backward(dout, qkv, out, lse, cu, 513, 12, 64)))
    torch.cuda.synchronize()
    for r in results:
        assert all(torch.equal(a, b) for a, b in zip(first, r))


def test_gradient_against_differences(pe, cuda_device):
    """<gradient, v> against the central difference of the 64-bit output along v."""
    lengths, n_heads, hw = [130, 20], 2, 40
    qkv, dout, cu = _case(lengths, n_heads, cuda_device, seed=9)
    dqkv = _both(qkv, dout, cu, 130, n_heads, hw)[2].double()
    bound = R.attention(qkv, dout, lengths, n_heads, hw)[1][2]
    gen = torch.Generator(device=cuda_device).manual_seed(10)
    for _ in range(3):
        v = torch.randn(qkv.shape, generator=gen, device=cuda_device, dtype=torch.float64)
        h = 1e-5
        up, down = (float((R.attention(qkv.double() + s * h * v, dout, lengths, n_heads, hw)[0][0] * dout.double()).sum())
                    for s in (1, -1))
        # the difference itself is good to h^2 and to the cancellation of two sums: 1e-6 of their size
        assert abs((up - down) / (2 * h) - float((dqkv * v).sum())) <= float((bound * v.abs()).sum()) + 1e-6


@pytest.mark.parametrize("hw", [None, 64])
def test_rotation_inside(pe, cuda_device, hw):
    """With a table: q and k rotated on the way in (rounded to bf16, as everywhere in the package), the
    gradient turned back on the way out."""
    from flash_modernbert_b200 import ops

    lengths, nh = [150, 33, 1, 20], 3
    raw, dout, cu = _case(lengths, nh, cuda_device, seed=11)
    table = ops.rope_table(10000.0, 160, cuda_device)
    pos = torch.cat([torch.arange(s) for s in lengths]).to(cuda_device)
    rotated = ops.rope_qk_inplace(raw.clone(), pos, table, nh)
    (out, _, grad), (e_out, _, e_grad) = R.attention(rotated, dout, lengths, nh, hw)
    cos, sin = table.double()[pos].unsqueeze(1).split(32, dim=-1)
    g, e = grad.view(-1, 3, nh, 64).clone(), e_grad.view(-1, 3, nh, 64).clone()
    for i in (0, 1):
        # the accumulators are turned in fp32 before the one rounding: the bound turns with them
        g[:, i] = R.rotate(g[:, i], cos, -sin)
        e[:, i] = R.rotate(e[:, i], cos.abs(), -sin.abs()).abs() + R.rotate(e[:, i], cos.abs(), sin.abs()).abs() \
            + R.EPS * g[:, i].abs()
    leaf = raw.clone().requires_grad_(True)
    y = ops.attention_varlen_qkv_train(leaf, cu, 150, nh, hw, position_ids=pos, table=table)
    y.backward(dout)
    ops.check_status(cuda_device)
    assert torch.equal(leaf.detach(), raw)
    assert float(((y.detach().double() - out).abs() - e_out).max()) <= 0
    assert float(((leaf.grad.double().view_as(g) - g).abs() - e).max()) <= 0
    # without a table the operator takes the rotated qkv
    leaf2 = rotated.clone().requires_grad_(True)
    y2 = ops.attention_varlen_qkv_train(leaf2, cu, 150, nh, hw)
    assert torch.equal(y2.detach(), y.detach())
    y2.backward(dout)
    assert float(((leaf2.grad.double() - grad).abs() - e_grad).max()) <= 0


def test_bad_boundaries_and_positions_are_reported(pe, cuda_device):
    from flash_modernbert_b200 import _lib, ops

    qkv, dout, cu = _case([50, 60], 2, cuda_device, seed=12)
    out, lse = ops.attention_varlen_qkv_lse(qkv, cu, 60, 2, None)
    ops.check_status(cuda_device)
    for bad in ([0, 50, 111], [0, 60, 50], [-3, 50, 110]):
        wrong = torch.tensor(bad, dtype=torch.int32, device=cuda_device)
        g = ops.attention_varlen_qkv_backward(dout, qkv, out, lse, wrong, 60, 2, None)
        assert g.shape == qkv.shape
        with pytest.raises(_lib.NativeLibraryError, match="303"):
            ops.check_status(cuda_device)
    table = ops.rope_table(10000.0, 40, cuda_device)
    pos = torch.arange(110, device=cuda_device)
    ops.attention_varlen_qkv_backward(dout, qkv, out, lse, cu, 60, 2, None, position_ids=pos, table=table)
    with pytest.raises(_lib.NativeLibraryError, match="302"):
        ops.check_status(cuda_device)
    ops.check_status(cuda_device)


def test_strided_and_offset_inputs(pe, cuda_device):
    """Slices of wider buffers and views that start off a 16-byte boundary give the bits of contiguous copies."""
    from flash_modernbert_b200 import ops

    qkv, dout, cu = _case([70, 90], 2, cuda_device, seed=13)
    out, lse, dqkv = _both(qkv, dout, cu, 90, 2, 64)
    wide = torch.zeros(160, qkv.shape[1] + 6, dtype=torch.bfloat16, device=cuda_device)
    wide[:, 3:-3] = qkv
    flat = torch.zeros(dout.numel() + 1, dtype=torch.bfloat16, device=cuda_device)
    flat[1:] = dout.reshape(-1)
    off = flat[1:].view_as(dout)
    assert off.data_ptr() % 16 != 0
    out2, lse2 = ops.attention_varlen_qkv_lse(wide[:, 3:-3], cu, 90, 2, 64)
    assert torch.equal(out2, out) and torch.equal(lse2, lse)
    lse_t = lse.t().contiguous().t()
    assert torch.equal(ops.attention_varlen_qkv_backward(off, wide[:, 3:-3], out, lse_t, cu, 90, 2, 64), dqkv)


def test_captured_and_replayed(pe, cuda_device):
    """One graph for a capacity of tokens and sequences serves other contents and boundaries."""
    from flash_modernbert_b200 import ops

    nh, hw, cap = 2, 64, 400
    static = _case([cap], nh, cuda_device, seed=14)
    cu = torch.tensor([0, 100, 300, 400], dtype=torch.int32, device=cuda_device)

    def step():
        out, lse = ops.attention_varlen_qkv_lse(static[0], cu, cap, nh, hw)
        return out, lse, ops.attention_varlen_qkv_backward(static[1], static[0], out, lse, cu, cap, nh, hw)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for lengths in ([100, 200, 100], [1, 0, 70], [200, 150, 50]):
        qkv, dout, _ = _case([cap], nh, cuda_device, seed=15 + lengths[0])
        static[0].copy_(qkv)
        static[1].copy_(dout)
        cu.copy_(torch.tensor([0] + lengths).cumsum(0).to(torch.int32))
        graph.replay()
        ref, bound = R.attention(qkv, dout, lengths, nh, hw)
        _within(captured, ref, bound, lengths)
