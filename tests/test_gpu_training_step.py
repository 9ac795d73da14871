"""The training operators in one step, as a training loop would chain them: projection, rotated packed
attention, dropout with the residual, vocabulary logits, token log-probabilities, and back.  Every
operator's gradient is compared with the 64-bit formula at the values it was given in that step."""
from __future__ import annotations

import pytest
import torch

import training_reference as R

pytestmark = pytest.mark.gpu

LENGTHS, HEADS, WIDTH, VOCAB, P = [37, 1, 0, 200, 64, 129], 2, 128, 517, 0.1


def _data(device, seed=0):
    gen = torch.Generator().manual_seed(seed)
    total = sum(LENGTHS)
    cu = torch.zeros(len(LENGTHS) + 1, dtype=torch.int32)
    cu[1:] = torch.tensor(LENGTHS).cumsum(0)
    targets = torch.randint(0, VOCAB, (total,), generator=gen)
    targets[::5] = -100
    put = lambda t: t.to(device, torch.bfloat16)  # noqa: E731
    return {
        "x": put(torch.randn(total, WIDTH, generator=gen)),
        "wqkv": put(torch.randn(3 * WIDTH, WIDTH, generator=gen) * WIDTH ** -0.5),
        "head": put(torch.randn(VOCAB, WIDTH, generator=gen) * WIDTH ** -0.5),
        "cu": cu.to(device), "pos": torch.cat([torch.arange(s) for s in LENGTHS]).to(device),
        "targets": targets.to(device), "weight": torch.rand(total, generator=gen).to(device),
        "rng": torch.tensor([1234, 5], dtype=torch.int64, device=device),
    }


@pytest.mark.parametrize("hw", [None, 16])
def test_step_with_autograd(pe, cuda_device, hw):
    from flash_modernbert_b200 import ops

    d = _data(cuda_device)
    table = ops.rope_table(10000.0, 200, cuda_device)
    x, wqkv, head = (d[k].requires_grad_(True) for k in ("x", "wqkv", "head"))
    qkv = x @ wqkv.t()
    ctx = ops.attention_varlen_qkv_train(qkv, d["cu"], max(LENGTHS), HEADS, hw, position_ids=d["pos"], table=table)
    h = ops.dropout(ctx, P, d["rng"], residual=x)
    logits = h @ head.t()
    r = ops.token_logprobs(logits, d["targets"], top_k=5)
    loss = -(r.logprobs * d["weight"]).sum() - 0.01 * r.entropy.sum()
    for t in (qkv, ctx, h, logits):
        t.retain_grad()
    loss.backward()
    ops.check_status(cuda_device)

    # log-probabilities: relative to p 2^-17 and the exponent's 2^-22 of the largest difference, then one
    # rounding; |log p + entropy| < 40 for logits of this size
    g, e = -d["weight"], torch.full_like(d["weight"], -0.01)
    ref = R.logprobs_gradient(logits.detach(), d["targets"], g, e, torch.zeros_like(g))
    p = torch.softmax(logits.detach().double(), -1)
    rel = 2.0 ** -17 + 2 * float(logits.detach().abs().max()) * 2.0 ** -22
    bound = R.EPS * ref.abs() + rel * p * (g.abs() + 40 * e.abs()).double().unsqueeze(-1) * (1 + R.EPS) \
        + 2.0 ** -23 * g.abs().double().unsqueeze(-1)
    assert float(((logits.grad.double() - ref).abs() - bound).max()) <= 0
    chosen, entropy, _, ids, _ = R.logprobs(logits.detach(), d["targets"], top_k=5)
    assert torch.equal(r.top_ids, ids)
    assert float((loss.detach().double() - (-(chosen * d["weight"]).sum() - 0.01 * entropy.sum())).abs()) <= 2.0 ** -16 * (
        float((chosen.abs() * d["weight"]).sum()) + 0.01 * float(entropy.sum()))

    # dropout with the residual
    keep, scale = R.dropout_keep(ctx.numel(), P, 1234, 5)
    keep = keep.view(ctx.shape).to(cuda_device)
    sum_ = torch.where(keep, ctx.detach().double() * scale, torch.zeros((), dtype=torch.float64, device=cuda_device))
    bound = R.EPS * (sum_ + x.detach().double()).abs() + 2.0 ** -22 * (sum_.abs() + x.detach().double().abs())
    assert float(((h.detach().double() - sum_ - x.detach().double()).abs() - bound).max()) <= 0
    back = torch.where(keep, h.grad.double() * scale, torch.zeros_like(sum_))
    assert float(((ctx.grad.double() - back).abs() - (R.EPS + 2.0 ** -22) * back.abs()).max()) <= 0

    # attention, on the rotated q and k as they were rounded; its gradient turned back in fp32
    rotated = ops.rope_qk_inplace(qkv.detach().clone(), d["pos"], table, HEADS)
    (out, _, grad), (e_out, _, e_grad) = R.attention(rotated, ctx.grad, LENGTHS, HEADS, hw)
    assert float(((ctx.detach().double() - out).abs() - e_out).max()) <= 0
    cos, sin = table.double()[d["pos"]].unsqueeze(1).split(32, dim=-1)
    grad, e_grad = (t.view(-1, 3, HEADS, 64).clone() for t in (grad, e_grad))
    for i in (0, 1):
        grad[:, i] = R.rotate(grad[:, i], cos, -sin)
        e_grad[:, i] = R.rotate(e_grad[:, i], cos.abs(), -sin.abs()).abs() \
            + R.rotate(e_grad[:, i], cos.abs(), sin.abs()).abs() + R.EPS * grad[:, i].abs()
    assert float(((qkv.grad.double().view_as(grad) - grad).abs() - e_grad).max()) <= 0

    # the leaves: the residual's share and the projection's
    share = h.grad.double() + qkv.grad.double() @ wqkv.detach().double()
    size = h.grad.double().abs() + qkv.grad.double().abs() @ wqkv.detach().double().abs()
    # each share rounded to bf16, then their sum
    assert float(((x.grad.double() - share).abs() - 3 * R.EPS * size - R.EPS * share.abs()).max()) <= 0
    assert all(bool(torch.isfinite(t.grad).all()) for t in (x, wqkv, head))


def test_captured_step(pe, cuda_device):
    """The same chain from the operators' own backward calls, captured once: each replay uses the numbers
    that `rng` holds then and gives the bits of the eager calls."""
    from flash_modernbert_b200 import ops

    d = _data(cuda_device, seed=1)
    table = ops.rope_table(10000.0, 200, cuda_device)
    longest = max(LENGTHS)

    def step():
        qkv = ops.rope_qk_inplace(d["x"] @ d["wqkv"].t(), d["pos"], table, HEADS)
        ctx, lse = ops.attention_varlen_qkv_lse(qkv, d["cu"], longest, HEADS, 16)
        h = ops.dropout(ctx, P, d["rng"], residual=d["x"])
        logits = h @ d["head"].t()
        r = ops.token_logprobs(logits, d["targets"])
        d_logits = ops.token_logprobs_backward(logits, d["targets"], r, -d["weight"], inplace=True)
        d_h = d_logits @ d["head"]
        d_ctx = ops.dropout_backward(d_h, P, d["rng"])
        d_qkv = ops.attention_varlen_qkv_backward(d_ctx, qkv, ctx, lse, d["cu"], longest, HEADS, 16,
                                                  position_ids=d["pos"], table=table)
        d["rng"][1] += ops.dropout_positions(ctx.numel())
        return r.logprobs, d_h, d_qkv

    start = d["rng"].clone()
    eager = []
    for _ in range(3):
        eager.append([t.clone() for t in step()])
    assert not torch.equal(eager[0][2], eager[1][2])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        result = step()
    d["rng"].copy_(start)
    for i in range(3):
        graph.replay()
        for name, a, b in zip(("logprobs", "d_h", "d_qkv"), result, eager[i]):
            assert torch.equal(a, b), (i, name)
    ops.check_status(cuda_device)
