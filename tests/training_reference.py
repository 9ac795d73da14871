"""The training operators in 64 bits, from their definitions, with a bound for every element of what
the kernels may be off by.

The bounds count roundings: EPS = 2^-8 is half a step of bf16 relative to the value (what P, dS and
the results are rounded to), ETA = 2^-16 covers what is done in fp32 (exponentials, sums of up to
some thousand products) with a wide margin and stays far below EPS.
"""
from __future__ import annotations

import math

import numpy as np
import torch

EPS = 2.0 ** -8
ETA = 2.0 ** -16


def attention(qkv, dout, lengths, n_heads, half_window):
    """(out, lse, dqkv) of the packed attention and bounds of the kernels' errors, all float64.
    Rows outside the sequences: 0, -inf, 0. `qkv` [T, 3 * n_heads * 64] as the kernels read it."""
    total = qkv.shape[0]
    dev = qkv.device
    x = qkv.double().view(total, 3, n_heads, 64)
    go = dout.double().view(total, n_heads, 64)
    out = torch.zeros(total, n_heads, 64, dtype=torch.float64, device=dev)
    lse = torch.full((n_heads, total), -math.inf, dtype=torch.float64, device=dev)
    grad = torch.zeros_like(x)
    e_out, e_lse, e_grad = torch.zeros_like(out), torch.zeros_like(lse), torch.zeros_like(grad)
    begin = 0
    for s in lengths:
        here = slice(begin, begin + s)
        begin += s
        if s == 0:
            continue
        q, k, v = (x[here, i].transpose(0, 1) for i in range(3))  # [nh, s, 64]
        g = go[here].transpose(0, 1)
        scores = q @ k.transpose(1, 2) / 8.0
        size = q.abs() @ k.abs().transpose(1, 2) / 8.0
        if half_window is not None:
            i = torch.arange(s, device=dev)
            scores = scores.masked_fill((i[:, None] - i[None, :]).abs() > half_window, -math.inf)
        z = torch.logsumexp(scores, dim=-1)
        p = torch.exp(scores - z.unsqueeze(-1))
        o = p @ v
        dp = g @ v.transpose(1, 2)
        delta = (g * o).sum(-1, keepdim=True)
        ds = p * (dp - delta)
        # out: P rounded, then the result
        eo = (EPS + ETA) * (p @ v.abs()) + EPS * o.abs()
        # delta comes from the rounded out; dP and delta are fp32 sums; dS is rounded
        e_delta = (g.abs() * eo).sum(-1, keepdim=True) + ETA * (g.abs() * o.abs()).sum(-1, keepdim=True)
        e_ds = p * (e_delta + ETA * (g.abs() @ v.abs().transpose(1, 2))) + (EPS + ETA) * ds.abs()
        out[here] = o.transpose(0, 1)
        lse[:, here] = z
        dq, dk, dv = ds @ k / 8.0, ds.transpose(1, 2) @ q / 8.0, p.transpose(1, 2) @ g
        for i, (value, error) in enumerate(((dq, e_ds @ k.abs() / 8.0), (dk, e_ds.transpose(1, 2) @ q.abs() / 8.0),
                                            (dv, (EPS + ETA) * (p.transpose(1, 2) @ g.abs())))):
            grad[here, i] = value.transpose(0, 1)
            e_grad[here, i] = (error * (1 + EPS) + EPS * value.abs()).transpose(0, 1)
        e_out[here] = (eo * (1 + EPS)).transpose(0, 1)
        e_lse[:, here] = ETA + 2.0 ** -20 * torch.where(p > 0, size, torch.zeros_like(size)).amax(-1)
    return ((out.view(total, -1), lse, grad.view(total, -1)),
            (e_out.view(total, -1), e_lse, e_grad.view(total, -1)))


def rotate(x, cos, sin):
    """x [T, heads, 64]: the pair (j, j + 32) turned by its angle."""
    lo, hi = x[..., :32], x[..., 32:]
    return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], dim=-1)


def philox(counter, seed):
    """Philox4x32-10 on numpy uint64 counters: [n, 4] 32-bit words."""
    mask = np.uint64(0xFFFFFFFF)
    half = np.uint64(32)
    c = [counter & mask, counter >> half, np.zeros_like(counter), np.zeros_like(counter)]
    k0, k1 = seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> half) ^ c[1] ^ np.uint64(k0), b & mask, (a >> half) ^ c[3] ^ np.uint64(k1), a & mask]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack(c, axis=1)


def dropout_keep(n, p, seed, position):
    """Which of n elements survive, and the factor of the survivors."""
    with np.errstate(over="ignore"):
        counter = np.arange((n + 7) // 8, dtype=np.uint64) + np.uint64(position % 2 ** 64)
    words = philox(counter, seed).astype(np.uint32)
    fields = np.stack([words & 0xFFFF, words >> 16], axis=2).reshape(-1)[:n]
    threshold = int(math.floor(p * 65536.0 + 0.5))
    return torch.from_numpy(fields >= threshold), (65536.0 / (65536 - threshold) if threshold < 65536 else 0.0)


def logprobs(logits, targets, top_k=0, ignore_index=-100):
    """(logprobs, entropy, lse, top_ids, top_logprobs) in float64; equal logits by lowest index."""
    x = logits.double()
    logp = torch.log_softmax(x, dim=-1)
    kept = targets != ignore_index
    at = torch.where(kept, targets, torch.zeros_like(targets))
    chosen = torch.where(kept, logp.gather(-1, at.unsqueeze(-1)).squeeze(-1), torch.zeros_like(logp[..., 0]))
    p = torch.exp(logp)
    entropy = -torch.where(p == 0, torch.zeros_like(p), p * logp).sum(-1)
    ids = torch.sort(x, dim=-1, descending=True, stable=True)[1][..., :top_k]
    return chosen, entropy, torch.logsumexp(x, -1), ids, logp.gather(-1, ids)


def logprobs_gradient(logits, targets, g, h, z, ignore_index=-100):
    logp = torch.log_softmax(logits.double(), dim=-1)
    p = torch.exp(logp)
    finite = torch.where(p == 0, torch.zeros_like(p), logp)
    entropy = -(p * finite).sum(-1, keepdim=True)
    kept = targets != ignore_index
    g = torch.where(kept, g.double(), torch.zeros_like(g.double())).unsqueeze(-1)
    d = p * (z.double().unsqueeze(-1) - g - h.double().unsqueeze(-1) * (finite + entropy))
    return d.scatter_add(-1, torch.where(kept, targets, torch.zeros_like(targets)).unsqueeze(-1), g)
