"""The training operators of the packed encoder, as measured workloads: attention over packed
sequences with its gradient, counter-based dropout, and log-probabilities over a vocabulary with
entropy, top alternatives and their gradient.

`run` is one pass through an operator. With `own` false it is the plain form (elementary torch
operations in fp32, rounded once at the end); with `own` true it is the call a user makes of the
package. `exact` gives the same outputs from the definitions in 64 bits.
"""
from __future__ import annotations

import importlib.util
import math
import random
import sys
from pathlib import Path

import numpy as np
import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_HEAD = 64
_IGNORED = -100


def _package():
    """The package directory carries a hyphen, so it is loaded under its module name by path."""
    name = "flash_modernbert_b200"
    if name not in sys.modules:
        root = Path(__file__).resolve().parent.parent / "flash-modernbert_b200"
        spec = importlib.util.spec_from_file_location(name, root / "__init__.py",
                                                      submodule_search_locations=[str(root)])
        module = importlib.util.module_from_spec(spec)
        sys.modules[name] = module
        spec.loader.exec_module(module)
    from flash_modernbert_b200 import ops

    return ops


def _device() -> torch.device:
    return torch.device("cuda", torch.cuda.current_device()) if torch.cuda.is_available() else torch.device("cpu")


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------


def listed() -> list[dict]:
    return [
        # One packed handful of search queries in a fine-tuning step: a latency chain.
        dict(name="attention_four_queries", op="attention", kind="queries", n=4, len_seed=1, heads=12, window=64,
             rotate=False),
        # A contrastive query batch, 1,024 queries of 8 to 48 tokens (the query workload).
        dict(name="attention_queries", op="attention", kind="queries", n=1024, len_seed=2, heads=12, window=-1,
             rotate=False),
        # The document workload (512 documents, log-normal around 400 tokens), a full-attention layer.
        dict(name="attention_documents", op="attention", kind="documents", n=512, len_seed=4, heads=12, window=-1,
             rotate=False),
        # The same documents in a sliding-window layer, two thirds of a model's layers.
        dict(name="attention_documents_window", op="attention", kind="documents", n=512, len_seed=4, heads=12,
             window=64, rotate=False),
        # Long documents of 2,048 to 8,192 tokens, a full-attention layer of a small model (four heads).
        dict(name="attention_long", op="attention", kind="long", n=5, len_seed=5, heads=4, window=-1, rotate=False),
        # Queries, documents, single tokens and empty slots in one batch, an odd window, 28 heads, and
        # the position rotation inside the operator: through autograd, as a model's layer calls it.
        dict(name="attention_mixed_rotated", op="attention", kind="mixed", n=61, len_seed=4, heads=28, window=200,
             rotate=True),
        # Masked-token predictions for one short request: top 20 alternatives of three positions.
        dict(name="logprobs_request", op="logprobs", rows=3, vocab=50368, type="bf16", top_k=20, grad=False,
             forbidden=True),
        # The masked positions of a pretraining step (30 % of some 27,000 tokens), loss and gradient.
        dict(name="logprobs_masked_lm", op="logprobs", rows=8192, vocab=50368, type="bf16", top_k=0, grad=True,
             forbidden=False),
        # A large vocabulary with an odd size kept in fp32, loss and gradient with the entropy in it.
        dict(name="logprobs_large_vocab", op="logprobs", rows=515, vocab=256001, type="fp32", top_k=5, grad=True,
             forbidden=False),
        # Scoring a reranker's tokens: fp16 logits of an odd vocabulary, five alternatives.
        dict(name="logprobs_scoring", op="logprobs", rows=2049, vocab=30011, type="fp16", top_k=5, grad=False,
             forbidden=True),
        # A small fp32 activation with an odd width (a classifier head).
        dict(name="dropout_head", op="dropout", rows=33, width=769, type="fp32", p=0.5, residual=False),
        # Dropout of an attention output added to the residual stream of the document workload.
        dict(name="dropout_residual", op="dropout", rows=306851, width=768, type="bf16", p=0.1, residual=True),
    ]


def _log_uniform(rng: random.Random, lo: float, hi: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random) -> dict:
    op = rng.choice(["attention", "attention", "logprobs", "dropout"])
    if op == "attention":
        kind = rng.choice(["queries", "documents", "mixed", "long"])
        n = _log_uniform(rng, 1, {"queries": 1024, "long": 5}.get(kind, 128))
        return dict(op=op, kind=kind, n=n, len_seed=rng.randrange(1 << 20),
                    heads=rng.choice([1, 3, 4, 12] if kind == "long" else [1, 3, 4, 12, 28]),
                    window=rng.choice([-1, -1, 64, 64, _log_uniform(rng, 1, 400)]), rotate=rng.random() < 0.4)
    if op == "logprobs":
        vocab = _log_uniform(rng, 500, 262144)
        rows = _log_uniform(rng, 1, max(2, min(8192, 130_000_000 // vocab)))
        return dict(op=op, rows=rows, vocab=vocab, type=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                    top_k=rng.choice([0, 1, 5, 20]), grad=rng.random() < 0.6, forbidden=rng.random() < 0.4)
    width = _log_uniform(rng, 60, 5000)
    rows = _log_uniform(rng, 1, 150_000_000 // width)
    return dict(op=op, rows=rows, width=width, type=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                p=rng.choice([0.05, 0.1, 0.3, 0.5]), residual=rng.random() < 0.5)


def _lengths(case: dict) -> list[int]:
    rng = random.Random(case["len_seed"])

    def query():
        return rng.randint(8, 48)

    def document():
        return min(8192, max(64, int(round(math.exp(rng.gauss(math.log(400.0), 0.8))))))

    n = case["n"]
    if case["kind"] == "queries":
        return [query() for _ in range(n)]
    if case["kind"] == "documents":
        return [document() for _ in range(n)]
    if case["kind"] == "long":
        return [rng.randint(2048, 8192) for _ in range(n)]
    out = [query() if i % 2 else document() for i in range(n)]
    if n > 4:  # a window of a server: single tokens and unused slots among the rest
        out[1], out[n // 2], out[-1] = 1, 0, 0
    return out


def _pairs(lengths: list[int], window: int) -> int:
    """(query, key) pairs that attend: all of a sequence's, or those at most `window` apart."""
    total = 0
    for s in lengths:
        w = s - 1 if window < 0 else min(window, s - 1)
        total += s * (2 * w + 1) - w * (w + 1) if s > 0 else 0
    return total


def work(case: dict) -> dict:
    """Forward and backward together: every input read once, every output written once."""
    if case["op"] == "attention":
        lengths = _lengths(case)
        t, h = sum(lengths), case["heads"] * _HEAD
        # reads qkv and dout; writes out and dqkv (lse is an output of the direct call only)
        elements = 3 * h + h + h + 3 * h
        return {"bytes": 2 * t * elements + (0 if case["rotate"] else 4 * t * case["heads"]),
                # two products forward; scores, dP, dV, dK, dQ backward
                "flops": 14 * _HEAD * case["heads"] * _pairs(lengths, case["window"])}
    if case["op"] == "logprobs":
        n, b = case["rows"] * case["vocab"], _BYTES[case["type"]]
        return {"bytes": n * b * (2 if case["grad"] else 1) + case["rows"] * (20 + 12 * case["top_k"]),
                "flops": n * (10 if case["grad"] else 5)}
    n, b = case["rows"] * case["width"], _BYTES[case["type"]]
    return {"bytes": n * b * (5 if case["residual"] else 4), "flops": 2 * n}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------


def _rotation_table(positions: int, device) -> torch.Tensor:
    """bf16 [positions, 64]: the cosines of the 32 frequencies of theta 160,000, then the sines."""
    inv = 160_000.0 ** (-torch.arange(0, _HEAD, 2, dtype=torch.float64, device=device) / _HEAD)
    angle = torch.outer(torch.arange(positions, dtype=torch.float64, device=device), inv)
    return torch.cat([angle.cos(), angle.sin()], dim=1).to(torch.bfloat16)


def prepare(case: dict, seed: int) -> dict:
    dev = _device()
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=gen, device=dev) * scale

    if case["op"] == "attention":
        lengths = _lengths(case)
        total, nh = sum(lengths), case["heads"]
        qkv = normal(total, 3 * nh * _HEAD).to(torch.bfloat16)
        dout = normal(total, nh * _HEAD, scale=0.05).to(torch.bfloat16)
        cu = torch.tensor([0] + lengths, dtype=torch.int64).cumsum(0).to(torch.int32).to(dev)
        state = dict(case=case, lengths=lengths, qkv=qkv, dout=dout, cu_seqlens=cu, max_seqlen=max(lengths + [1]),
                     positions=None, table=None)
        if case["rotate"]:
            state["positions"] = torch.cat([torch.arange(s, device=dev) for s in lengths if s > 0])
            state["table"] = _rotation_table(8192, dev)
            qkv.requires_grad_(True)
        return state
    dtype = _TYPES[case["type"]]
    if case["op"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        # a trained head: most of the mass on a few tokens, the rest spread out
        logits = normal(rows, vocab, scale=2.0)
        hot = torch.randint(0, vocab, (rows, 8), generator=gen, device=dev)
        logits.scatter_add_(1, hot, normal(rows, 8, scale=3.0) + 6.0)
        if case["forbidden"]:  # a third of the vocabulary may not be produced
            closed = torch.rand(vocab, generator=gen, device=dev) < 1 / 3
            closed[0] = False
            logits.masked_fill_(closed, -math.inf)
        logits = logits.to(dtype)
        targets = torch.randint(0, vocab, (rows,), generator=gen, device=dev)
        if case["forbidden"]:
            targets = torch.where(closed[targets], torch.zeros_like(targets), targets)
        if case["grad"]:
            skip = torch.rand(rows, generator=gen, device=dev) < 0.05
            targets = torch.where(skip, torch.full_like(targets, _IGNORED), targets)
        return dict(case=case, logits=logits, targets=targets,
                    d_logprobs=torch.full((rows,), -1.0 / rows, device=dev),
                    d_entropy=torch.full((rows,), -0.01 / rows, device=dev))
    shape = (case["rows"], case["width"])
    return dict(case=case, x=normal(*shape).to(dtype), dy=normal(*shape).to(dtype),
                residual=normal(*shape).to(dtype) if case["residual"] else None,
                # seed and position of the generator, kept on the device so that a captured step can move on
                rng=torch.tensor([0x5EED_0000_0000 + seed, 7 * seed], dtype=torch.int64, device=dev))


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------


def run(state: dict):
    op = state["case"]["op"]
    if own:
        return {"attention": _own_attention, "logprobs": _own_logprobs, "dropout": _own_dropout}[op](state)
    return {"attention": _plain_attention, "logprobs": _plain_logprobs, "dropout": _plain_dropout}[op](state)


def _window(case: dict):
    return None if case["window"] < 0 else case["window"]


def _own_attention(state: dict):
    ops, case = _package(), state["case"]
    qkv, cu, longest, nh, window = state["qkv"], state["cu_seqlens"], state["max_seqlen"], case["heads"], _window(case)
    if case["rotate"]:
        out = ops.attention_varlen_qkv_train(qkv, cu, longest, nh, window, position_ids=state["positions"],
                                             table=state["table"])
        (dqkv,) = torch.autograd.grad(out, qkv, state["dout"])
        return out.detach(), dqkv
    out, lse = ops.attention_varlen_qkv_lse(qkv, cu, longest, nh, window)
    dqkv = ops.attention_varlen_qkv_backward(state["dout"], qkv, out, lse, cu, longest, nh, window)
    return out, lse, dqkv


def _own_logprobs(state: dict):
    ops, case = _package(), state["case"]
    r = ops.token_logprobs(state["logits"], state["targets"], top_k=case["top_k"], ignore_index=_IGNORED)
    outputs = [r.logprobs, r.entropy, r.lse]
    if case["top_k"]:
        outputs += [r.top_ids, r.top_logprobs]
    if case["grad"]:
        outputs.append(ops.token_logprobs_backward(state["logits"], state["targets"], r, state["d_logprobs"],
                                                   state["d_entropy"], ignore_index=_IGNORED))
    return outputs


def _own_dropout(state: dict):
    ops, p = _package(), state["case"]["p"]
    y = ops.dropout(state["x"], p, state["rng"], residual=state["residual"])
    return y, ops.dropout_backward(state["dy"], p, state["rng"])


# ---- the plain forms --------------------------------------------------------


def _rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """x [T, heads, 64], the pair (j, j + 32) turned by the angle of frequency j."""
    lo, hi = x[..., :32], x[..., 32:]
    return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], dim=-1)


def _groups(lengths: list[int], heads: int):
    """Sequences of like length together, padded to the longest of a group, so that a group's
    scores stay below 2^28 elements."""
    starts, at = [], 0
    for s in lengths:
        starts.append(at)
        at += s
    order = sorted((i for i in range(len(lengths)) if lengths[i] > 0), key=lambda i: -lengths[i])
    i = 0
    while i < len(order):
        longest = lengths[order[i]]
        count = max(1, (1 << 28) // (heads * longest * longest))
        group = [j for j in order[i:i + count] if 2 * lengths[j] > longest or longest <= 64]
        i += len(group)
        yield longest, [starts[j] for j in group], [lengths[j] for j in group]


def _plain_attention(state: dict):
    case, dev = state["case"], state["qkv"].device
    nh, window = case["heads"], case["window"]
    total = state["qkv"].shape[0]
    scale = _HEAD ** -0.5
    with torch.no_grad():
        q, k, v = state["qkv"].float().view(total, 3, nh, _HEAD).unbind(1)
        dout = state["dout"].float().view(total, nh, _HEAD)
        if case["rotate"]:
            cos, sin = state["table"].float()[state["positions"]].unsqueeze(1).split(32, dim=-1)
            q, k = _rotate(q, cos, sin), _rotate(k, cos, sin)
        out = torch.zeros(total, nh, _HEAD, device=dev)
        lse = torch.zeros(nh, total, device=dev)
        dqkv = torch.zeros(total, 3, nh, _HEAD, device=dev)
        for longest, starts, lens in _groups(state["lengths"], nh):
            step = torch.arange(longest, device=dev)
            length = torch.tensor(lens, device=dev).unsqueeze(1)
            inside = step < length                                          # [n, L]
            at = (torch.tensor(starts, device=dev).unsqueeze(1) + step).clamp_(max=total - 1)
            qb, kb, vb, gb = (x[at].transpose(1, 2) for x in (q, k, v, dout))   # [n, nh, L, 64]
            allowed = inside.unsqueeze(1) & inside.unsqueeze(2)
            if window >= 0:
                allowed = allowed & ((step.unsqueeze(0) - step.unsqueeze(1)).abs() <= window)
            allowed = allowed.unsqueeze(1)
            s = (qb @ kb.transpose(2, 3)) * scale
            s = s.masked_fill(~allowed, -math.inf)
            top = s.amax(dim=-1, keepdim=True)
            top = torch.where(top == -math.inf, torch.zeros_like(top), top)
            p = torch.exp(s - top)
            z = p.sum(dim=-1, keepdim=True)
            z = torch.where(z == 0, torch.ones_like(z), z)                  # rows of the padding
            p = p / z
            o = p @ vb
            dp = gb @ vb.transpose(2, 3)
            delta = (p * dp).sum(dim=-1, keepdim=True)
            ds = p * (dp - delta) * scale
            where = at[inside]
            out[where] = o.transpose(1, 2)[inside]
            lse[:, where] = (top + torch.log(z)).squeeze(-1).transpose(1, 2)[inside].transpose(0, 1)
            dqkv[where, 0] = (ds @ kb).transpose(1, 2)[inside]
            dqkv[where, 1] = (ds.transpose(2, 3) @ qb).transpose(1, 2)[inside]
            dqkv[where, 2] = (p.transpose(2, 3) @ gb).transpose(1, 2)[inside]
        if case["rotate"]:
            for part in (0, 1):
                dqkv[:, part] = _rotate(dqkv[:, part], cos, -sin)
        result = out.view(total, -1).to(torch.bfloat16), dqkv.view(total, -1).to(torch.bfloat16)
    return result if case["rotate"] else (result[0], lse, result[1])


def _plain_logprobs(state: dict):
    case, targets = state["case"], state["targets"]
    x = state["logits"].float()
    top = x.amax(dim=1, keepdim=True)
    e = torch.exp(x - top)
    z = e.sum(dim=1, keepdim=True)
    lse = top + torch.log(z)
    logp = x - lse
    p = e / z
    entropy = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(dim=1)
    kept = targets != _IGNORED
    at = torch.where(kept, targets, torch.zeros_like(targets)).unsqueeze(1)
    outputs = [torch.where(kept, logp.gather(1, at).squeeze(1), torch.zeros_like(entropy)), entropy, lse.squeeze(1)]
    if case["top_k"]:
        values, ids = torch.sort(x, dim=1, descending=True, stable=True)   # ties: the lowest index first
        outputs += [ids[:, :case["top_k"]].contiguous(), values[:, :case["top_k"]] - lse]
    if case["grad"]:
        g = torch.where(kept, state["d_logprobs"], torch.zeros_like(entropy)).unsqueeze(1)
        h = state["d_entropy"].unsqueeze(1)
        d = -g * p - torch.where(p > 0, h * p * (logp + entropy.unsqueeze(1)), torch.zeros_like(p))
        d.scatter_add_(1, at, g)
        outputs.append(d.to(x.dtype if case["type"] == "fp32" else _TYPES[case["type"]]))
    return outputs


def _mul32(a: torch.Tensor, m: int) -> tuple[torch.Tensor, torch.Tensor]:
    """High and low halves of the 64-bit product of 32-bit numbers held in int64."""
    low = (a & 0xFFFF) * m
    high = (a >> 16) * m + (low >> 16)
    return high >> 16, ((high & 0xFFFF) << 16) | (low & 0xFFFF)


def _plain_keep(n: int, threshold: int, rng: torch.Tensor) -> torch.Tensor:
    """Philox4x32-10 (Salmon et al., 2011): counter = position + element // 8, key = seed; each of
    the eight 16-bit fields of its 128 bits decides one element: kept if not below the threshold."""
    block = torch.arange((n + 7) // 8, dtype=torch.int64, device=rng.device) + rng[1]
    c = [block & 0xFFFFFFFF, (block >> 32) & 0xFFFFFFFF, torch.zeros_like(block), torch.zeros_like(block)]
    k0, k1 = rng[0] & 0xFFFFFFFF, (rng[0] >> 32) & 0xFFFFFFFF
    for _ in range(10):
        h0, l0 = _mul32(c[0], 0xD2511F53)
        h1, l1 = _mul32(c[2], 0xCD9E8D57)
        c = [h1 ^ c[1] ^ k0, l1, h0 ^ c[3] ^ k1, l0]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    fields = torch.stack([f for word in c for f in (word & 0xFFFF, word >> 16)], dim=1)
    return fields.view(-1)[:n] >= threshold


def _threshold(p: float) -> int:
    """The drop probability in units of 2^-16; survivors are scaled by what it makes of them."""
    return int(math.floor(p * 65536.0 + 0.5))


def _plain_dropout(state: dict):
    case, x = state["case"], state["x"]
    threshold = _threshold(case["p"])
    keep = _plain_keep(x.numel(), threshold, state["rng"]).view(x.shape)
    scale = 65536.0 / (65536 - threshold)
    outputs = []
    for value, residual in ((x, state["residual"]), (state["dy"], None)):
        y = torch.where(keep, value.float() * scale, torch.zeros((), device=x.device))
        if residual is not None:
            y = y + residual.float()
        outputs.append(y.to(x.dtype))
    return tuple(outputs)


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------


def exact(case: dict, seed: int):
    with torch.enable_grad():
        return {"attention": _exact_attention, "logprobs": _exact_logprobs, "dropout": _exact_dropout}[case["op"]](
            case, prepare(case, seed))


def _exact_attention(case: dict, state: dict):
    """Softmax attention per sequence and group of heads, its gradient by automatic differentiation."""
    nh, dev = case["heads"], state["qkv"].device
    total = state["qkv"].shape[0]
    x = state["qkv"].detach().double().view(total, 3, nh, _HEAD)
    gout = state["dout"].double().view(total, nh, _HEAD)
    out = torch.zeros(total, nh, _HEAD, dtype=torch.float64, device=dev)
    lse = torch.zeros(nh, total, dtype=torch.float64, device=dev)
    grad = torch.zeros_like(x)
    begin = 0
    for s in state["lengths"]:
        if s == 0:
            continue
        here = slice(begin, begin + s)
        far = None
        if 0 <= case["window"] < s - 1:
            index = torch.arange(s, device=dev)
            far = (index[:, None] - index[None, :]).abs() > case["window"]
        turn = None
        if state["table"] is not None:
            c = state["table"][state["positions"][here]].double()
            turn = torch.complex(c[:, :32], c[:, 32:]).unsqueeze(1)
        at_once = max(1, min(nh, (1 << 27) // (s * s)))
        for h0 in range(0, nh, at_once):
            heads = slice(h0, min(nh, h0 + at_once))
            leaf = x[here, :, heads].clone().requires_grad_(True)
            q, k, v = leaf.unbind(1)
            if turn is not None:
                q, k = (torch.view_as_real(torch.complex(z[..., :32], z[..., 32:]) * turn).transpose(-1, -2).flatten(-2)
                        for z in (q, k))
            scores = torch.einsum("ihd,jhd->hij", q, k) / 8.0
            if far is not None:
                scores = scores.masked_fill(far, -math.inf)
            z = torch.logsumexp(scores, dim=-1)
            o = torch.einsum("hij,jhd->ihd", torch.exp(scores - z.unsqueeze(-1)), v)
            (grad[here, :, heads],) = torch.autograd.grad(o, leaf, gout[here, heads])
            out[here, heads], lse[heads, here] = o.detach(), z.detach()
        begin += s
    flat = out.view(total, -1), grad.view(total, -1)
    return flat if case["rotate"] else (flat[0], lse, flat[1])


def _exact_logprobs(case: dict, state: dict):
    rows, parts = case["rows"], []
    step = max(1, (1 << 26) // case["vocab"])
    for r0 in range(0, rows, step):
        here = slice(r0, min(rows, r0 + step))
        targets = state["targets"][here]
        x = state["logits"][here].double().requires_grad_(True)
        logp = torch.log_softmax(x, dim=1)
        kept = targets != _IGNORED
        chosen = logp.gather(1, targets.clamp(min=0).unsqueeze(1)).squeeze(1)
        chosen = torch.where(kept, chosen, torch.zeros_like(chosen))
        finite = torch.where(x == -math.inf, torch.zeros_like(logp), logp)
        entropy = -(torch.exp(logp) * finite).sum(dim=1)
        part = [chosen.detach(), entropy.detach(), torch.logsumexp(x.detach(), dim=1)]
        if case["top_k"]:
            ids = torch.argsort(x.detach(), dim=1, descending=True, stable=True)[:, :case["top_k"]]
            part += [ids, logp.detach().gather(1, ids)]
        if case["grad"]:
            loss = (chosen * state["d_logprobs"][here].double() + entropy * state["d_entropy"][here].double()).sum()
            part += torch.autograd.grad(loss, x)
        parts.append(part)
    return [torch.cat(column) for column in zip(*parts)]


def _exact_dropout(case: dict, state: dict):
    n = case["rows"] * case["width"]
    seed, position = (int(v) for v in state["rng"].tolist())
    mask = np.uint64(0xFFFFFFFF)
    half = np.uint64(32)
    counter = np.arange((n + 7) // 8, dtype=np.uint64) + np.uint64(position)
    words = [counter & mask, counter >> half, np.zeros_like(counter), np.zeros_like(counter)]
    key = [seed & 0xFFFFFFFF, seed >> 32]
    for r in range(10):
        k0, k1 = ((k + r * w) & 0xFFFFFFFF for k, w in zip(key, (0x9E3779B9, 0xBB67AE85)))
        a, b = words[0] * np.uint64(0xD2511F53), words[2] * np.uint64(0xCD9E8D57)
        words = [(b >> half) ^ words[1] ^ np.uint64(k0), b & mask, (a >> half) ^ words[3] ^ np.uint64(k1), a & mask]
    fields = np.stack([w.astype(np.uint32) for w in words], axis=1).view("<u2").reshape(-1)[:n]
    threshold = _threshold(case["p"])
    keep = torch.from_numpy((fields >= threshold).reshape(case["rows"], case["width"])).to(state["x"].device)
    scale = 65536.0 / (65536 - threshold)
    y = state["x"].double() * scale * keep
    if state["residual"] is not None:
        y = y + state["residual"].double()
    return y, state["dy"].double() * scale * keep
