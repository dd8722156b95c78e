"""Attention over a paged cache, block selection and eviction by weight, in 64 bits on the CPU.

No counterpart in the reference (it leaves attention to its engine): written from the definitions that
``include/triattention_hip.h`` states, one sequence and one row at a time.  A row only ever touches the
tokens it sees, so whatever lies elsewhere (garbage behind a sequence, NaN in a draft of another branch)
cannot reach it.
"""
from __future__ import annotations

import math

import torch


def rows_of(cache: torch.Tensor, table, tokens: int, scales: torch.Tensor | None = None):
    """Rows [tokens, H, D] of a sequence in float64 and which of them exist (a page outside the pool has none).
    ``cache`` [blocks, block_size, H, D] of any type, ``scales`` [blocks, block_size, H] or None."""
    nb, bs, h, d = cache.shape
    pages = torch.tensor([int(table[t // bs]) for t in range(tokens)], dtype=torch.long)
    there = (pages >= 0) & (pages < nb)
    at = (pages.clamp(0, nb - 1), torch.tensor([t % bs for t in range(tokens)], dtype=torch.long))
    raw = cache.view(torch.uint8)[at].view(cache.dtype) if cache.dtype == torch.float8_e4m3fn else cache[at]
    x = raw.double().reshape(tokens, h, d)
    if scales is not None:
        x = x * scales[at].double().reshape(tokens, h, 1)
    return x, there


def ancestors(parents) -> list:
    """The set a row sees among the new tokens: itself and its ancestors; a parent outside [0, own index) is none."""
    line = []
    for i, p in enumerate(parents):
        line.append({i} | (line[p] if 0 <= p < i else set()))
    return line


def attend(q: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, there: torch.Tensor, parents, scale: float):
    """One sequence: ``q`` [n, Hq, D], ``keys`` / ``values`` [T, H, D] float64, ``parents`` of the n new tokens (the last n of
    the T).  Returns float64 (out [n, Hq, D], lse [n, Hq], weights [T, H] summed over rows and the heads of a KV head,
    mean_abs [n, Hq, D]: the weighted mean of |v|, reach [n, Hq]: the largest sum |q_d k_d|)."""
    n, hq, d = q.shape
    t, h, _ = keys.shape
    g = hq // h
    out = torch.zeros(n, hq, d, dtype=torch.float64)
    mean_abs = torch.zeros_like(out)
    lse = torch.full((n, hq), -math.inf, dtype=torch.float64)
    reach = torch.zeros(n, hq, dtype=torch.float64)
    weights = torch.zeros(t, h, dtype=torch.float64)
    line = ancestors(parents)
    for i in range(n):
        sees = torch.tensor([j for j in range(t) if bool(there[j]) and (j < t - n or (j - (t - n)) in line[i])], dtype=torch.long)
        if sees.numel() == 0:
            continue
        for k in range(hq):
            x = q[i, k].double()
            s = (keys[sees, k // g] @ x) * scale
            z = torch.logsumexp(s, 0)
            if float(z) == -math.inf:
                continue
            p = torch.exp(s - z)
            out[i, k] = p @ values[sees, k // g]
            mean_abs[i, k] = p @ values[sees, k // g].abs()
            lse[i, k] = z
            reach[i, k] = (keys[sees, k // g].abs() @ x.abs()).max()
            weights[sees, k // g] += p
    return out, lse, weights, mean_abs, reach


def bounds_of(cache: torch.Tensor, table, tokens: int, dtype, scales: torch.Tensor | None = None):
    """Least and largest key [blocks of the sequence, H, 2, D] in ``dtype``; scaled fp8 keys are products in float32."""
    x, _ = rows_of(cache, table, tokens, scales)
    x = x.float()
    bs = cache.shape[1]
    parts = [x[i:i + bs] for i in range(0, tokens, bs)]
    return torch.stack([torch.stack([p.amin(0), p.amax(0)], 1) for p in parts]).to(dtype)


def choose_blocks(q: torch.Tensor, bounds: torch.Tensor, top: int, sinks: int, recent: int, group_max: bool) -> list:
    """Blocks of one sequence per KV head, ascending: ``q`` [Hq, D], ``bounds`` [blocks, H, 2, D]."""
    nb, h, _, d = bounds.shape
    g = q.shape[0] // h
    chosen = []
    for k in range(h):
        x = q[k * g:(k + 1) * g].double()
        s = torch.maximum(x[:, None] * bounds[:, k, 0].double(), x[:, None] * bounds[:, k, 1].double()).sum(-1)
        s = (s.amax(0) if group_max else s.mean(0)).float()
        most = torch.finfo(torch.float32).max
        s = torch.where(torch.isnan(s), most, s).clamp(max=most)
        s[:sinks] = math.inf
        s[max(0, nb - recent):] = math.inf
        order = sorted(range(nb), key=lambda j: (-float(s[j]), j))
        chosen.append(sorted(order[:top]))
    return chosen


def weight_scores(weights: torch.Tensor, layer_reduce: str | None, shared: bool, window: int, prefill: int) -> torch.Tensor:
    """Selection scores of one sequence from its weights [L, T, H]: [rows, T] float32 (rows: layers, then heads)."""
    w = weights.double()
    if layer_reduce == "mean":
        w = w.sum(0, keepdim=True) / w.shape[0]
    elif layer_reduce == "max":
        w = w.amax(0, keepdim=True)
    w = w.float().transpose(1, 2)
    if shared:
        w = w.amax(1, keepdim=True)
    w = w.reshape(-1, w.shape[-1]).clone()
    t = w.shape[1]
    w[:, max(0, t - window):] = math.inf
    w[:, :prefill] = math.inf
    return w


def keep_rows(scores: torch.Tensor, budget: int) -> list:
    """The budget largest of every row, ascending; the lowest index first among equals."""
    return [sorted(sorted(range(scores.shape[1]), key=lambda j: (-float(r[j]), j))[:budget]) for r in scores]
