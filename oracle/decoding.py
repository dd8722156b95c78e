"""What a decoding step does around attention, in 64 bits on the CPU: new tokens' rows normalised, rotated and written into a
paged cache, rows read back, drafted tokens verified, accepted rows moved.

No counterpart in the reference (it leaves these to its engine): written from the definitions that
``include/triattention_hip.h`` states, one row and one sequence at a time.
"""
from __future__ import annotations

import math

import torch

LARGEST_FP8 = 448.0
LEAST_SCALE = 2.0 ** -126


def normed(x: torch.Tensor, weight, eps: float) -> torch.Tensor:
    """[..., D] in float64, times ``weight`` [D] over the root mean square of each row; ``weight`` None: as it is."""
    x = x.double()
    if weight is None:
        return x
    return x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps) * weight.double()


def rotated(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, freq_axes, half: bool, scale: float = 1.0) -> torch.Tensor:
    """``x`` [rows, heads, D] float64, ``positions`` [axes, rows] int64, ``freq_axes`` a list of D / 2 axes or None.  What 32 bits, in which the
    rotation is stated, cannot hold is infinite."""
    rows, heads, d = x.shape
    f = d // 2
    out = torch.empty_like(x)
    for k in range(f):
        axis = freq_axes[k] if freq_axes is not None and 0 <= freq_axes[k] < positions.shape[0] else 0
        t = positions[axis].double() * float(inv_freq[k])
        c, s = torch.cos(t)[:, None] * scale, torch.sin(t)[:, None] * scale
        i, j = (k, k + f) if half else (2 * k, 2 * k + 1)
        out[..., i] = x[..., i] * c - x[..., j] * s
        out[..., j] = x[..., j] * c + x[..., i] * s
    return torch.where(out.abs() > torch.finfo(torch.float32).max, torch.sign(out) * math.inf, out)


def row_scale(x: torch.Tensor) -> torch.Tensor:
    """Scales [...] of rows [..., D]: the largest finite magnitude / 448, at least 2^-126."""
    fine = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x))
    return (fine.amax(-1) / LARGEST_FP8).clamp(min=LEAST_SCALE)


def places(seq_lens, starts, num_rows: int, tables, block: int, num_blocks: int):
    """Per row (sequence, page, offset), None for a row that no sequence has, page -1 where the row is not cached."""
    got: list = [None] * num_rows
    for b, t in enumerate(seq_lens):
        n = starts[b + 1] - starts[b]
        for i in range(n):
            row = starts[b] + i
            if not 0 <= row < num_rows:
                continue
            at = t - n + i
            page = int(tables[b][at // block]) if at >= 0 else -1
            got[row] = (b, page if 0 <= page < num_blocks else -1, at % block if at >= 0 else 0)
    return got


# ------------------------------------------------------------------------------ verification
def draw(weights: torch.Tensor, u: float) -> int:
    """The least index whose running sum exceeds u of the whole; behind rounding or u >= 1 the last of any weight, -1 if none."""
    some = torch.nonzero(weights > 0).view(-1)
    if some.numel() == 0:
        return -1
    u = u if u > 0 else 0.0
    running = torch.cumsum(weights, 0)
    over = torch.nonzero((running > u * float(running[-1])) & (weights > 0)).view(-1)
    return int(over[0]) if over.numel() else int(some[-1])


def distribution(row: torch.Tensor, temperature: float, probs: bool) -> torch.Tensor:
    """A row's weights over their sum, float64 (all zero: nothing to draw)."""
    x = row.double()
    if probs:
        w = torch.where((x > 0) & torch.isfinite(x), x, torch.zeros_like(x))
    else:
        x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
        x = x.clamp(max=torch.finfo(torch.float32).max)
        top = x.max()
        if float(top) == -math.inf:
            return torch.zeros_like(x)
        gap = x - top
        w = torch.where(gap == 0, torch.ones_like(x), torch.where(torch.isneginf(gap), torch.zeros_like(x), torch.exp(gap / temperature)))
    total = float(w.sum())
    return w / total if total > 0 else w


def largest(row: torch.Tensor) -> int:
    """The first of the largest numbers, -1 where every one is -inf or NaN."""
    x = torch.where(torch.isnan(row.double()), torch.full_like(row.double(), -math.inf), row.double())
    x = x.clamp(max=torch.finfo(torch.float32).max)
    top = x.max()
    return -1 if float(top) == -math.inf else int(torch.nonzero(x == top).view(-1)[0])


def verify_sequence(target, tokens, uniforms, parents, temperature: float, draft=None, probs: bool = False):
    """One sequence: ``target`` [n, V], ``tokens`` [n], ``uniforms`` [n, 2], ``parents`` a list or None, ``draft`` [n, V] or None.  Returns
    (accepted rows, next token)."""
    n = target.shape[0]
    if n == 0:
        return [], -1
    greedy = not temperature > 0
    here, path = 0, [0]
    while True:
        u = float(uniforms[here, 1])
        if draft is not None and not greedy:
            p = distribution(target[here], temperature, probs)
            nxt = here + 1
            if nxt >= n:
                return path, draw(p, u)
            tok, accept_u = int(tokens[nxt]), float(uniforms[nxt, 0])
            q = draft[nxt].double()
            q = torch.where((q > 0) & torch.isfinite(q), q, torch.zeros_like(q))
            accept_u = accept_u if accept_u > 0 else 0.0
            if 0 <= tok < target.shape[1] and accept_u * float(q[tok]) < float(p[tok]):
                here = nxt
                path.append(here)
                continue
            rest = (p - q).clamp(min=0)
            return path, draw(rest if float(rest.sum()) > 0 and float(p.sum()) > 0 else p, u)
        token = largest(target[here]) if greedy else draw(distribution(target[here], temperature, probs), u)
        children = [j for j in range(here + 1, n) if (parents[j] if parents is not None else j - 1) == here]
        match = [j for j in children if int(tokens[j]) == token and token >= 0]
        if not match:
            return path, token
        here = match[0]
        path.append(here)


# -------------------------------------------------------------------------------- acceptance
def accepted_moves(rows, count: int, n: int):
    """(from, to) among a sequence's n new tokens; a list ends where it does not ascend within them."""
    moves, last = [], -1
    for j in range(min(count, n, len(rows))):
        r = int(rows[j])
        if not last < r < n:
            break
        moves.append((r, j))
        last = r
    return moves
