"""Heads turned to their positions, paged key/value caches and attention on them, in float64 on the CPU.

TEST INFRASTRUCTURE ONLY (see the package docstring).

The reference has neither pages nor rotations of its own (it routes the wrapped model's cache tensors: src/tensor_parallel/aux_actions.py:7-15); the definitions are
closed forms, written here sequence by sequence and position by position. Pinned (tests/test_oracle_paged.py) by transformers' rotary functions, by oracle/attention.py on contiguous
caches, and by what a rotation keeps.
"""
import math

import torch


def heads(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, scaling: float = 1.0, interleaved: bool = False, norm=None, eps: float = 1e-6) -> torch.Tensor:
    """x [rows, heads, D] in float64: normed where there is a weight, then its pairs turned to the rows' positions."""
    x = x.double()
    if norm is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * norm.double()
    half = inv_freq.numel()
    angle = positions.double()[:, None] * inv_freq.double()
    return turned(x, torch.cos(angle) * scaling, torch.sin(angle) * scaling, interleaved) if half else x


def turned(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, interleaved: bool) -> torch.Tensor:
    out = x.double().clone()
    for i in range(cos.shape[-1]):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + cos.shape[-1])
        c, s = cos[:, i, None].double(), sin[:, i, None].double()
        out[..., a] = x[..., a].double() * c - x[..., b].double() * s
        out[..., b] = x[..., b].double() * c + x[..., a].double() * s
    return out


def rows_of(rows: int, lengths, starts=None, counts=None):
    """[(first row, new rows, positions)] of each sequence, lists of numbers."""
    out = []
    for b, length in enumerate(lengths):
        if starts is not None:
            out.append((starts[b], starts[b + 1] - starts[b], length))
        else:
            each = rows // len(lengths)
            out.append((b * each, each if counts is None else counts[b], length))
    return out


def gathered(pool: torch.Tensor, table, length: int) -> torch.Tensor:
    """[heads, length, D] of one sequence, zeros for pages that the pool does not have."""
    pages, H, page, D = pool.shape
    out = torch.zeros(H, length, D, dtype=torch.float64)
    for j in range(0, length, page):
        at = table[j // page]
        if 0 <= at < pages:
            n = min(page, length - j)
            out[:, j:j + n] = pool[at, :, :n].double()
    return out


def attend(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table, seqs, scale: float):
    """(out, weight) [rows, Hq, D] in float64: the attention of the new rows, and sum_j p_j |v_j|, which bounds what rounded probabilities can do. Rows of no sequence are NaN. Values that a row
    does not see are left out of its sum altogether."""
    rows, Hq, D = q.shape
    Hkv = k_pages.shape[1]
    out, weight = torch.full((rows, Hq, D), math.nan, dtype=torch.float64), torch.full((rows, Hq, D), math.nan, dtype=torch.float64)
    for b, (first, n, length) in enumerate(seqs):
        if n == 0:
            continue
        k, v = gathered(k_pages, table[b], length), gathered(v_pages, table[b], length)
        finite = bool(torch.isfinite(v).all())
        for h in range(Hq):
            kv = h * Hkv // Hq
            s = (q[first:first + n, h].double() @ k[kv].T) * scale
            unseen = torch.arange(length) > (torch.arange(n) + length - n)[:, None]
            p = torch.softmax(s.masked_fill(unseen, -math.inf), 1).masked_fill(unseen.all(1, keepdim=True), 0.0) if length else torch.zeros(n, 0, dtype=torch.float64)
            if finite:
                out[first:first + n, h], weight[first:first + n, h] = p @ v[kv], p @ v[kv].abs()
            else:
                for i in range(n):
                    seen = ~unseen[i]
                    out[first + i, h], weight[first + i, h] = p[i, seen] @ v[kv][seen], p[i, seen] @ v[kv][seen].abs()
    return out, weight
