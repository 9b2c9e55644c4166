"""Pages for new tokens and the verification of drafted ones, on the CPU.

Sequence by sequence, as the operators are defined; none has a counterpart in the
reference, which neither pages its caches nor drafts.
"""
from __future__ import annotations

import numpy as np
import torch


def plan(lengths, new_tokens, page_table, held, free_pages, n_free, page, tokens, reset=None):
    """A dict of what paged_plan returns and leaves behind, as numpy arrays."""
    lens = [max(int(x), 0) for x in lengths]
    new = [max(int(x), 0) for x in new_tokens]
    table, free = np.array(page_table), np.array(free_pages)
    B, width = table.shape
    held = [min(max(int(x), 0), width) for x in held]
    top = min(max(int(n_free[0]), 0), len(free))
    for b in range(B):
        if reset is not None and int(reset[b]):
            for i in range(held[b]):
                if top < len(free):
                    free[top] = table[b, i]
                    top += 1
            held[b] = lens[b] = 0
    cu, rows, positions = [0], np.full(tokens, -1), np.full(tokens, -1)
    asked, room = 0, top
    for b in range(B):
        first, end = cu[-1], cu[-1] + new[b]
        cu.append(end)
        rows[first:end] = b
        if lens[b] + new[b] > width * page or end > tokens:
            continue
        need = max(0, -(-(lens[b] + new[b]) // page) - held[b]) if new[b] else 0
        asked += need
        if need and asked > room:
            continue
        for _ in range(need):
            top -= 1
            table[b, held[b]] = free[top]
            held[b] += 1
        positions[first:end] = np.arange(lens[b], lens[b] + new[b])
        lens[b] += new[b]
    return {"cu_seqlens": np.minimum(cu, tokens), "rows": rows, "positions": positions,
            "lengths": np.array(lens), "page_table": table, "held": np.array(held),
            "free_pages": free, "n_free": np.array([top])}


def probabilities(row: torch.Tensor, temperature: float) -> torch.Tensor:
    """softmax(row / temperature) fp64; certain of the first largest id where the largest is not
    finite (NaN counts as larger than all) or the temperature is 0."""
    row = row.double()
    best = int(torch.isnan(row).nonzero()[0]) if bool(row.isnan().any()) else int(
        (row == row.max()).nonzero()[0])
    if temperature <= 0 or not bool(torch.isfinite(row[best])):
        p = torch.zeros_like(row)
        p[best] = 1
        return p
    return torch.softmax((row - row[best]) / temperature, 0)


def verify(logits, draft_tokens, u, temperature=1.0, draft_probs=None, counts=None):
    """(tokens [B, K + 1], accepted [B], margin [B]): margin is the smallest distance, in
    probability, of a decision from its border."""
    B, K = draft_tokens.shape
    V = logits.shape[-1]
    tokens, accepted = torch.full((B, K + 1), -1, dtype=torch.int32), torch.zeros(B, dtype=torch.int32)
    margin = torch.ones(B, dtype=torch.float64)
    for b in range(B):
        n = K if counts is None else min(max(int(counts[b]), 0), K)
        t, q = 0, None
        while True:
            p = probabilities(logits[b, t], temperature)
            if t == n:
                rest = p
                break
            x = int(draft_tokens[b, t])
            q = torch.zeros(V, dtype=torch.float64)
            if draft_probs is not None:
                q = draft_probs[b, t].double()
            elif 0 <= x < V:
                q[x] = 1
            if 0 <= x < V:
                gap = float(p[x]) - (0.5 if temperature <= 0 else float(u[b, t]) * float(q[x]))
                if temperature > 0:
                    margin[b] = min(margin[b], abs(gap))
                if gap > 0:
                    tokens[b, t] = x
                    t += 1
                    continue
            rest = torch.where(q.isnan(), p, torch.where(p > q, p - q, 0))
            rest = rest if temperature > 0 and float(rest.sum()) > 0 else p
            break
        c = rest.cumsum(0)
        last = int(rest.nonzero()[-1])
        if temperature <= 0:
            tokens[b, t] = last
        else:
            goal = float(c[-1]) * float(u[b, K])
            tokens[b, t] = min(int(torch.searchsorted(c, goal, right=True)), last)
            borders = c[:last]
            if len(borders):
                margin[b] = min(margin[b], float((borders - goal).abs().min()))
        accepted[b] = t
    return tokens, accepted, margin
