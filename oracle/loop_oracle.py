"""Definitions of a decoding loop's operators in 64 bits, one sequence at a time:
the verification of drafted tokens and the page tables of a step.

No reference counterpart (the reference computes whole sequences only).
"""

from __future__ import annotations

import numpy as np


def parents_of(tree: list[int] | None, n: int) -> list[int]:
    """The token behind which each one was drafted; -1: none."""
    if tree is None:
        return list(range(-1, n - 1))
    return [max((k for k in range(i) if tree[i] >> k & 1), default=-1) for i in range(n)]


def distribution(row: np.ndarray, temperature: float) -> np.ndarray:
    """Softmax of a row of logits; NaN and -inf have no chance, infinite ones share."""
    x = np.where(np.isnan(row), -np.inf, row.astype(np.float64))
    top = x.max()
    if top == -np.inf:
        return np.zeros_like(x)
    w = (x == top).astype(np.float64) if top == np.inf else np.exp((x - top) / temperature)
    return w / w.sum()


def verify(logits: np.ndarray, tokens: list[int], uniform: list[float], *, tree: list[int] | None = None, count: int | None = None,
           draft_logits: np.ndarray | None = None, temperature: float = 1.0) -> tuple[list[int], int]:
    """The kept places of one sequence, and its next token. logits [n, vocab], draft_logits [n - 1, vocab]."""
    n, vocab = logits.shape
    count = n if count is None else min(max(count, 0), n)
    if count == 0:
        return [], -1
    parent = parents_of(tree, n)
    path = [0]
    while True:
        node = path[-1]
        children = [i for i in range(1, count) if parent[i] == node]
        if temperature == 0:
            row = np.where(np.isnan(logits[node]), -np.inf, logits[node].astype(np.float64))
            best = int(row.argmax()) if row.max() > -np.inf else -1
            down = next((i for i in children if best >= 0 and tokens[i] == best), None)
            if down is None:
                return path, best
            path.append(down)
            continue
        p = distribution(logits[node], temperature)
        q = distribution(draft_logits[node], temperature) if draft_logits is not None and children else None
        r, total, down = p.copy(), 1.0, None
        for i in children:
            t = tokens[i]
            known = 0 <= t < vocab
            chance = 1.0 if q is None else (q[t] if known else 0.0)
            if known and uniform[i] * chance * total < r[t]:
                down = i
                break
            if q is None:
                if known:
                    r[t] = 0.0
            else:
                r = np.maximum(r / total - q, 0.0)
            total = r.sum()
            if q is not None and total == 0.0:
                r, total = p.copy(), 1.0
        if down is not None:
            path.append(down)
            continue
        if r.sum() == 0.0:
            r = p
        if r.sum() == 0.0:
            return path, -1
        run = np.cumsum(r)
        past = np.nonzero((run > uniform[0] * run[-1]) & (r > 0))[0]
        return path, int(past[0]) if len(past) else int(np.nonzero(r > 0)[0][-1])


def plan(table: np.ndarray, held: list[int], lens: list[int], free: list[int], count: int, n: int, news: list[int] | None,
         page_size: int):
    """(table, held, free, count, granted, slots) after a step's pages are given out."""
    table, held, free = table.copy(), list(held), list(free)
    B, W = table.shape
    room = len(free)
    count = min(max(count, 0), room)
    told, held = held, [min(max(h, 0), W) for h in held]
    news = [n] * B if news is None else [min(max(k, 0), n) for k in news]
    have = [max(l, 0) for l in lens]
    want = [-(-(h + k) // page_size) for h, k in zip(have, news)]
    back = []
    for b in range(B):
        if want[b] <= W:
            for k in range(want[b], held[b]):
                back.append(int(table[b, k]))
                table[b, k] = -1
    for j, page in enumerate(back):
        at = count + len(back) - 1 - j
        if at < room:
            free[at] = page
    count = min(count + len(back), room)
    granted, asked, top = [], 0, count
    for b in range(B):
        lack = max(want[b] - held[b], 0) if want[b] <= W else 0
        asked += lack
        ok = want[b] <= W and (lack == 0 or asked <= top)
        granted.append(news[b] if ok else 0)
        if ok:
            for k in range(held[b], want[b]):
                count -= 1
                table[b, k] = free[count]
            held[b] = want[b]
        else:
            held[b] = told[b]  # left as it was
    slots = np.full((B, n), -1, dtype=np.int64)
    for b in range(B):
        for i in range(granted[b]):
            pos = have[b] + i
            page = int(table[b, pos // page_size])
            if page >= 0:
                slots[b, i] = page * page_size + pos % page_size
    return table, held, free, count, granted, slots
