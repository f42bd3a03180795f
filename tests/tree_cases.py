"""Trees of drafted tokens of the tests: shapes, what a row sees, attention over it in 64 bits, and page tables by hand."""
import random

import numpy as np
import torch

import paged_cases as PC


def tree(rows, seed=0, depth=8):
    """Parents of a tree of `rows` rows in any order in which parents come first, up to `depth` levels."""
    rng = random.Random(seed * 1000 + rows)
    parents, levels = [-1], [0]
    while len(parents) < rows:
        p = rng.choice([-1] * (rng.random() < 0.2) + [i for i, l in enumerate(levels) if l < depth - 1])
        parents.append(p)
        levels.append(0 if p < 0 else levels[p] + 1)
    return parents[:rows]


def chain(rows):
    return list(range(-1, rows - 1))


def depths(parents):
    out = []
    for p in parents:
        out.append(0 if p < 0 else out[p] + 1)
    return out


def seen(position, parents, row, window):
    """Positions in the pages that a row sees, in order."""
    up, at = [], row
    while at >= 0:
        up.append(position + at)
        at = parents[at]
    low = max(0, position + len(up) - window) if window else 0
    # (The rows above a row lie as far from it in the text as they are many.)
    if window:
        up = up[:window]
    return list(range(low, position)) + up[::-1]


def attention(q, keys, values, position, parents, window, softcap, scale):
    """One sequence in 64 bits, as paged_cases.attention: the outputs, the weights' sum of |v|, and the largest sum of |q k| * scale."""
    rows, heads, d = q.shape
    group = heads // keys.shape[1]
    q, keys, values = q.double(), keys.double(), values.double()
    out, spread, most = torch.empty_like(q), torch.empty_like(q), torch.empty(rows, heads, dtype=torch.float64)
    for r in range(rows):
        mine = torch.tensor(seen(position, parents, r, window))
        for h in range(heads):
            kk, vv = keys[mine, h // group], values[mine, h // group]
            s = kk @ q[r, h] * scale
            if softcap:
                s = softcap * torch.tanh(s / softcap)
            w = torch.softmax(s, 0)
            out[r, h] = w @ vv if not torch.isnan(vv).any() else (w[:, None] * vv).sum(0)
            spread[r, h] = w @ vv.abs()
            most[r, h] = ((kk * q[r, h]).abs().sum(1) * abs(scale)).max()
    return out, spread, most


def check(cache, layer, items, trees, q, got, tensors, window=0, softcap=0.0):
    at = 0
    for seq, ((position, rows), parents) in enumerate(zip(items, trees)):
        if not rows:
            continue
        n = position + rows
        keys, values = cache.rows(layer, seq, n)
        want, spread, most = attention(q[at:at + rows].cpu(), keys, values, position, parents, window, softcap, cache.d ** -0.5)
        tol = PC.tolerance(want, spread, most, cache.pages, tensors, cache.d, n)
        mine = got[at:at + rows].cpu().double()
        assert torch.equal(mine.isnan(), want.isnan()), (seq, "NaN reaches other outputs than it should")
        off = ((mine - want).abs() / tol).nan_to_num(0.0)
        assert off.max() <= 1.0, (seq, float(off.max()), float((mine - want).abs().nan_to_num().max()))
        at += rows


def flat(trees):
    return np.array([p for t in trees for p in t], np.int32)


def fit(table, pages, free, count, wanted):
    """Page tables to `wanted` pages by hand, on lists: the new count and who was refused."""
    back = [(s, c) for s, w in enumerate(wanted) for c in range(w, pages[s])]
    for s, c in reversed(back):
        free[count] = table[s][c]
        count += 1
    for s, w in enumerate(wanted):
        pages[s] = min(pages[s], w)
    asked, refused, left = 0, [], count
    for s, w in enumerate(wanted):
        more = w - pages[s]
        asked += more
        refused.append(more > 0 and asked > left)
        if refused[-1]:
            continue
        for c in range(pages[s], w):
            count -= 1
            table[s][c] = free[count]
        pages[s] = w
    return count, refused


def walk(parents, tokens, chosen):
    """The accepted path of one tree, and the choice at its end."""
    path = [0]
    while True:
        below = [r for r, p in enumerate(parents) if p == path[-1] and tokens[r] == chosen[path[-1]]]
        if not below:
            return path, chosen[path[-1]]
        path.append(below[0])
