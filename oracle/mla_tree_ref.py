"""CPU restatement of the operators on trees of drafted tokens -- test infrastructure only.

The reference has none of them.  ``plan`` follows each node's parents up to its root, ``accept`` walks down from node 0,
``attend`` scores one query at a time over the keys that it sees, in 64 bits.
"""
from __future__ import annotations

import numpy as np
import torch

PAGE = 64


def lineage(parents, i):
    """Node i's ancestors and itself, or None where the way up does not end at a root."""
    line = {i}
    while parents[i] != -1:
        if not 0 <= parents[i] < i:
            return None
        i = parents[i]
        line.add(i)
    return line


def plan(parents, lens, table, tree_lens=None):
    """(mask [B][s] of sets, positions, slots, prefix) as lists; a set is empty for no node."""
    mask, positions, slots, prefix = [], [], [], []
    for b, row in enumerate(parents):
        s = len(row)
        n = s if tree_lens is None else min(max(tree_lens[b], 0), s)
        fits = lens[b] >= n
        p = lens[b] - n if fits else 0
        prefix.append(p)
        lines = [lineage(row, i) if fits and i < n else None for i in range(s)]
        lines = [line if line is not None and all(j < n for j in line) else set() for line in lines]
        mask.append(lines)
        positions.append([p + len(line) - 1 if line else -1 for line in lines])
        at = []
        for i in range(s):
            page, r = divmod(p + i, PAGE)
            ok = fits and i < n and page < len(table[b]) and 0 <= table[b][page] < 2 ** 31 // PAGE - 1
            at.append(table[b][page] * PAGE + r if ok else -1)
        slots.append(at)
    return mask, positions, slots, prefix


def bits(line) -> int:
    """A set of nodes as the signed 64-bit word that holds its bits."""
    v = sum(1 << j for j in line)
    return v - (1 << 64) if v >= 1 << 63 else v


def accept(mask, prefix, tokens, targets):
    """(path, counts, next, keep_lens) of the plan's sets."""
    paths, counts, after, keep = [], [], [], []
    for lines, p, tok, tgt in zip(mask, prefix, tokens, targets):
        path = [0] if lines[0] == {0} else []
        while path:
            kids = [i for i, line in enumerate(lines) if line and line == lines[path[-1]] | {i} and i > path[-1] and tok[i] == tgt[path[-1]]]
            if not kids:
                break
            path.append(kids[0])
        paths.append(path + [-1] * (len(lines) - len(path)))
        counts.append(len(path))
        after.append(tgt[path[-1]] if path else -1)
        keep.append(p + len(path))
    return paths, counts, after, keep


def attend(q, kv, table, prefix, mask, scale):
    """q [B, s, H, 576], kv [pages, 64, 576] (64 bits); out [B, s, H, 512], lse [B, H, s], and per element of the output
    sum_t w_t |v_t|, and per row scale * max_t sum_d |q_d k_td| (what bounds of the rounding errors take)."""
    B, s, H, _ = q.shape
    out, lse = torch.zeros(B, s, H, 512, dtype=torch.float64), torch.full((B, H, s), -np.inf, dtype=torch.float64)
    size, reach = torch.zeros_like(out), torch.zeros_like(lse)
    for b in range(B):
        for i in range(s):
            t = torch.tensor(list(range(prefix[b])) + [prefix[b] + j for j in sorted(mask[b][i])], dtype=torch.long)
            t = t[t < PAGE * table.shape[1]]
            if not len(t):
                continue
            k = kv[table[b].long()[t // PAGE], t % PAGE]
            z = q[b, i] @ k.T * scale
            w = torch.softmax(z, -1)
            lse[b, :, i] = torch.logsumexp(z, -1)
            out[b, i] = w @ k[:, :512]
            size[b, i] = w @ k[:, :512].abs()
            reach[b, :, i] = (q[b, i].abs() @ k.abs().T).amax(-1) * scale
    return out, lse, size, reach
