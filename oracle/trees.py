"""Trees of drafted tokens, restated row by row on the CPU: the checker of tree_rows, tree_accept and paged_attention_tree.  No counterpart in
the reference, which generates a token at a time."""
from __future__ import annotations

import math
from typing import List, Sequence, Tuple

import torch


def family(parents: Sequence[int], i: int) -> List[int]:
    """Row i of a tree and its ancestors; a parent comes first, anything else is none."""
    out = [i]
    while 0 <= parents[i] < i:
        i = parents[i]
        out.append(i)
    return out


def rows(parents: Sequence[int], cu: Sequence[int], context_lens: Sequence[int], most: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """positions [T] and what every row sees of its tree, bool [T, words * 64]."""
    T, words = len(parents), (most + 63) // 64
    positions, seen = torch.zeros(T, dtype=torch.int64), torch.zeros((T, words * 64), dtype=torch.bool)
    for a, b, ctx in zip(cu, cu[1:], context_lens):
        tree = parents[a:b]
        for i in range(min(b - a, words * 64)):
            up = family(tree, i)
            positions[a + i] = ctx - (b - a) + len(up) - 1
            seen[a + i, up] = True
    return positions, seen


def pack(seen: torch.Tensor) -> torch.Tensor:
    """bool [T, words * 64] -> int64 [T, words], bit j of word i for column 64 i + j."""
    T = seen.size(0)
    return (seen.view(T, -1, 64).to(torch.int64) << torch.arange(64)).sum(-1)


def accept(tokens: Sequence[int], parents: Sequence[int], chosen: Sequence[int], cu: Sequence[int], most: int):
    """(rows kept, their numbers, the token behind them) of every sequence."""
    kept = []
    for a, b in zip(cu, cu[1:]):
        n = min(b - a, most)
        path = [0] if n > 0 else []
        while path:
            at = path[-1]
            children = [c for c in range(at + 1, n) if parents[a + c] == at and tokens[a + c] == chosen[a + at]]
            if not children:
                break
            path.append(children[0])
        kept.append((path, chosen[a + path[-1]] if path else -1))
    return kept


def attention(q: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, seen: torch.Tensor, scale: float):
    """One sequence in 64 bits: q [n, Hq, d], keys / values [ctx, Hkv, d], seen bool [n, n] (column j: the j-th of the last n keys).  Returns the
    outputs [n, Hq, d], the same with the values' magnitudes, and the largest sum of a score's magnitudes, for tolerances."""
    n, hq, d = q.shape
    ctx, hkv = keys.size(0), keys.size(1)
    group = hq // hkv
    mask = torch.ones((n, ctx), dtype=torch.bool, device=q.device)
    for j in range(n):
        if ctx - n + j >= 0:
            mask[:, ctx - n + j] = seen[:, j]
    out, size, most = torch.zeros((n, hq, d), dtype=torch.float64, device=q.device), torch.zeros((n, hq, d), dtype=torch.float64, device=q.device), 0.0
    if ctx == 0:
        return out, size, most
    for h in range(hq):
        qh, k, v = q[:, h].double(), keys[:, h // group].double(), values[:, h // group].double()
        s = (qh @ k.t().contiguous() * scale).masked_fill(~mask, -math.inf)
        most = max(most, float((qh.abs() @ torch.nan_to_num(k.abs(), 0.0, 0.0).t().contiguous()).max()) * scale)
        top = s.max(1, keepdim=True).values
        w = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
        total = w.sum(1, keepdim=True)
        w = w / torch.where(total == 0, torch.ones_like(total), total)
        # (a key that a row does not see has no say, whatever its value)
        for i in range(n) if not bool(torch.isfinite(v).all()) else [slice(None)]:
            rows = mask[i] if isinstance(i, int) else slice(None)
            out[i, h] = w[i][..., rows] @ v[rows]
            size[i, h] = w[i][..., rows] @ v[rows].abs()
    return out, size, most
