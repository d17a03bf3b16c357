"""Plain 64-bit restatements of what a generation step over a sliding window computes: attention with a window and sinks over the paged
cache, penalties on logits, the block bookkeeping of a step.  TEST INFRASTRUCTURE (see oracle/__init__.py): never imported by the product.
"""
from __future__ import annotations

import math
from typing import List, Optional, Sequence, Tuple

import numpy as np
import torch


def seen(pos: int, window_left: int, sinks: int) -> List[int]:
    """The keys that the token at position pos sees."""
    return [j for j in range(pos + 1) if j >= pos - window_left or j < sinks]


def window_attention(q: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor, tables: torch.Tensor, lens_q: Sequence[int],
                     ctx: Sequence[int], scale: float, window_left: int, sinks: int, alibi: Optional[torch.Tensor] = None
                     ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Row by row over the keys it sees and no others.  q [T, Hq, d], CPU tensors.  Returns (out, mass, lse) in 64 bits: mass [T, Hq, d] =
    sum p |v|, which rounding errors of the probabilities scale with; lse [T, Hq]."""
    T, hq, d = q.shape
    hkv, bs = value_cache.size(1), value_cache.size(3)
    out, mass = torch.zeros((T, hq, d), dtype=torch.float64), torch.zeros((T, hq, d), dtype=torch.float64)
    lse = torch.full((T, hq), math.inf, dtype=torch.float64)
    row = 0
    for b, (lq, lk) in enumerate(zip(lens_q, ctx)):
        for i in range(lq):
            pos = lk - lq + i
            keys = seen(pos, window_left, sinks)
            if keys:
                at = torch.tensor(keys)
                block, off = tables[b, at // bs].long(), at % bs
                k = key_cache[block, :, :, off, :].flatten(2).double().repeat_interleave(hq // hkv, 1)  # [n, Hq, d]
                v = value_cache[block, :, :, off].double().repeat_interleave(hq // hkv, 1)
                s = torch.einsum("hd,nhd->hn", q[row].double(), k) * scale
                if alibi is not None:
                    s = s + alibi.double()[:, None] * (at - pos).double()
                w = torch.exp(s - s.amax(1, keepdim=True))
                lse[row] = s.amax(1) + torch.log(w.sum(1))
                w = w / w.sum(1, keepdim=True)
                out[row] = torch.einsum("hn,nhd->hd", w, v)
                mass[row] = torch.einsum("hn,nhd->hd", w, v.abs())
            row += 1
    return out, mass, lse


def penalize(logits: torch.Tensor, said: Sequence[Sequence[int]], prompt: Sequence[int], repetition, frequency, presence,
             bias: Optional[torch.Tensor] = None, allowed: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Token by token, 64 bits.  bias [S, >= V]; allowed bool [S, V]."""
    out = logits.double().clone()
    S, V = out.shape
    for s in range(S):
        counts: dict = {}
        for i, t in enumerate(said[s]):
            if 0 <= t < V:
                counts[t] = counts.get(t, 0) + (1 if i >= prompt[s] else 0)
        for t, n in counts.items():
            x = float(out[s, t])
            x = x / float(repetition[s]) if x > 0 else x * float(repetition[s])
            out[s, t] = x - float(frequency[s]) * n - (float(presence[s]) if n > 0 else 0.0)
    if bias is not None:
        out += bias[:, :V].double()
    if allowed is not None:
        out[~allowed] = -math.inf
    return out


class StepBlocks:
    """A pool and its requests as lists, step by step (hipattn_step_blocks)."""

    def __init__(self, block_size: int, num_blocks: int, requests: int, columns: int, window_left: int = -1, sinks: int = 0):
        self.bs, self.columns, self.window, self.sinks = block_size, columns, window_left, sinks
        self.free = list(range(num_blocks))
        self.head, self.ring = 0, list(range(num_blocks))
        self.kv, self.gone = [0] * requests, [0] * requests
        self.tables = [[0] * columns for _ in range(requests)]

    def _blocks(self, tokens: int) -> int:
        return -(-tokens // self.bs)

    def live(self, r: int) -> List[int]:
        """The columns of request r that hold a block of its own."""
        sunk = self._blocks(self.sinks) if self.window >= 0 else 0
        return [c for c in range(self._blocks(self.kv[r])) if c < sunk or c >= self.gone[r]]

    def step(self, new: Sequence[int], rows: int, per_request: int = 0) -> dict:
        R, nb = len(new), len(self.ring)
        sunk = self._blocks(self.sinks) if self.window >= 0 else 0
        tail = self.head + len(self.free)
        for r in range(R):
            dead = max(self.gone[r], max(0, self.kv[r] - self.window) // self.bs) if self.window >= 0 else self.gone[r]
            for c in self.live(r):
                if new[r] < 0 or sunk <= c < dead:
                    self.free.append(self.tables[r][c])
                    self.ring[tail % nb] = self.tables[r][c]
                    tail += 1
            self.gone[r] = 0 if new[r] < 0 else dead
            if new[r] < 0:
                self.kv[r] = 0
        served, pos, slots, taken = [], [0] * rows, [-1] * rows, 0
        asked_blocks = asked_rows = used = 0
        free_blocks = len(self.free)
        cu, last = [0], []
        for r in range(R):
            n, kv = max(new[r], 0), self.kv[r]
            if n and (kv + n > self.columns * self.bs or n > (per_request or rows)):
                served.append(-2)
                n = 0
            elif n:
                need = self._blocks(kv + n) - self._blocks(kv)
                asked_blocks += need
                asked_rows += n
                if asked_blocks > free_blocks or (not per_request and asked_rows > rows):
                    served.append(-1)
                    n = 0
                else:
                    served.append(n)
            else:
                served.append(0)
            begin = r * per_request if per_request else used
            for c in range(self._blocks(kv), self._blocks(kv + n)):
                self.tables[r][c] = self.free.pop(0)
                self.head += 1
                taken += 1
            for i in range(n):
                pos[begin + i] = kv + i
                slots[begin + i] = self.tables[r][(kv + i) // self.bs] * self.bs + (kv + i) % self.bs
            self.kv[r] = kv + n
            used += n
            cu.append(used)
            last.append(begin + n - 1 if n else 0)
        return dict(state=[[k, g] for k, g in zip(self.kv, self.gone)], ends=[self.head, self.head + len(self.free)], served=served,
                    context_lens=[k if s > 0 else 0 for k, s in zip(self.kv, served)], seqlens_q=cu, logit_idxs=last, positions=pos,
                    slot_mapping=slots, totals=[used, sum(s < 0 for s in served), len(self.free), taken])


def allow_bits(allowed: torch.Tensor) -> torch.Tensor:
    """bool [S, V] -> packed u8 [S, 4 ceil(V / 32)], bit k of byte i = token 8 i + k."""
    S, V = allowed.shape
    bits = np.zeros((S, 4 * ((V + 31) // 32) * 8), dtype=np.uint8)
    bits[:, :V] = allowed.numpy()
    return torch.from_numpy(np.packbits(bits, axis=1, bitorder="little"))
