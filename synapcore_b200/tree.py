"""Trees of drafted tokens: attention masks, and drafters that propose them.

A tree is a list of parent indices in which a node comes after its parent;
node 0, the root, is the last token already decided (its K/V is not in the
cache yet), parent -1.
"""
from __future__ import annotations

from typing import List, Optional, Protocol, Sequence, Tuple

import torch

MAX_TREE_NODES = 256  # nodes of one sequence that KVPool.tree_attn takes


def tree_mask(parents: Sequence[Sequence[int]], device: Optional[torch.device] = None
              ) -> Tuple[torch.Tensor, torch.Tensor]:
    """(mask int64 [total, W], depth int32 [total]) of several trees' nodes in
    a row, for KVPool.tree_attn and rotary positions: bit j % 64 of word
    j // 64 of a node's mask is set for the node itself and its ancestors. A
    parent of -1 starts a tree of its own (depth 0)."""
    words = max([1] + [-(-len(p) // 64) for p in parents])
    if words * 64 > MAX_TREE_NODES:
        raise ValueError(f"a tree has more than {MAX_TREE_NODES} nodes")
    rows: List[List[int]] = []
    depth: List[int] = []
    for par in parents:
        bits: List[int] = []
        deep: List[int] = []
        for i, p in enumerate(par):
            if not -1 <= p < i:
                raise ValueError(f"node {i} has parent {p}: a parent comes before its children")
            bits.append((1 << i) | (bits[p] if p >= 0 else 0))
            deep.append(deep[p] + 1 if p >= 0 else 0)
        depth.extend(deep)
        for b in bits:
            w = [(b >> (64 * k)) & 0xFFFFFFFFFFFFFFFF for k in range(words)]
            rows.append([x - (1 << 64) if x >> 63 else x for x in w])
    mask = torch.tensor(rows, dtype=torch.int64).view(-1, words)
    d = torch.tensor(depth, dtype=torch.int32)
    return (mask, d) if device is None else (mask.to(device), d.to(device))


class TreeDrafter(Protocol):
    """Proposes the tokens that a sequence may go on with."""

    def propose(self, tokens: Sequence[int], max_nodes: int) -> Tuple[List[int], List[int]]:
        """(drafted tokens, parents) after `tokens` (prompt and generated), at
        most max_nodes of them: parents[i] is the index of an earlier drafted
        token, or -1 for one that follows tokens[-1] directly."""


class PromptLookupDrafter:
    """Drafts from the sequence itself: what followed earlier occurrences of
    its last `ngram` tokens (the latest `branches` of them, `length` tokens
    each), joined into one tree by their common beginnings."""

    def __init__(self, ngram: int = 2, length: int = 8, branches: int = 3):
        if ngram < 1 or length < 1 or branches < 1:
            raise ValueError("ngram, length and branches must be positive")
        self.ngram, self.length, self.branches = int(ngram), int(length), int(branches)

    def propose(self, tokens: Sequence[int], max_nodes: int) -> Tuple[List[int], List[int]]:
        toks = [int(t) for t in tokens]
        n = self.ngram
        out: List[int] = []
        parents: List[int] = []
        child = {}  # (parent, token) -> node
        found = 0
        tail = toks[-n:]
        for at in range(len(toks) - n - 1, -1, -1):
            if found == self.branches or len(out) >= max_nodes:
                break
            if toks[at:at + n] != tail:
                continue
            found += 1
            cur = -1
            for t in toks[at + n:at + n + self.length]:
                nxt = child.get((cur, t))
                if nxt is None:
                    if len(out) >= max_nodes:
                        break
                    nxt = len(out)
                    out.append(t)
                    parents.append(cur)
                    child[(cur, t)] = nxt
                cur = nxt
        return out, parents
