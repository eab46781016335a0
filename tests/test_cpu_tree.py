"""Host side of the tree operators: masks, axis maps, drafters, refusals that
need no GPU."""
import ctypes

import pytest
import torch

from synapcore_b200 import PromptLookupDrafter, rope_axis_map, tree_mask
from synapcore_b200 import _native as N


def test_tree_mask_of_two_trees():
    mask, depth = tree_mask([[-1, 0, 0, 1], [-1]])
    assert mask.tolist() == [[0b0001], [0b0011], [0b0101], [0b1011], [0b1]]
    assert depth.tolist() == [0, 1, 1, 2, 0]


@pytest.mark.parametrize("n", [1, 63, 64, 65, 128, 256])
def test_tree_mask_of_a_chain_fills_words(n):
    mask, depth = tree_mask([[i - 1 for i in range(n)]])
    assert tuple(mask.shape) == (n, -(-n // 64)) and depth.tolist() == list(range(n))
    bits = [sum((m & 0xFFFFFFFFFFFFFFFF) << (64 * k) for k, m in enumerate(row)) for row in mask.tolist()]
    assert bits == [(1 << (i + 1)) - 1 for i in range(n)]


def test_tree_mask_refuses():
    assert tree_mask([])[0].shape[0] == 0
    for bad in ([[0]], [[-1, 2, 0]], [[-2]], [[-1] * 257]):
        with pytest.raises(ValueError):
            tree_mask(bad)


def test_rope_axis_map():
    assert rope_axis_map([2, 1, 1]).tolist() == [0, 0, 1, 2]
    assert rope_axis_map([2, 1, 1], interleaved=True).tolist() == [0, 1, 2, 0]
    m = rope_axis_map([24, 20, 20], interleaved=True).tolist()
    assert m[:6] == [0, 1, 2, 0, 1, 2] and m[60:] == [0] * 4 and [m.count(a) for a in range(3)] == [24, 20, 20]
    assert rope_axis_map([64]).tolist() == [0] * 64
    for bad in ([], [0, 0], [-1, 2]):
        with pytest.raises(ValueError):
            rope_axis_map(bad)
    with pytest.raises(ValueError):
        rope_axis_map([1, 2, 1], interleaved=True)


def test_prompt_lookup_drafter_joins_branches():
    d = PromptLookupDrafter(ngram=2, length=3, branches=2)
    toks = [1, 2, 3, 4, 9, 1, 2, 3, 5, 8, 1, 2]
    out, par = d.propose(toks, 16)
    # the later occurrence first: 3 5 8; the earlier shares its 3: 3 4 9
    assert out == [3, 5, 8, 4, 9] and par == [-1, 0, 1, 0, 3]
    assert d.propose(toks, 2) == ([3, 5], [-1, 0])
    assert d.propose(toks, 0) == ([], [])
    assert d.propose([1], 4) == ([], [])
    assert d.propose([7, 7, 7, 7], 4)[0] == [7, 7]
    with pytest.raises(ValueError):
        PromptLookupDrafter(ngram=0)


def test_null_handles_are_refused():
    lib, p = N.lib(), ctypes.c_void_p()
    assert lib.sckv_tree_attn_workspace_bytes(p, 4, 8) == 0
    assert lib.sckv_verify_tree_workspace_bytes(p, 4, 100) == 0
    assert lib.sckv_append_rope_axes_workspace_bytes(p, 4) == 0
    bad = -1  # SCKV_ERR_INVALID_ARG
    assert lib.sckv_tree_attn(p, 0, p, 0, 8, 1, 1, p, p, p, 1, 1, p, 1, 1.0, p, 0, p, 0, p) == bad
    assert lib.sckv_compact_tree(p, 0, 1, 1, p, 1, p, p, p, 1, 1, p) == bad
    assert lib.sckv_verify_tree(p, p, 0, 10, 1, 10, p, p, p, 1, 1, p, p, p, p, 0, p) == bad
    assert lib.sckv_append_rope_axes(p, 0, p, 1024, p, 8, 0, 0, p, 1024, p, 1024, 0, p, p, 1e-6, p, 1.0, p, 1, 1, p, 1,
                                     1, p, p, p, 1, 1, p, 0, p) == bad
