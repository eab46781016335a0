"""Calls of the tree step at its edges: pools with few pages, page scales of
rejected nodes, values past f16, infinite values, fp32 outputs, repeated calls.

Tolerances count roundings, half a step each, as in test_gpu_tree.
"""
import pytest
import torch

from stub_model import CFG, TorchStubModel, make_weights, prompts
from synapcore_b200 import ContinuousBatchScheduler, PagedKVCache
from synapcore_b200 import _native as N

pytestmark = pytest.mark.gpu

D = 128


class Flat:
    """Drafts as many tokens as it may, all of them wrong guesses for the next one."""

    def propose(self, tokens, max_nodes):
        return [(int(tokens[-1]) + 7 + i) % 500 for i in range(max_nodes)], [-1] * max_nodes


# ------------------------------------------------------------------- pages
def test_begin_tree_without_enough_pages_changes_nothing(cuda_device):
    dev = cuda_device
    c = PagedKVCache(2, 2, D, 5, 4, 8, "fp16", device=dev)
    for s, n in (("a", 14), ("b", 33)):
        c.add_sequence(s)
        k = torch.randn(2, n, 2, D, device=dev).half()
        c.append_prefill(s, k, k)
    table, lens, state = c.block_table.clone(), list(c.lengths), c.pool.alloc_state()
    with pytest.raises(N.SCKVPoolExhausted):
        c.begin_tree([18, 17])  # a page each, of one that is free
    assert c.pool.status()[0] == N.SCKV_OK
    assert torch.equal(c.block_table, table) and c.lengths == lens and c.ctx_lens[:2].tolist() == lens
    assert c.pool.alloc_state() == state
    cu, ctx = c.begin_tree([18, 15])  # the one free page
    assert cu.tolist() == [0, 18, 33] and ctx.tolist() == lens
    none = torch.zeros(2, dtype=torch.int32, device=dev)
    c.commit_tree(none[:, None], none, [0, 0])
    assert torch.equal(c.block_table, table) and c.pool.alloc_state()["free"] == state["free"]
    # an error recorded before stays for its reader
    bad = torch.tensor([99], dtype=torch.int32, device=dev)
    c.pool.free_pages(bad)
    with pytest.raises(N.SCKVPoolExhausted):
        c.begin_tree([18, 17])
    assert c.pool.status()[0] == N.SCKV_ERR_BOUNDS
    c.pool.clear_status()


def test_scheduler_drafts_less_when_pages_are_few(cuda_device):
    """A pool that holds the plain decode but not every draft: the same tokens, no error."""
    dev = cuda_device
    model = TorchStubModel(make_weights(), dev)
    work = [(prompts()[0], 14), (prompts()[4], 30)]

    def run(drafter, pages):
        c = PagedKVCache(CFG["num_layers"], CFG["hkv"], CFG["head_dim"], pages, 4, 8, "fp16", device=dev)
        s = ContinuousBatchScheduler(model, c, max_batch_size=2, drafter=drafter)
        for i, (p, n) in enumerate(work):
            s.submit_request(f"r{i}", p, max_new_tokens=n, stop_token_ids=set())
        s.run_until_complete()
        c.check()
        assert c.n_live == 0 and c.pool.alloc_state()["allocated"] == 0
        return {r: list(q.generated_ids) for r, q in s.completed_requests.items()}, s

    plain, _ = run(None, 5)
    got, s = run(Flat(), 5)
    assert got == plain and s.drafted_tokens > 0
    assert run(Flat(), 64)[1].drafted_tokens > s.drafted_tokens
