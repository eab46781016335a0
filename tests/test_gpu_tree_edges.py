"""Calls of the tree step at its edges: pools with few pages, page scales of
rejected nodes, values past f16, infinite values, fp32 outputs, repeated calls.

Tolerances count roundings, half a step each, as in test_gpu_tree.
"""
import pytest
import torch

from stub_model import CFG, TorchStubModel, make_weights, prompts
from synapcore_b200 import ContinuousBatchScheduler, KVPool, PagedKVCache, rope_inv_freq
from synapcore_b200 import _native as N
from test_gpu_tree import gen, rope_reference, tables, values

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


# ---------------------------------------------------------- e4m3 page scales
@pytest.mark.parametrize("src", [torch.bfloat16, torch.float32])
def test_append_rope_axes_fp8_keeps_keys_past_f16(cuda_device, src):
    """A key beyond f16's range (1e6 here) enters an FP8 pool with its value, rounded once."""
    dev, g = cuda_device, gen(3, cuda_device)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    T, hq, hkv = 21, 4, 2
    bt, pages = tables([T], dev, 2)
    pool = KVPool(1, hkv, D, pages, "fp8_e4m3", device=dev)
    x = (1e6 * torch.randn(T, hq + 2 * hkv, D, generator=g, device=dev)).to(src)
    freq, axis = rope_inv_freq(1e4, D, dev), torch.zeros(64, dtype=torch.int32, device=dev)
    pos = torch.arange(T, dtype=torch.int32, device=dev)
    pool.append_rope_axes(0, x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:], pos, axis, i32([0, T]), i32([0]), bt, freq)
    pool.raise_on_status()
    k, size = rope_reference(x[:, hq:hq + hkv], None, 0.0, pos[None], axis, freq, 1.0)
    ref = [(k, size), (x[:, hq + hkv:].double(), torch.zeros_like(size))]
    now = values(pool)[0]
    for t in range(T):
        pg, sl = int(bt[0, t // 16]), t % 16
        for kv, (want, size) in enumerate(ref):
            # e4m3: half a step of the value (2^-4) or of the smallest code (2^-10 of a scale unit), 2^-23 of the
            # division; the rotation: a few fp32 steps of the row's size
            s = pool.scale_view()[0, pg, kv].double()[:, None]
            assert torch.isfinite(s).all()
            err, tol = (now[pg, kv, :, sl] - want[t]).abs(), 80 * 2.0 ** -24 * size[t]
            assert (err <= 1.001 * tol + (2.0 ** -4 + 2.0 ** -20) * want[t].abs() + s * 2.0 ** -10).all()
