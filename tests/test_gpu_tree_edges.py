"""Calls of the tree step at its edges: pools with few pages, page scales of
rejected nodes, values past f16, infinite values, fp32 outputs, repeated calls.

Tolerances count roundings, half a step each, as in test_gpu_tree.
"""
import math

import numpy as np
import pytest
import torch

from stub_model import CFG, TorchStubModel, make_weights, prompts
from synapcore_b200 import (ContinuousBatchScheduler, KVPool, PagedKVCache, PromptLookupDrafter, rope_inv_freq,
                            tree_mask)
from synapcore_b200 import _native as N
from test_gpu_tree import KINDS, fill_pool, gen, reference, rope_reference, tables, tolerance, values

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


def _fp8_cache(dev, ctx, L=2, H=2, pages=64):
    g = gen(13, dev)
    c = PagedKVCache(L, H, D, pages, len(ctx) + 1, 12, "fp8_e4m3", device=dev)
    for i, n in enumerate(ctx):
        c.add_sequence(i)
        if n:
            c.append_prefill(i, *(torch.randn(L, n, H, D, generator=g, device=dev).half() for _ in range(2)))
    return c


def _page_bytes(c):
    """Codes and scales of every row's pages, in order of the table."""
    out = []
    for s in range(c.n_live):
        ids = torch.tensor(c.page_ids(s), dtype=torch.int64, device=c.device)
        out.append((c.pool.pool_view()[:, ids].clone(), c.pool.scale_view()[:, ids].clone()))
    return out


@pytest.mark.parametrize("size", [40.0, 1e5, math.inf, math.nan])
@pytest.mark.parametrize("rope", [False, True])
def test_fp8_rows_survive_rejected_nodes_bit_for_bit(cuda_device, size, rope):
    """Nodes of any size in a row's last page, none accepted: codes and scales of the committed pages are as before."""
    dev, g = cuda_device, gen(14, cuda_device)
    ctx, n = [14, 33, 16, 0, 47], [9, 20, 3, 5, 1]
    c = _fp8_cache(dev, ctx)
    before, free = _page_bytes(c), c.pool.alloc_state()["free"]
    freq, axis = rope_inv_freq(1e4, D, dev), torch.zeros(64, dtype=torch.int32, device=dev)
    cu, ctx_d = c.begin_tree(n)
    T = sum(n)
    for l in range(2):
        x = torch.randn(T, 8, D, generator=g, device=dev)
        x[::2] *= size
        x = x.bfloat16()
        if rope:
            pos = torch.zeros(T, dtype=torch.int32, device=dev)
            c.append_tree_rope(l, x[:, :4], x[:, 4:6], x[:, 6:], pos, axis, cu, ctx_d, freq)
        else:
            c.append_tree(l, x[:, 4:6].contiguous(), x[:, 6:].contiguous(), cu, ctx_d)
    none = torch.zeros(len(n), dtype=torch.int32, device=dev)
    c.commit_tree(none[:, None], none, [0] * len(n))
    c.check()
    assert c.lengths == ctx and c.pool.alloc_state()["free"] == free
    for (codes, scales), (b_codes, b_scales), m in zip(_page_bytes(c), before, ctx):
        assert torch.equal(scales, b_scales)
        assert torch.equal(codes.permute(0, 2, 3, 1, 4, 5).reshape(2, 2, 2, -1, D)[:, :, :, :m],
                           b_codes.permute(0, 2, 3, 1, 4, 5).reshape(2, 2, 2, -1, D)[:, :, :, :m])


@pytest.mark.parametrize("src", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rope", [False, True])
def test_fp8_commit_equals_an_append_of_the_accepted_rows(cuda_device, src, rope):
    """Codes and scales after a step are those of appending the accepted tokens alone, whatever the others held."""
    dev, g = cuda_device, gen(15, cuda_device)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    ctx, n = [14, 33, 16, 0, 47, 5], [30, 20, 3, 40, 1, 2]
    paths = [[0, 3, 4, 17, 29], [0], [0, 2], list(range(0, 40, 2)), [], [0, 1]]
    a, b = _fp8_cache(dev, ctx), _fp8_cache(dev, ctx)
    cu, ctx_d = a.begin_tree(n)
    T = sum(n)
    first = [sum(n[:r]) for r in range(len(n))]
    rows = torch.tensor([first[r] + j for r, p in enumerate(paths) for j in p], dtype=torch.int64, device=dev)
    keep = [len(p) for p in paths]
    kcu = i32([sum(keep[:r]) for r in range(len(n) + 1)])
    freq, axis = rope_inv_freq(1e4, D, dev), torch.zeros(64, dtype=torch.int32, device=dev)
    pos = torch.randint(0, 500, (T,), generator=g, device=dev, dtype=torch.int32)
    kept = torch.zeros(T, dtype=torch.bool, device=dev)
    kept[rows] = True
    b._grow_rows(0, keep)
    for l in range(2):
        x = torch.randn(T, 8, D, generator=g, device=dev)
        x[~kept] *= 300.0
        x = x.to(src)
        k, v = x[:, 4:6], x[:, 6:]
        if rope:
            a.append_tree_rope(l, x[:, :4], k, v, pos, axis, cu, ctx_d, freq)
            b.pool.append_rope_axes(l, x[rows, :4], k[rows], v[rows], pos[rows], axis, kcu, ctx_d,
                                    b.block_table[:len(n)], freq)
        else:
            a.append_tree(l, k.contiguous(), v.contiguous(), cu, ctx_d)
            b.pool.append(k[rows], v[rows], kcu, ctx_d, b.block_table[:len(n)], layer0=l)
        x.fill_(7.0)  # the caller's buffers are its own again
    P = max(keep)
    a.commit_tree(i32([p + [-1] * (P - len(p)) for p in paths]), i32(keep), keep)
    a.check()
    b.check()
    for r in range(len(n)):
        b.lengths[r] += keep[r]
    assert a.lengths == b.lengths
    for (ca, sa), (cb, sb), m in zip(_page_bytes(a), _page_bytes(b), a.lengths):
        assert torch.equal(sa, sb)
        rows = [x.permute(0, 2, 3, 1, 4, 5).reshape(2, 2, 2, -1, D)[:, :, :, :m] for x in (ca, cb)]
        assert torch.equal(*rows)


def test_fp8_commit_reports_a_bad_path(cuda_device):
    """A path out of range is reported and reads nothing out of bounds."""
    dev = cuda_device
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    for path in ([[0, 900]], [[0, -5]], [[3, 2]], [[0, 2 ** 31 - 1]]):
        c = _fp8_cache(dev, [20])
        cu, ctx = c.begin_tree([4])
        k = torch.randn(4, 2, D, device=dev).half()
        for l in range(2):
            c.append_tree(l, k, k, cu, ctx)
        c.commit_tree(i32(path), i32([2]), [2])
        assert c.pool.status()[0] == N.SCKV_ERR_BOUNDS and c.lengths == [22]
        c.pool.clear_status()


def test_fp8_step_captured_after_an_eager_call(cuda_device):
    """What a replay writes counts, not what an eager call of the same layer wrote before it."""
    dev = cuda_device
    c = _fp8_cache(dev, [20])
    cu, ctx = c.begin_tree([3])
    x = torch.randn(3, 2, D, generator=gen(18, dev), device=dev).half()
    half, buf = (x * 0.5).half(), (x * 0.5).half()
    for l in range(2):
        c.append_tree(l, half, half, cu, ctx)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for l in range(2):
            c.append_tree(l, buf, buf, cu, ctx)
    buf.copy_(x)
    graph.replay()
    path = torch.tensor([[0, 2]], dtype=torch.int32, device=dev)
    c.commit_tree(path, torch.tensor([2], dtype=torch.int32, device=dev), [2])
    c.check()
    torch.cuda.synchronize()
    for got in c.gather(0, torch.float32):
        want = x[[0, 2]].float().permute(1, 0, 2)
        # e4m3: half a step (2^-4) or of the smallest code, for the append and, moved, two growths
        assert ((got[:, :, -2:] - want).abs() <= 3 * (2.0 ** -4 * want.abs() + 6.0 / 448 * 2.0 ** -10)).all()


def test_fp8_step_refuses_fewer_rows_than_nodes(cuda_device):
    dev = cuda_device
    c = _fp8_cache(dev, [20, 7])
    before = _page_bytes(c)
    cu, ctx = c.begin_tree([4, 6])
    x = torch.randn(9, 8, D, device=dev).half()
    axis = torch.zeros(64, dtype=torch.int32, device=dev)
    with pytest.raises(ValueError):
        c.append_tree(0, x[:, 4:6].contiguous(), x[:, 6:].contiguous(), cu, ctx)
    with pytest.raises(ValueError):
        pos = torch.zeros(9, dtype=torch.int32, device=dev)
        c.append_tree_rope(0, x[:, :4], x[:, 4:6], x[:, 6:], pos, axis, cu, ctx, rope_inv_freq(1e4, D, dev))
    none = torch.zeros(2, dtype=torch.int32, device=dev)
    c.commit_tree(none[:, None], none, [0, 0])
    c.check()
    assert all(torch.equal(a, b) for x, y in zip(_page_bytes(c), before) for a, b in zip(x, y))


def test_fp8_commit_of_some_layers(cuda_device):
    """A step over the first layers only leaves the others' pages alone."""
    dev, g = cuda_device, gen(16, cuda_device)
    c = _fp8_cache(dev, [20, 7], L=3)
    before = _page_bytes(c)
    cu, ctx = c.begin_tree([4, 6])
    k, v = (torch.randn(10, 2, D, generator=g, device=dev).half() for _ in range(2))
    for l in range(2):
        c.append_tree(l, k, v, cu, ctx)
    path = torch.tensor([[0, 3], [0, 2]], dtype=torch.int32, device=dev)
    c.commit_tree(path, torch.tensor([2, 1], dtype=torch.int32, device=dev), [2, 1])
    c.check()
    assert c.lengths == [22, 8]
    for (codes, scales), (b_codes, b_scales), m in zip(_page_bytes(c), before, (20, 7)):
        rows = [x[2].permute(1, 2, 0, 3, 4).reshape(2, 2, -1, D)[:, :, :m] for x in (codes, b_codes)]
        assert torch.equal(*rows) and torch.equal(scales[2], b_scales[2])
    got = c.gather(0, torch.float32)[0]
    for at, node in ((20, 0), (21, 3)):
        for l in range(2):
            # one rounding of e4m3 (2^-4, or half the smallest code's 2^-9 of the page's scale unit)
            want = k[node].float()
            assert ((got[l, :, at] - want).abs() <= 2.0 ** -4 * want.abs() + 5.0 / 448 * 2.0 ** -10).all()


@pytest.mark.parametrize("rope", [False, True])
def test_fp8_step_of_a_padded_batch_and_of_a_capture(cuda_device, rope):
    """Rows behind the last node are nobody's; a captured append leaves its rows to the move."""
    dev, g = cuda_device, gen(17, cuda_device)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    freq, axis = rope_inv_freq(1e4, D, dev), torch.zeros(64, dtype=torch.int32, device=dev)
    x = torch.randn(9, 8, D, generator=g, device=dev).half()
    pos, path = torch.zeros(9, dtype=torch.int32, device=dev), i32([[0, 2], [1, -1]])

    def step(c, captured):
        cu, ctx = c.begin_tree([4, 2])

        def append():
            for l in range(2):
                if rope:
                    c.append_tree_rope(l, x[:, :4], x[:, 4:6], x[:, 6:], pos, axis, cu, ctx, freq)
                else:
                    c.append_tree(l, x[:, 4:6].contiguous(), x[:, 6:].contiguous(), cu, ctx)

        if captured:
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                append()
            graph.replay()
            assert not c._tree_layers
        else:
            append()
        c.commit_tree(path, i32([2, 1]), [2, 1])
        c.check()
        torch.cuda.synchronize()
        return [c.gather(s, torch.float32) for s in range(2)]

    a, b = (step(_fp8_cache(dev, [20, 5]), captured) for captured in (False, True))
    for s, rows in ((0, [0, 2]), (1, [5])):  # (positions of 0: the rotation changes nothing)
        for kv, col in ((0, slice(4, 6)), (1, slice(6, 8))):
            want = x[rows][:, col].float().permute(1, 0, 2)
            for got, n in ((a, 1), (b, 3)):
                # e4m3: half a step (2^-4), or of the smallest code, for the append and, moved, two growths
                new = got[s][kv][:, :, -len(rows):]
                assert ((new - want).abs() <= n * (2.0 ** -4 * want.abs() + 6.0 / 448 * 2.0 ** -10)).all()


# ----------------------------------------------------------------- scheduler
@pytest.mark.parametrize("drafter", ["flat", "lookup"])
def test_engine_scheduler_with_a_drafter_says_the_same(cuda_device, drafter):
    """A reference-style engine: its tokens with a drafter are those without."""
    from stub_model import StubEngine

    def run(d):
        s = ContinuousBatchScheduler(StubEngine(make_weights(), "11" * 32), 4, device=cuda_device, drafter=d)
        for i, p in enumerate(prompts()):
            s.submit_request(f"r{i}", p, max_new_tokens=9, stop_token_ids=set())
        steps = s.run_until_complete()
        s.cache.check()
        return s, steps

    plain, _ = run(None)
    s, steps = run(Flat() if drafter == "flat" else PromptLookupDrafter())
    assert {r: q.generated_ids for r, q in s.completed_requests.items()} == \
        {r: q.generated_ids for r, q in plain.completed_requests.items()}
    for rid, q in s.completed_requests.items():
        assert isinstance(q.last_logits, np.ndarray) and q.last_logits.ndim == 1
        assert int(q.last_logits.argmax()) == q.generated_ids[-1]
        assert [t for st in steps for t in st["accepted_tokens"].get(rid, [])] == q.generated_ids


def test_scheduler_picks_as_the_plain_step_where_fp32_ties(cuda_device):
    """64-bit logits that differ below fp32: the largest wins, not the first of what fp32 holds as equal."""
    dev = cuda_device

    class Close(TorchStubModel):
        def logits(self, h):
            x = super().logits(h).double()
            top = x.max(-1, keepdim=True)
            x[:, 3:4] = top.values * (1 - 1e-12 * top.values.sign())  # a hair below the largest, at a low index
            return x

    def run(d):
        m = Close(make_weights(), dev)
        c = PagedKVCache(CFG["num_layers"], CFG["hkv"], CFG["head_dim"], 64, 4, 16, "fp16", device=dev)
        s = ContinuousBatchScheduler(m, c, max_batch_size=2, drafter=d)
        s.submit_request("r", prompts()[0], max_new_tokens=6, stop_token_ids=set())
        s.run_until_complete()
        return s.completed_requests["r"].generated_ids

    plain = run(None)
    assert 3 not in plain and run(Flat()) == plain


@pytest.mark.parametrize("kind", ["bf16", "int8", "fp8_e4m3"])
def test_scheduler_with_a_drafter_on_every_pool(cuda_device, kind):
    """Runs of every pool type end with clean pages; each emitted token is the argmax of the logits given with it."""
    dev = cuda_device

    class Typed(TorchStubModel):
        def attn_in(self, layer, h, positions):
            q, k, v = super().attn_in(layer, h, positions)
            return (q.bfloat16(), k.bfloat16(), v.bfloat16()) if kind == "bf16" else (q, k, v)

    model = Typed(make_weights(), dev)
    c = PagedKVCache(CFG["num_layers"], CFG["hkv"], CFG["head_dim"], 64, 8, 16, kind, device=dev)
    s = ContinuousBatchScheduler(model, c, max_batch_size=4, drafter=PromptLookupDrafter(ngram=1, length=4))
    for i, p in enumerate(prompts()):
        s.submit_request(f"r{i}", p, max_new_tokens=9, stop_token_ids=set())
    steps = s.run_until_complete()
    c.check()
    assert c.n_live == 0 and c.pool.alloc_state()["allocated"] == 0
    for rid, q in s.completed_requests.items():
        assert len(q.generated_ids) == 9 and int(q.last_logits.argmax()) == q.generated_ids[-1]
        assert [t for st in steps for t in st["accepted_tokens"].get(rid, [])] == q.generated_ids


# ----------------------------------------------------------------- attention
@pytest.mark.parametrize("kind", ["fp16", "bf16", "int8"])
@pytest.mark.parametrize("hq,hkv,ctx,nodes", [
    (4, 2, [300], [4]),              # 8 rows: four copies in the query tile
    (8, 2, [140, 77], [13, 9]),      # 52, 36: two
    (8, 2, [500], [31]),             # 124: one
    (16, 2, [400, 30], [40, 25]),    # 320, 200: two query tiles, and 64 more rows
    (8, 1, [9000], [6]),             # one item over many SMs
])
def test_tree_attn_infinite_values_of_committed_tokens(cuda_device, kind, hq, hkv, ctx, nodes):
    """A committed V of +inf, -inf, both or NaN gives every row that, in its dim alone."""
    dev = cuda_device
    bt, pages = tables([c + n for c, n in zip(ctx, nodes)], dev, 1)
    pool = KVPool(1, hkv, D, pages, kind, device=dev)
    fill_pool(pool, gen(1, dev))

    def put(b, pos, d, x):
        page, slot = int(bt[b, pos // 16]), pos % 16
        if kind == "int8":  # code * scale past f16's range; the row's other codes are 0
            pool.pool_view()[0, page, 1, :, slot] = 0
            pool.scale_view()[0, page, 1, :, slot] = 60000.0
            pool.pool_view()[0, page, 1, :, slot, d] = 100 if x > 0 else -100
        else:
            pool.pool_view()[0, page, 1, :, slot, d] = x

    inf = math.inf
    for b, c in enumerate(ctx):
        put(b, c // 2, 5, inf)
        put(b, c - 1, 70, -inf)
        put(b, 0, 71, inf)
        put(b, 1, 71 if c > 30 else 72, -inf)
        if kind != "int8":
            put(b, 2, 100, math.nan)
            put(b, c + 1, 5, -inf)     # a node's: rows that see it have both signs
            put(b, c + 1, 120, inf)
    cu = [sum(nodes[:i]) for i in range(len(nodes) + 1)]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    mask = tree_mask([[-1] + [i // 2 for i in range(n - 1)] for n in nodes], dev)[0]
    qt = torch.bfloat16 if kind == "bf16" else torch.float16
    q = torch.randn(cu[-1], hq, D, generator=gen(2, dev), device=dev).to(qt)
    ref, absum, big = reference(values(pool), 0, q, cu, ctx, bt, mask, D ** -0.5)
    assert ref.isinf().any() and ref.isnan().any()
    for out_dtype in (qt, torch.float32):
        out = pool.tree_attn(0, q, i32(cu), i32(ctx), bt, mask, out_dtype=out_dtype).double()
        pool.raise_on_status()
        assert torch.equal(out.isnan(), ref.isnan())
        assert torch.equal(out.isinf(), ref.isinf()) and torch.equal(out[ref.isinf()], ref[ref.isinf()])
        ok = torch.isfinite(ref)
        assert ((out - ref).abs()[ok] <= tolerance(kind, qt, out_dtype, ref, absum, big)[ok]).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hq,hkv,ctx,nodes", [
    (4, 4, [0, 1, 15, 16, 17, 63, 64, 65, 130, 200], [1, 2, 1, 5, 16, 17, 0, 33, 64, 3]),
    (8, 2, [3, 77], [20, 9]),
    (7, 1, [1, 2, 5], [13, 1, 2]),
    (16, 2, [2, 33, 5], [40, 35, 7]),
    (8, 1, [6000], [16]),
])
def test_tree_attn_fp32_outputs_have_fp32_weights(cuda_device, kind, hq, hkv, ctx, nodes):
    """An fp32 output is not held to f16 weights (2^-11): on every pool its error is that of two-part weights."""
    dev = cuda_device
    bt, pages = tables([c + n for c, n in zip(ctx, nodes)], dev, 3)
    pool = KVPool(1, hkv, D, pages, kind, device=dev)
    fill_pool(pool, gen(4, dev))
    cu = [sum(nodes[:i]) for i in range(len(nodes) + 1)]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    mask = tree_mask([[-1] + [i // 2 for i in range(n - 1)] if n else [] for n in nodes], dev)[0]
    qt = torch.bfloat16 if kind == "bf16" else torch.float16
    q = torch.randn(cu[-1], hq, D, generator=gen(5, dev), device=dev).to(qt)
    scale = D ** -0.5 / 16  # small scores: the dot products' own rounding is below the weights'
    vals = values(pool)
    ref, absum, big = reference(vals, 0, q, cu, ctx, bt, mask, scale)
    out = pool.tree_attn(0, q, i32(cu), i32(ctx), bt, mask, scale=scale, out_dtype=torch.float32)
    pool.raise_on_status()
    # a weight: its two parts 2^-16 (bf16; f16 2^-22), 128-term fp32 dot products, the exponential and the sums 2^-16
    w = 2.0 ** -16 + big * 128 * 2.0 ** -24 + 2.0 ** -16
    # and half a step of the smallest f16, 2^-25 of 2^6 times the weight, of every |v| (FP8: in units of at most
    # four times the largest page scale)
    floor = torch.zeros_like(ref)
    for b, (t0, t1) in enumerate(zip(cu, cu[1:])):
        ids = bt[b, :-(-(ctx[b] + t1 - t0) // 16)].long()
        for h in range(hq):
            size = vals[0, ids, 1, h // (hq // hkv)].abs().sum((0, 1))
            if kind == "fp8_e4m3":
                s = pool.scale_view()[0, ids, 1, h // (hq // hkv)]
                size = size * 4 * float(s.max() / s.min()) if len(ids) else size
            floor[t0:t1, h] = size * 2.0 ** -31
    err, tol = (out.double() - ref).abs(), 2.0 ** -24 * ref.abs() + 2 * w * absum + floor + 1e-7
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("seqs,ctx,hq,hkv", [(40, 300, 4, 2), (15, 1251, 64, 8), (3, 5000, 8, 2)])
def test_tree_attn_repeats_itself(cuda_device, kind, seqs, ctx, hq, hkv):
    """Shares and orders are fixed: a thousand calls give the same bits, with another stream's calls beside them."""
    dev = cuda_device
    r = torch.Generator().manual_seed(seqs)
    nodes = torch.randint(1, 30, (seqs,), generator=r).tolist()
    lens = [ctx - 3 * b for b in range(seqs)]
    bt, pages = tables([c + n for c, n in zip(lens, nodes)], dev, 3)
    pools = [KVPool(1, hkv, D, pages, kind, device=dev) for _ in range(2)]
    cu = [sum(nodes[:i]) for i in range(seqs + 1)]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    mask = torch.randint(-2 ** 62, 2 ** 62, (cu[-1], 1), generator=gen(6, dev), device=dev)
    qt = torch.bfloat16 if kind == "bf16" else torch.float16
    args = []
    for i, p in enumerate(pools):
        fill_pool(p, gen(7 + i, dev))
        q = torch.randn(cu[-1], hq, D, generator=gen(9 + i, dev), device=dev).to(qt)
        args.append((0, q, i32(cu), i32(lens), bt, mask))
    first = [p.tree_attn(*a) for p, a in zip(pools, args)]
    wrong = [torch.zeros((), dtype=torch.int64, device=dev) for _ in range(2)]
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(1000):
        for p, a, f, w, s in zip(pools, args, first, wrong, streams):
            with torch.cuda.stream(s):
                w += (p.tree_attn(*a, stream=s).view(torch.int16) != f.view(torch.int16)).any()
    torch.cuda.synchronize()
    assert [int(w) for w in wrong] == [0, 0]
    for p in pools:
        p.raise_on_status()
