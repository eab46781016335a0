"""Speculative decoding operators on the GPU against plain 64-bit forms.

Tolerances count roundings, half a step each (h = eps / 2: f16 2^-11, bf16
2^-8, f32 2^-24).
"""
import math

import pytest
import torch

from synapcore_b200 import (ContinuousBatchScheduler, KVPool, PagedAttentionLayer, PagedKVCache, PromptLookupDrafter,
                            SCKVError, rope_axis_map, rope_inv_freq, tree_mask)
from synapcore_b200 import _native as N

pytestmark = pytest.mark.gpu

D = 128
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TORCH = {"fp16": torch.float16, "bf16": torch.bfloat16}
KINDS = ["fp16", "bf16", "int8", "fp8_e4m3"]


def gen(seed, dev):
    return torch.Generator(device=dev).manual_seed(seed)


def fill_pool(pool, g):
    """Random rows of different sizes in every slot."""
    v = pool.pool_view()
    x = torch.randn(v.shape, generator=g, device=v.device)
    x *= torch.exp(0.5 * torch.randn(v.shape[:-1] + (1,), generator=g, device=v.device))
    if pool.kv_dtype in TORCH:
        v.copy_(x)
    elif pool.kv_dtype == "int8":
        s = (x.abs().amax(-1) / 127).clamp_min(1e-7)
        pool.scale_view().copy_(s)
        v.copy_(torch.clamp(torch.round(x / s[..., None]), -127, 127))
    else:
        s = x.abs().amax((-1, -2)) / 448
        pool.scale_view().copy_(s)
        v.copy_((x / s[..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8))


def values(pool):
    """[L, P, 2, H, 16, D] in 64 bits, as the cache stands for them."""
    v = pool.pool_view()
    if pool.kv_dtype == "int8":
        return (v.float() * pool.scale_view().float()[..., None]).half().double()
    if pool.kv_dtype == "fp8_e4m3":
        return v.view(torch.float8_e4m3fn).double() * pool.scale_view().double()[..., None, None]
    return v.double()


def tables(lens, dev, seed, spare=2, extra_cols=0):
    blocks = [-(-n // 16) for n in lens]
    ids = torch.randperm(sum(blocks) + spare, generator=torch.Generator().manual_seed(seed)).tolist()
    cols = max(1, max(blocks)) + extra_cols
    rows, at = [], 0
    for b in blocks:
        rows.append(ids[at:at + b] + [-1] * (cols - b))
        at += b
    return torch.tensor(rows, dtype=torch.int32, device=dev), sum(blocks) + spare


def bits_of(mask, n):
    """[T, n] truth values of an int64 [T, W] mask's first n bits."""
    j = torch.arange(n, device=mask.device)
    w = mask[:, (j // 64).clamp_max(mask.shape[1] - 1)]
    return ((w >> (j % 64)) & 1).bool() & (j < 64 * mask.shape[1])


def reference(vals, layer, q, cu, ctx, bt, mask, scale):
    """(out, sum of p |v| with a floor for the smallest p, bound of the scores' size) in 64 bits; rows of no
    sequence are NaN."""
    T, hq, _ = q.shape
    out = torch.full((T, hq, D), math.nan, dtype=torch.float64, device=q.device)
    absum = torch.zeros_like(out)
    big = 0.0
    H = vals.shape[3]
    G = hq // H
    for b in range(len(ctx)):
        t0, n = cu[b], cu[b + 1] - cu[b]
        L = ctx[b] + n
        if n == 0:
            continue
        kv = vals[layer, bt[b, :-(-L // 16)].long()].permute(1, 2, 0, 3, 4).reshape(2, H, -1, D)[:, :, :L]
        sees = torch.cat([torch.ones(n, ctx[b], dtype=torch.bool, device=q.device), bits_of(mask[t0:t0 + n], n)], 1)
        for h in range(hq):
            K, V = kv[0, h // G], kv[1, h // G]
            s = (q[t0:t0 + n, h].double() @ K.T) * scale
            s = s.masked_fill(~sees, -math.inf)
            m = s.amax(1, keepdim=True)
            p = torch.where(sees, torch.exp(s - torch.where(m.isinf() & (m < 0), torch.zeros_like(m), m)),
                            torch.zeros_like(s))
            l = p.sum(1, keepdim=True)
            w = torch.where(l > 0, p / torch.where(l > 0, l, torch.ones_like(l)), p)
            # a weight of 0 keeps what it hides out of the row
            out[t0:t0 + n, h] = torch.stack([(w[i][sees[i]] @ V[sees[i]]) if sees[i].any() else
                                             torch.zeros(D, dtype=torch.float64, device=q.device) for i in range(n)]) \
                if not torch.isfinite(V).all() else w @ V
            absum[t0:t0 + n, h] = w @ torch.nan_to_num(V, 0.0, 0.0, 0.0).abs()
            z = (q[t0:t0 + n, h].double().abs() @ torch.nan_to_num(K, 0.0, 0.0, 0.0).abs().T) * scale
            big = max(big, float(z.max()) if z.numel() else 0.0)
            # of the smallest weights: half a step of a subnormal f16 (2^-25) of 2^6 times the weight, times |v|
            absum[t0:t0 + n, h] += torch.nan_to_num(V, 0.0, 0.0, 0.0).abs().sum(0) * 2.0 ** (-31 + 11)
    return out, absum, big


def tolerance(kind, q_dtype, out_dtype, ref, absum, big):
    """|out - ref| <= h(out) |ref| + (relative error of a weight) * 2 sum p |v|:
    a weight carries the rounding of P (f16 2^-11; bf16 as hi + lo, 2^-16), of
    the 128-term fp32 dot product (128 * 2^-24 of `big`, in the exponent), of q
    where it is rounded (h of `big`), and 2^-21 of the exponential; the weighted
    sum of up to 2^14 rows adds the same order as the dot product (counted
    with the 2)."""
    hp = 2.0 ** -16 if kind == "bf16" else 2.0 ** -11
    hq = 2.0 ** -11 if q_dtype == torch.float32 else 0.0
    w = hp + big * (128 * 2.0 ** -24 + hq) + 2.0 ** -16
    # int8 pages: fp16(code * scale) is what the cache stands for, nothing more is rounded
    return HALF[out_dtype] * ref.abs() + 2 * w * absum + 1e-7


def check_attn(dev, kind, hq, hkv, ctx, nodes, seed, q_dtype=None, out_dtype=None, mask=None, layer=1, words=None,
               scale=None, poison=True):
    q_dtype = q_dtype or (torch.bfloat16 if kind == "bf16" else torch.float16)
    out_dtype = out_dtype or q_dtype
    bt, pages = tables([c + n for c, n in zip(ctx, nodes)], dev, seed)
    pool = KVPool(2, hkv, D, pages, kind, device=dev)
    g = gen(seed, dev)
    fill_pool(pool, g)
    cu = [0]
    for n in nodes:
        cu.append(cu[-1] + n)
    T = cu[-1]
    words = words or max(1, -(-max(nodes + [1]) // 64))
    if mask is None:
        mask = torch.randint(-2 ** 62, 2 ** 62, (T, words), generator=g, device=dev) * 2 + \
            torch.randint(0, 2, (T, words), generator=g, device=dev)
    q = (2 * torch.randn(T, hq, D, generator=g, device=dev)).to(q_dtype)
    scale = D ** -0.5 if scale is None else scale
    ref, absum, big = reference(values(pool), layer, q, cu, ctx, bt, mask, scale)
    if poison:  # slots that hold no token may hold anything
        used = torch.zeros(pages, 16, dtype=torch.bool, device=dev)
        for b, (c, n) in enumerate(zip(ctx, nodes)):
            pos = torch.arange(c + n, device=dev)
            used[bt[b, pos // 16].long(), pos % 16] = True
        view = pool.pool_view().permute(1, 4, 0, 2, 3, 5)
        if kind in TORCH:
            view[~used] = math.nan
        elif kind == "fp8_e4m3":
            view[~used] = 0x7F
        else:
            pool.scale_view().permute(1, 4, 0, 2, 3)[~used] = math.inf
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    out = pool.tree_attn(layer, q, i32(cu), i32(ctx), bt, mask, scale=scale, out_dtype=out_dtype)
    pool.raise_on_status()
    assert out.dtype == out_dtype and tuple(out.shape) == (T, hq, D)
    assert torch.isfinite(out).all()
    err = (out.double() - ref).abs()
    tol = tolerance(kind, q_dtype, out_dtype, ref, absum, big)
    assert (err <= tol).all(), (float((err / tol).max()), float(err.max()))
    return out


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hq,hkv", [(4, 4), (8, 2), (7, 1), (16, 2), (3, 1)])
def test_tree_attn_small_lengths(cuda_device, kind, hq, hkv):
    ctx = [0, 1, 15, 16, 17, 63, 64, 65, 130, 200]
    nodes = [1, 2, 1, 5, 16, 17, 0, 33, 64, 3]
    check_attn(cuda_device, kind, hq, hkv, ctx, nodes, seed=hq * 10 + hkv)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hq,hkv,ctx,nodes", [
    (8, 8, [1500], [9]),
    (8, 1, [4097, 3], [32, 64]),
    (12, 2, [1023, 1024, 1025, 700], [21, 22, 43, 1]),
    (32, 8, [2000] * 3, [16, 12, 31]),
])
def test_tree_attn_longer(cuda_device, kind, hq, hkv, ctx, nodes):
    check_attn(cuda_device, kind, hq, hkv, ctx, nodes, seed=len(ctx) + hq)


@pytest.mark.parametrize("kind", ["fp16", "fp8_e4m3"])
@pytest.mark.parametrize("nodes", [65, 130, 200, 256])
def test_tree_attn_many_nodes(cuda_device, kind, nodes):
    check_attn(cuda_device, kind, 8, 2, [100, 61], [nodes, nodes - 64], seed=nodes, words=4)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("seqs", [40, 333])
def test_tree_attn_many_sequences(cuda_device, kind, seqs):
    """More items than SMs, of every length."""
    r = torch.Generator().manual_seed(seqs)
    ctx = torch.randint(0, 300, (seqs,), generator=r).tolist()
    nodes = torch.randint(0, 20, (seqs,), generator=r).tolist()
    check_attn(cuda_device, kind, 4, 2, ctx, nodes, seed=seqs)


@pytest.mark.parametrize("kind,q_dtype,out_dtype", [
    ("fp16", torch.float32, torch.float32), ("fp16", torch.bfloat16, torch.float16),
    ("int8", torch.float32, torch.bfloat16), ("fp8_e4m3", torch.bfloat16, torch.float32),
    ("bf16", torch.bfloat16, torch.float32)])
def test_tree_attn_types(cuda_device, kind, q_dtype, out_dtype):
    check_attn(cuda_device, kind, 8, 2, [300, 77], [20, 9], seed=5, q_dtype=q_dtype, out_dtype=out_dtype)


@pytest.mark.parametrize("kind", KINDS)
def test_tree_attn_rows_that_see_nothing_are_zero(cuda_device, kind):
    mask = torch.zeros(9, 1, dtype=torch.int64, device=cuda_device)
    mask[3] = 0b1000
    mask[8] = -1  # bits past the sequence's nodes are ignored
    out = check_attn(cuda_device, kind, 8, 2, [0, 40], [5, 4], seed=2, mask=mask)
    assert (out[[0, 1, 2, 4]] == 0).all() and (out[3] != 0).any()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("scale", [1e-4, 1.0])
def test_tree_attn_scales(cuda_device, kind, scale):
    """Near-uniform weights, and scores of several hundred."""
    check_attn(cuda_device, kind, 4, 1, [500, 31], [13, 40], seed=3, scale=scale)


def test_tree_attn_rising_scores(cuda_device):
    """The running maximum moves at every tile."""
    dev = cuda_device
    for kind in KINDS:
        ctx, nodes = [700], [10]
        bt, pages = tables([710], dev, 1)
        pool = KVPool(1, 1, D, pages, kind, device=dev)
        g = gen(4, dev)
        k = torch.randn(1, 710, 1, D, generator=g, device=dev) * 0.1 + \
            torch.linspace(0, 4, 710, device=dev)[None, :, None, None]
        v = torch.randn(1, 710, 1, D, generator=g, device=dev) * torch.linspace(0.01, 30, 710, device=dev)[:, None, None]
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
        pool.append(k, v, i32([0, 710]), i32([0]), bt)
        q = torch.ones(10, 4, D, device=dev).to(torch.bfloat16 if kind == "bf16" else torch.float16)
        mask = tree_mask([[i - 1 for i in range(10)]], dev)[0]
        ref, absum, big = reference(values(pool), 0, q, [0, 10], ctx, bt, mask, D ** -0.5)
        out = pool.tree_attn(0, q, i32([0, 10]), i32(ctx), bt, mask, out_dtype=torch.float32)
        err = (out.double() - ref).abs()
        assert (err <= tolerance(kind, q.dtype, torch.float32, ref, absum, big)).all(), kind


@pytest.mark.parametrize("kind", ["fp16", "bf16", "fp8_e4m3"])
@pytest.mark.parametrize("which,bad", [("v", math.inf), ("v", math.nan), ("k", math.nan), ("k", math.inf)])
def test_tree_attn_hidden_nodes_may_hold_anything(cuda_device, kind, which, bad):
    """A node whose K or V is not finite reaches the rows that see it, and no other."""
    dev = cuda_device
    if kind == "fp8_e4m3" and bad == math.inf:
        pytest.skip("e4m3 has no infinity")
    ctx, nodes = [70], [12]
    bt, pages = tables([82], dev, 1)
    pool = KVPool(1, 2, D, pages, kind, device=dev)
    fill_pool(pool, gen(1, dev))
    pos = 70 + 5
    row = pool.pool_view()[0, int(bt[0, pos // 16]), 0 if which == "k" else 1, :, pos % 16]
    row[:, 37] = 0x7F if kind == "fp8_e4m3" else bad
    parents = [-1, 0, 0, 1, 2, 0, 5, 5, 3, 6, 1, 4]
    mask = tree_mask([parents], dev)[0]
    q = torch.randn(12, 4, D, generator=gen(2, dev), device=dev).to(torch.bfloat16 if kind == "bf16" else torch.float16)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    out = pool.tree_attn(0, q, i32([0, 12]), i32(ctx), bt, mask)
    sees = bits_of(mask, 12)[:, 5]
    ref, absum, big = reference(values(pool), 0, q, [0, 12], ctx, bt, mask, D ** -0.5)
    assert torch.isfinite(out[~sees]).all()
    err = (out.double() - ref).abs()[~sees]
    assert (err <= tolerance(kind, q.dtype, q.dtype, ref, absum, big)[~sees]).all()
    # (a score of -inf, from an infinite key, has weight 0: those rows stay finite)
    assert torch.equal(torch.isfinite(out[sees][..., 37]), torch.isfinite(ref[sees][..., 37]))
    if (which, bad) != ("k", math.inf):
        assert not torch.isfinite(out[sees][..., 37]).any()
    if which == "v":  # the other dims of those rows are as they should be
        keep = [d for d in range(D) if d != 37]
        err = (out.double() - ref).abs()[sees][..., keep]
        assert (err <= tolerance(kind, q.dtype, q.dtype, ref, absum, big)[sees][..., keep]).all()


def test_tree_attn_leaves_foreign_rows_and_reports(cuda_device):
    dev = cuda_device
    bt, pages = tables([60, 60, 60], dev, 1)
    pool = KVPool(1, 2, D, pages, "fp16", device=dev)
    fill_pool(pool, gen(1, dev))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    q = torch.randn(12, 4, D, device=dev).half()
    mask = torch.full((12, 1), -1, dtype=torch.int64, device=dev)
    # a context past the table, and a negative one: reported, their rows left; rows 10, 11 are nobody's
    out = torch.full((12, 4, D), 7.0, device=dev, dtype=torch.float16)
    pool.tree_attn(0, q, i32([0, 4, 8, 10]), i32([10, 100, -1]), bt, mask, out=out)
    code, _, kernel, count = pool.status()
    assert code == N.SCKV_ERR_BOUNDS and kernel == 18 and count >= 2
    pool.clear_status()
    assert (out[4:] == 7).all() and (out[:4] != 7).any()
    ref = pool.tree_attn(0, q[:4], i32([0, 4]), i32([10]), bt, mask[:4])
    assert torch.equal(out[:4], ref)
    # a page id that is none
    bad = bt.clone()
    bad[0, 0] = pages + 5
    pool.tree_attn(0, q[:4], i32([0, 4]), i32([10]), bad, mask[:4])
    assert pool.status()[0] == N.SCKV_ERR_BOUNDS
    pool.clear_status()
    # more nodes than the mask has bits
    q2, m2 = torch.randn(65, 4, D, device=dev).half(), torch.zeros(65, 1, dtype=torch.int64, device=dev)
    pool.tree_attn(0, q2, i32([0, 65]), i32([0]), torch.cat([bt[:1], bt[1:2]], 1), m2)
    assert pool.status()[0] == N.SCKV_ERR_BOUNDS
    pool.clear_status()


def test_tree_attn_refusals(cuda_device):
    dev = cuda_device
    bt, pages = tables([40], dev, 1)
    pool = KVPool(1, 2, D, pages, "bf16", device=dev)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    q = torch.randn(4, 4, D, device=dev).bfloat16()
    mask = torch.ones(4, 1, dtype=torch.int64, device=dev)
    ok = (0, q, i32([0, 4]), i32([10]), bt, mask)
    pool.tree_attn(*ok)
    with pytest.raises(SCKVError):
        pool.tree_attn(0, q.half(), *ok[2:])
    for bad in [dict(i=1, v=q[:, :3]), dict(i=1, v=q[..., :64]), dict(i=0, v=1), dict(i=5, v=mask[:3]),
                dict(i=5, v=torch.ones(4, 5, dtype=torch.int64, device=dev)), dict(i=3, v=i32([])),
                dict(i=4, v=bt[:0]), dict(i=2, v=i32([0, 4]).cpu())]:
        args = list(ok)
        args[bad["i"]] = bad["v"]
        with pytest.raises(ValueError):
            pool.tree_attn(*args)
    for i, v in [(2, torch.tensor([0, 4], device=dev)), (5, mask.int())]:
        args = list(ok)
        args[i] = v
        with pytest.raises(TypeError):
            pool.tree_attn(*args)
    for kw in [dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(max_blocks=99),
               dict(out=torch.empty(3, 4, D, device=dev)),
               dict(workspace=torch.empty(0, dtype=torch.uint8, device=dev))]:
        if "workspace" in kw and pool.tree_attn_workspace_bytes(4, 4) == 0:
            continue
        with pytest.raises(ValueError):
            pool.tree_attn(*ok, **kw)
    assert pool.tree_attn(0, q[:0], i32([0]), i32([]), bt[:0], mask[:0]).shape[0] == 0
    small = KVPool(1, 2, 64, 4, "fp16", device=dev)
    with pytest.raises(SCKVError) as e:
        small.tree_attn(0, torch.randn(4, 4, 64, device=dev).half(), *ok[2:])
    assert e.value.code == N.SCKV_ERR_UNSUPPORTED


def test_tree_attn_streams_and_graph(cuda_device):
    """Two calls in flight on two streams, and captured calls replayed on new inputs."""
    dev = cuda_device
    bt, pages = tables([900, 333], dev, 3)
    pool = KVPool(1, 2, D, pages, "fp16", device=dev)
    fill_pool(pool, gen(1, dev))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    cu, ctx = i32([0, 10, 17]), i32([880, 300])
    mask = tree_mask([[-1] + list(range(9)), [-1, 0, 0, 0, 1, 1, 2]], dev)[0]
    qs = [torch.randn(17, 8, D, generator=gen(i, dev), device=dev).half() for i in range(6)]
    want = [pool.tree_attn(0, q, cu, ctx, bt, mask) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    got = [pool.tree_attn(0, q, cu, ctx, bt, mask, stream=streams[i % 2]) for i, q in enumerate(qs)]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    q = qs[0].clone()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(pool.tree_attn(0, q, cu, ctx, bt, mask))
        graphs.append(g)
    for i in (3, 4):
        q.copy_(qs[i])
        for g, o in zip(graphs, outs):
            o.zero_()
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, want[i]) for o in outs)


def test_tree_attn_chain_equals_prefill(cuda_device):
    """A chain is a causal prompt: the two kernels agree within their roundings."""
    dev = cuda_device
    for kind in KINDS:
        bt, pages = tables([250], dev, 3)
        pool = KVPool(1, 2, D, pages, kind, device=dev)
        fill_pool(pool, gen(1, dev))
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
        q = torch.randn(40, 8, D, generator=gen(2, dev), device=dev)
        q = q.to(torch.bfloat16 if kind == "bf16" else torch.float16)
        mask = tree_mask([[i - 1 for i in range(40)]], dev)[0]
        ref, absum, big = reference(values(pool), 0, q, [0, 40], [200], bt, mask, D ** -0.5)
        a = pool.tree_attn(0, q, i32([0, 40]), i32([200]), bt, mask, out_dtype=torch.float32)
        b = pool.prefill_attn(0, q, i32([0, 40]), i32([200]), bt, out_dtype=torch.float32)
        # FP8 pages: the prompt kernel rounds code * scale to f16 (2^-11 of each value and score)
        more = (2.0 ** -11 * (1 + big) * 2 * absum) if kind == "fp8_e4m3" else 0.0
        # ... and its P is the weight itself in f16: half a subnormal step, 2^-25, of every |v|
        more = more + values(pool)[0, :, 1].abs().sum((0, 2)).repeat_interleave(4, 0)[None] * 2.0 ** -25
        tol = tolerance(kind, q.dtype, torch.float32, ref, absum, big)
        worst = float(((a.double() - b.double()).abs() / (2 * tol + more)).max())
        assert worst <= 1, (kind, worst)


# ------------------------------------------------------------------ rope
def rope_reference(x, w, eps, pos, axis, freq, scaling):
    x = x.double()
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    a = (pos.double()[axis.long()].T / scaling * freq.double())[:, None]
    x1, x2 = x[..., :D // 2], x[..., D // 2:]
    return torch.cat([x1 * a.cos() - x2 * a.sin(), x2 * a.cos() + x1 * a.sin()], -1), \
        torch.cat([x1.abs() + x2.abs()] * 2, -1)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hq,hkv,lens,axes,norm,src", [
    (4, 4, [1], 1, False, torch.float16),
    (7, 1, [5, 0, 18], 3, True, torch.bfloat16),
    (32, 8, [33, 1, 2], 2, True, torch.float32),
    (40, 2, [700, 500], 3, False, torch.float16),
])
def test_append_rope_axes(cuda_device, kind, hq, hkv, lens, axes, norm, src):
    dev, g = cuda_device, gen(7, cuda_device)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    start = [3 + 7 * b for b in range(len(lens))]
    bt, pages = tables([s + n for s, n in zip(start, lens)], dev, 2)
    T = sum(lens)
    cu = [sum(lens[:b]) for b in range(len(lens) + 1)]
    pool = KVPool(2, hkv, D, pages, kind, device=dev)
    fill_pool(pool, g)
    before = values(pool)
    x = torch.randn(T + 3, hq + 2 * hkv, D, generator=g, device=dev).to(src)
    q, k, v = x[:T, :hq], x[:T, hq:hq + hkv], x[:T, hq + hkv:]
    w = [(1 + 0.2 * torch.randn(D, generator=g, device=dev)).half() if norm else None for _ in range(2)]
    pos = torch.randint(0, 2 ** 31 - 1, (axes, T), generator=g, device=dev, dtype=torch.int32) >> 12
    pos[:, 0] = 0
    pos[-1, -1] = 2 ** 31 - 1
    axis = rope_axis_map({1: [64], 2: [40, 24], 3: [24, 20, 20]}[axes], interleaved=axes == 3, device=dev)
    freq = rope_inv_freq(1e6, D, dev)
    out_dt = torch.float32 if src == torch.float32 else src
    got = pool.append_rope_axes(1, q, k, v, pos, axis, i32(cu), i32(start), bt, freq, rope_scaling=2.0,
                                q_norm_w=w[0], k_norm_w=w[1], eps=1e-5)
    pool.raise_on_status()
    # roundings: the norm's factor and products, the angle's sin and cos and the two products, a few fp32 steps
    # each of the row's size (128-term sum of squares: 64 steps), then the output type's
    for kindx, y, wx in (("q", q, w[0]), ("k", k, w[1])):
        ref, size = rope_reference(y, wx, 1e-5, pos, axis, freq, 2.0)
        tol = size * 80 * 2.0 ** -24
        if kindx == "q":
            assert got.dtype == out_dt
            assert ((got.double() - ref).abs() <= tol + HALF[out_dt] * (ref.abs() + tol)).all()
        else:
            kref, ktol = ref, tol
    now = values(pool)
    for b in range(len(lens)):
        for t in range(cu[b], cu[b + 1]):
            p = start[b] + t - cu[b]
            pg, sl = int(bt[b, p // 16]), p % 16
            for kv, (ref, tol) in enumerate(((kref[t], ktol[t]), (v[t].double(), torch.zeros_like(ktol[t])))):
                cell = now[1, pg, kv, :, sl]
                if kind in TORCH:
                    h = HALF[TORCH[kind]]
                    assert ((cell - ref).abs() <= tol + h * (ref.abs() + tol) + 1e-7).all()
                elif kind == "int8":
                    # half a code, the scale's fp16 rounding (127 codes of it), the fp16 source and result
                    s = pool.scale_view()[1, pg, kv, :, sl].double()[:, None]
                    assert ((cell - ref).abs() <= tol + s * 0.51 + 4 * 2.0 ** -11 * ref.abs() + s * 127 * 2.0 ** -11).all()
                else:
                    # e4m3: half a step of the value (2^-4) or of the smallest code (2^-10 of 1 scale unit),
                    # several times where the page's scale grew (twice at most for these pages' few calls)
                    s = pool.scale_view()[1, pg, kv].double()[:, None]
                    assert ((cell - ref).abs() <= tol + 2.0 ** -11 * ref.abs() + 2.0 ** -4 * ref.abs() + s * 2.0 ** -10).all()
    # nothing else in the pool changed (FP8: rows of a touched page may be re-encoded)
    if kind != "fp8_e4m3":
        same = torch.ones(before.shape[1], 16, dtype=torch.bool, device=dev)
        for b in range(len(lens)):
            p = torch.arange(start[b], start[b] + lens[b], device=dev)
            same[bt[b, p // 16].long(), p % 16] = False
        assert torch.equal(before.permute(1, 4, 0, 2, 3, 5)[same], now.permute(1, 4, 0, 2, 3, 5)[same])
    assert torch.equal(before[0], now[0])


def test_append_rope_axes_equals_append_rope_at_near_positions(cuda_device):
    """One axis with the slots' own positions is append_rope (whose angle is formed in fp32: near positions only)."""
    dev, g = cuda_device, gen(8, cuda_device)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    bt, pages = tables([20], dev, 2)
    x = torch.randn(12, 12, D, generator=g, device=dev).half()
    w = (1 + 0.2 * torch.randn(D, generator=g, device=dev)).half()
    freq = rope_inv_freq(10000.0, D, dev)
    a, b = (KVPool(1, 2, D, pages, "fp16", device=dev) for _ in range(2))
    qa = a.append_rope(0, x[:, :8], x[:, 8:10], x[:, 10:], i32([0, 12]), i32([8]), bt, freq, q_norm_w=w, k_norm_w=w)
    pos = torch.arange(8, 20, dtype=torch.int32, device=dev)
    qb = b.append_rope_axes(0, x[:, :8], x[:, 8:10], x[:, 10:], pos, torch.zeros(64, dtype=torch.int32, device=dev),
                            i32([0, 12]), i32([8]), bt, freq, q_norm_w=w, k_norm_w=w)
    # the two differ by an fp32 angle (19 * 2^-24 at most) and a few fp32 steps before the same f16 rounding: one step
    for u, v in ((qa, qb), (a.pool_view(), b.pool_view())):
        u, v = u.double(), v.double()
        assert ((u - v).abs() <= 2.0 ** -10 * u.abs() + 1e-5).all()


def test_append_rope_axes_refusals_and_reports(cuda_device):
    dev = cuda_device
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    bt, pages = tables([40], dev, 2)
    pool = KVPool(1, 2, D, pages, "fp16", device=dev)
    x = torch.randn(4, 8, D, device=dev).half()
    freq = rope_inv_freq(10000.0, D, dev)
    axis = torch.zeros(64, dtype=torch.int32, device=dev)
    ok = dict(layer=0, q=x[:, :4], k_new=x[:, 4:6], v_new=x[:, 6:], positions=i32([[0, 1, 2, 3]]), axis_map=axis,
              cu_tokens=i32([0, 4]), start_pos=i32([0]), block_table=bt, inv_freq=freq)
    pool.append_rope_axes(**ok)
    for bad in [dict(layer=1), dict(k_new=x[:, 4:7]), dict(q=x[:3, :4]), dict(positions=i32([[0, 1]])),
                dict(axis_map=axis[:63]), dict(inv_freq=freq[:60]), dict(start_pos=i32([])), dict(max_blocks=50),
                dict(q_norm_w=torch.ones(4 * D, dtype=torch.float16, device=dev)),
                dict(q_out=torch.empty(4, 3, D, device=dev))]:
        with pytest.raises(ValueError):
            pool.append_rope_axes(**{**ok, **bad})
    for bad in [dict(positions=torch.zeros(1, 4, dtype=torch.int64, device=dev)), dict(v_new=x[:, 6:].float()),
                dict(q_norm_w=torch.ones(D, device=dev)), dict(q=x[:, :4].double())]:
        with pytest.raises(TypeError):
            pool.append_rope_axes(**{**ok, **bad})
    with pytest.raises(SCKVError):
        pool.append_rope_axes(**ok, rope_scaling=0.0)
    pool.raise_on_status()
    for bad in [dict(axis_map=axis + 1), dict(start_pos=i32([pages * 16])), dict(start_pos=i32([-3])),
                dict(block_table=torch.full_like(bt, -1))]:
        pool.append_rope_axes(**{**ok, **bad})
        assert pool.status()[0] == N.SCKV_ERR_BOUNDS, bad
        pool.clear_status()
    # tokens of no sequence are skipped
    out = torch.full((4, 4, D), 5.0, dtype=torch.float16, device=dev)
    keep = pool.pool_view().clone()
    pool.append_rope_axes(**{**ok, "cu_tokens": i32([1, 2]), "start_pos": i32([30])}, q_out=out)
    assert (out[[0, 2, 3]] == 5).all() and (out[1] != 5).any()
    assert int((keep != pool.pool_view()).any(-1).sum()) <= 4


# --------------------------------------------------------------- compact
@pytest.mark.parametrize("kind", ["fp16", "bf16", "int8"])
@pytest.mark.parametrize("d", [64, 128])
def test_compact_tree_moves_rows(cuda_device, kind, d):
    dev, g = cuda_device, gen(3, cuda_device)
    ctx = [0, 5, 16, 31, 100, 7, 40]
    nodes = [64, 20, 200, 40, 1, 9, 17]
    paths = [[0, 1, 2], [0, 3, 4, 19], list(range(0, 200, 3)), [1, 2, 39], [0], [], list(range(17))]
    bt, pages = tables([c + n for c, n in zip(ctx, nodes)], dev, 2)
    pool = KVPool(3, 2, d, pages, kind, device=dev)
    fill_pool(pool, g)
    want, ws = pool.pool_view().clone(), pool.scale_view().clone() if kind == "int8" else None
    P = max(len(p) for p in paths)
    for b, path in enumerate(paths):
        src = want.clone(), ws.clone() if ws is not None else None
        for j, i in enumerate(path):
            s, t = ctx[b] + i, ctx[b] + j
            sp, tp = int(bt[b, s // 16]), int(bt[b, t // 16])
            want[1:, tp, :, :, t % 16] = src[0][1:, sp, :, :, s % 16]
            if ws is not None:
                ws[1:, tp, :, :, t % 16] = src[1][1:, sp, :, :, s % 16]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    pool.compact_tree(bt, i32(ctx), i32([p + [-1] * (P - len(p)) for p in paths]), i32([len(p) for p in paths]),
                      layer0=1)
    pool.raise_on_status()
    assert torch.equal(pool.pool_view().view(torch.uint8), want.view(torch.uint8))
    if ws is not None:
        assert torch.equal(pool.scale_view(), ws)


def test_compact_tree_fp8(cuda_device):
    """Rows of other pages enter as an append of their values would."""
    dev, g = cuda_device, gen(3, cuda_device)
    ctx, paths = [5, 14, 0], [[0, 7, 20, 30, 31, 45], [1, 2, 40], list(range(1, 60, 3))]
    bt, pages = tables([70, 70, 70], dev, 2)
    pool = KVPool(2, 2, D, pages, "fp8_e4m3", device=dev)
    fill_pool(pool, g)
    pool.scale_view()[:, :, 1] *= torch.exp(torch.randn(2, pages, 2, generator=g, device=dev))
    codes, scales = pool.pool_view().clone(), pool.scale_view().clone()
    enc = lambda x: x.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)  # noqa: E731
    dec = lambda c: c.view(torch.float8_e4m3fn).float()  # noqa: E731
    for b, path in enumerate(paths):
        for blk in range((ctx[b] + len(path) - 1) // 16 + 1):
            dp = int(bt[b, blk])
            rows = {}
            for j, i in enumerate(path):
                if i != j and (ctx[b] + j) // 16 == blk:
                    s = ctx[b] + i
                    rows[(ctx[b] + j) % 16] = (int(bt[b, s // 16]), s % 16)
            if not rows:
                continue
            s_new = scales[:, dp].clone()
            for sp, sl in rows.values():
                if sp != dp:
                    top = (dec(codes[:, sp, :, :, sl]) * scales[:, sp][..., None]).abs().amax(-1)
                    s_new = torch.maximum(s_new, top / torch.full_like(top, 448.0))  # IEEE division, as the kernel's
            old = codes[:, dp].clone()
            first_moved = min(rows)
            for sl in range(16):
                if sl in rows:
                    sp, ss = rows[sl]
                    c, s = (old if sp == dp else codes[:, sp])[:, :, :, ss], scales[:, sp]
                elif sl < first_moved:
                    c, s = old[:, :, :, sl], scales[:, dp]
                else:
                    continue
                again = enc(dec(c) * s[..., None] / s_new[..., None])
                codes[:, dp, :, :, sl] = torch.where((s == s_new)[..., None], c, again)
            scales[:, dp] = s_new
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    P = max(map(len, paths))
    pool.compact_tree(bt, i32(ctx), i32([p + [-1] * (P - len(p)) for p in paths]), i32([len(p) for p in paths]))
    pool.raise_on_status()
    assert torch.equal(pool.scale_view(), scales)
    for b, path in enumerate(paths):  # every row that is a token afterwards
        for pos in range(ctx[b] + len(path)):
            pg = int(bt[b, pos // 16])
            assert torch.equal(pool.pool_view()[:, pg, :, :, pos % 16], codes[:, pg, :, :, pos % 16]), (b, pos)


def test_compact_tree_reports_and_refuses(cuda_device):
    dev = cuda_device
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    bt, pages = tables([40, 40], dev, 2)
    pool = KVPool(1, 2, D, pages, "fp16", device=dev)
    fill_pool(pool, gen(1, dev))
    keep = pool.pool_view().clone()
    for path, n, ctx in [([[0, 5, 5]], [3], [3]), ([[0, 5, 4]], [3], [3]), ([[-1, 2, 3]], [3], [3]),
                         ([[0, 1, 45]], [3], [3]), ([[0, 1, 5]], [4], [3]), ([[0, 1, 5]], [-1], [3]),
                         ([[0, 1, 5]], [3], [-2]), ([[0, 1, 2 ** 31 - 1]], [3], [30])]:
        pool.compact_tree(bt, i32(ctx), i32(path), i32(n))
        assert pool.status()[0] == N.SCKV_ERR_BOUNDS and pool.status()[2] == 20, (path, n, ctx)
        pool.clear_status()
        assert torch.equal(keep, pool.pool_view())
    for kw in [dict(layer0=1), dict(n_layers=2), dict(n_layers=0), dict(max_blocks=9)]:
        with pytest.raises(ValueError):
            pool.compact_tree(bt, i32([3]), i32([[0, 2]]), i32([2]), **kw)
    with pytest.raises(ValueError):
        pool.compact_tree(bt, i32([]), i32([[0, 2]]), i32([2]))
    with pytest.raises(TypeError):
        pool.compact_tree(bt, i32([3]), torch.zeros(1, 2, dtype=torch.int64, device=dev), i32([2]))


# ---------------------------------------------------------------- verify
def walk(logits, tokens, parents, cu, max_path):
    paths, keeps, nexts = [], [], []
    best = []
    for row in logits.float().cpu():
        top = torch.where(row.isnan(), torch.full_like(row, math.inf), row)
        nan = row.isnan().nonzero()
        best.append(int(nan[0]) if len(nan) else int((top == top.max()).nonzero()[0]))
    for a, z in zip(cu, cu[1:]):
        path, nxt = [], -1
        if z > a:
            path = [0]
            while len(path) < max_path:
                kids = [j for j in range(path[-1] + 1, z - a) if parents[a + j] == path[-1] and
                        tokens[a + j] == best[a + path[-1]]]
                if not kids:
                    break
                path.append(kids[0])
            nxt = best[a + path[-1]]
        paths.append(path + [-1] * (max_path - len(path)))
        keeps.append(len(path))
        nexts.append(nxt)
    return paths, keeps, nexts


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1, 7, 33, 1000, 4099, 50281])
@pytest.mark.parametrize("pad", [0, 3])
def test_verify_tree(cuda_device, dtype, vocab, pad):
    dev, g = cuda_device, gen(vocab, cuda_device)
    r = torch.Generator().manual_seed(vocab)
    sizes = [1, 0, 5, 17, 40, 70]
    cu = [sum(sizes[:i]) for i in range(len(sizes) + 1)]
    T = cu[-1]
    parents = [-1 if i == 0 else int(torch.randint(max(0, i - 6), i, (1,), generator=r)) for n in sizes for i in range(n)]
    # few distinct values: ties everywhere
    full = torch.randint(-4, 5, (T, vocab + pad), generator=g, device=dev).to(dtype)
    logits = full[:, pad:] if pad else full
    logits[3, vocab // 2] = math.nan
    logits[4] = -math.inf
    best = walk(logits, [0] * T, [-5] * T, list(range(T + 1)), 1)[2]
    tokens = [0] * T
    for a, n in zip(cu, sizes):
        for i in range(n):
            p = parents[a + i]
            tokens[a + i] = best[a + p] if p >= 0 and torch.rand(1, generator=r) < 0.8 else int(
                torch.randint(0, vocab, (1,), generator=r))
    pool = KVPool(1, 1, D, 1, "fp16", device=dev)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    for mp in (1, 3, 70):
        path, keep, nxt = pool.verify_tree(logits, i32(tokens), i32(parents), i32(cu), max_path=mp)
        assert (path.tolist(), keep.tolist(), nxt.tolist()) == walk(logits, tokens, parents, cu, mp)
    pool.raise_on_status()


def test_verify_tree_reports_and_refuses(cuda_device):
    dev = cuda_device
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    pool = KVPool(1, 1, D, 1, "fp16", device=dev)
    x = torch.randn(1030, 50, device=dev)
    par = i32([i - 1 for i in range(1030)])
    for cu in ([0, 1030], [0, 2000], [-1, 3], [5, 3]):
        path, keep, nxt = pool.verify_tree(x, par, par, i32(cu), max_path=4)
        assert keep.tolist() == [0] and nxt.tolist() == [-1] and path.tolist() == [[-1] * 4]
        assert pool.status()[0] == N.SCKV_ERR_BOUNDS and pool.status()[2] == 19
        pool.clear_status()
    for bad in [(x[0], par, par, i32([0, 4])), (x, par[:3], par, i32([0, 4])), (x[:, :0], par, par, i32([0, 4])),
                (x, par, par, i32([]))]:
        with pytest.raises(ValueError):
            pool.verify_tree(*bad)
    with pytest.raises(TypeError):
        pool.verify_tree(x, par.long(), par, i32([0, 4]))
    with pytest.raises(ValueError):
        pool.verify_tree(x, par, par, i32([0, 4]), max_path=0)
    path, keep, nxt = pool.verify_tree(x[:0], par[:0], par[:0], i32([0]))
    assert path.shape[0] == keep.numel() == nxt.numel() == 0


# -------------------------------------------------------------- together
@pytest.mark.parametrize("kind", KINDS)
def test_cache_tree_step(cuda_device, kind):
    """begin, append, attend, verify, commit: the cache afterwards is that of the accepted tokens alone."""
    dev, g = cuda_device, gen(11, cuda_device)
    L, H, hq = 2, 2, 8
    ctx, trees = [14, 33, 3], [[-1, 0, 0, 1, 2, 2, 4, 5], [-1], [-1] + [0] * 20]
    c = PagedKVCache(L, H, D, 40, 4, 8, kind, device=dev)
    src = torch.bfloat16 if kind == "bf16" else torch.float16
    for s, n in zip("abc", ctx):
        c.add_sequence(s)
        c.append_prefill(s, *(torch.randn(L, n, H, D, generator=g, device=dev).to(src) for _ in range(2)))
    before = [c.gather(s, torch.float32) for s in "abc"]
    free0 = c.pool.alloc_state()["free"]
    n = [len(t) for t in trees]
    cu, ctx_d = c.begin_tree(n)
    assert cu.tolist() == [0, 8, 9, 30] and ctx_d.tolist() == ctx
    k, v = (torch.randn(L, sum(n), H, D, generator=g, device=dev).to(src) for _ in range(2))
    mask, _ = tree_mask(trees, dev)
    q = torch.randn(sum(n), hq, D, generator=g, device=dev).to(src)
    for l in range(L):
        c.append_tree(l, k[l], v[l], cu, ctx_d)
        out = c.tree_attention(l, q, cu, ctx_d, mask)
        ref, absum, big = reference(values(c.pool), l, q, cu.tolist(), ctx, c.block_table, mask, D ** -0.5)
        assert ((out.double() - ref).abs() <= tolerance(kind, src, src, ref, absum, big)).all()
    for refused in (lambda: c.begin_tree([1]), lambda: c.decode_reserve(3), lambda: c.remove_sequence("a"),
                    lambda: c.fork("a", "z"), lambda: c.move_to_row("a", 1)):
        with pytest.raises(RuntimeError):
            refused()
    logits = torch.full((sum(n), 9), -1.0, device=dev)
    for i, t in ((0, 5), (2, 6), (4, 7), (8, 2), (9, 3)):
        logits[i, t] = 1.0
    tokens = torch.tensor([0, 1, 5, 0, 6, 0, 8, 0] + [0] + [0] + [4] * 9 + [3] + [4] * 10, dtype=torch.int32, device=dev)
    parents = torch.tensor([p for t in trees for p in t], dtype=torch.int32, device=dev)
    path, keep, nxt = c.pool.verify_tree(logits, tokens, parents, cu, max_path=max(n))
    assert keep.tolist() == [3, 1, 2] and nxt.tolist() == [7, 2, 0]
    assert path[0, :3].tolist() == [0, 2, 4] and path[2, :2].tolist() == [0, 10]
    c.commit_tree(path, keep, keep.tolist())
    c.check()
    assert c.lengths == [17, 34, 5] and c.ctx_lens[:3].tolist() == [17, 34, 5]
    used = [2, 3, 1]
    assert free0 - c.pool.alloc_state()["free"] == sum(used) - 1 - 3 - 1
    assert [(c.block_table[r] >= 0).sum().item() for r in range(3)] == used
    for r, (s, nodes) in enumerate(zip("abc", ([0, 2, 4], [8], [9, 19]))):
        for kv, new in enumerate((k, v)):
            now, old = c.gather(s, torch.float32)[kv], before[r][kv]
            want = torch.cat([old, new[:, nodes].permute(0, 2, 1, 3).float()], 2)
            if kind in TORCH:
                assert torch.equal(now, want)
            else:
                # int8: half a code of the row's 127 and the scale's and value's fp16 roundings; e4m3: 2^-4 of the
                # value (each time a page's scale grows) or half of the smallest code
                top = want.abs().amax(-1, keepdim=True) if kind == "int8" else want.abs().amax()
                tol = top * (0.51 / 127 + 2.0 ** -9) if kind == "int8" else 3 * 2.0 ** -4 * want.abs() + top * 2.0 ** -17
                assert ((now - want).abs() <= tol).all()
    # a dropped tree leaves the rows as they are
    lens, table = list(c.lengths), c.block_table.clone()
    c.begin_tree([30, 2, 16])
    zero = torch.zeros(3, dtype=torch.int32, device=dev)
    c.commit_tree(zero[:, None], zero, [0, 0, 0])
    assert c.lengths == lens and torch.equal(table, c.block_table)
    with pytest.raises(RuntimeError):
        c.commit_tree(zero[:, None], zero, [0, 0, 0])
    with pytest.raises(ValueError):
        c.begin_tree([1, 257, 1])
    c.begin_tree([2, 2])
    with pytest.raises(ValueError):
        c.commit_tree(zero[:2, None], zero[:2], [3, 0])
    with pytest.raises(ValueError):
        c.commit_tree(zero[:2, None], zero[:2], [2, 0])  # more than the path's width
    c.commit_tree(zero[:2, None], zero[:2], [1, 0])
    assert c.lengths[0] == lens[0] + 1


@pytest.mark.parametrize("kind", KINDS)
def test_attention_layer_tree_equals_decode(cuda_device, kind):
    """A chain through PagedAttentionLayer.tree is as many decode steps: same layer outputs and cached rows."""
    dev, g = cuda_device, gen(5, cuda_device)
    hid, hq, H, n = 256, 4, 2, 5
    wt = torch.bfloat16 if kind == "bf16" else torch.float16
    w = [(torch.randn(o, hid, generator=g, device=dev) / 16).to(wt) for o in (hq * D, H * D, H * D)]
    w_o = (torch.randn(hid, hq * D, generator=g, device=dev) / 22).to(wt)
    norm = [(1 + 0.1 * torch.randn(D, generator=g, device=dev)).half() for _ in range(2)]
    x0, x = torch.randn(20, hid, generator=g, device=dev), torch.randn(n, hid, generator=g, device=dev)
    outs, caches = [], []
    for tree in (False, True):
        c = PagedKVCache(1, H, D, 16, 2, 8, kind, device=dev)
        layer = PagedAttentionLayer(c, hq, rope_theta=10000.0)
        c.add_sequence("s")
        layer.prefill(0, "s", x0, *w, w_o, *norm)
        if tree:
            cu, ctx = c.begin_tree([n])
            mask, depth = tree_mask([[i - 1 for i in range(n)]], dev)
            outs.append(layer.tree(0, x, depth + 20, mask, cu, ctx, *w, w_o, *norm))
            path = torch.arange(n, dtype=torch.int32, device=dev)[None]
            c.commit_tree(path, torch.tensor([n], dtype=torch.int32, device=dev), [n])
        else:
            outs.append(torch.cat([layer.decode(0, x[i:i + 1], 1, *w, w_o, *norm) for i in range(n)]))
        c.check()
        caches.append(c.gather("s", torch.float32))
    # K and V come from the same products with fp32 accuracy: they round to the same code or its neighbour
    step = {"fp16": 2.0 ** -10, "bf16": 2.0 ** -7, "int8": 0.02, "fp8_e4m3": 2.0 ** -3 + 2.0 ** -4}[kind]
    for a, b in zip(*caches):
        top = a.abs().amax(-1, keepdim=True) if kind == "int8" else a.abs()
        assert ((a - b).abs() <= step * top + 1e-3 * a.abs().amax()).all()
    # roundings of q (f16; bf16) and P before o_proj, and of the cached rows above, averaged over the row
    tol = {"fp16": 4 * 2.0 ** -11, "bf16": 6 * 2.0 ** -8, "int8": 8 * 2.0 ** -8, "fp8_e4m3": 3 * 2.0 ** -4}[kind]
    assert float((outs[0] - outs[1]).norm() / outs[0].norm()) <= tol


class Oracle:
    """Drafts what one-by-one decoding says, with wrong branches around it."""

    def __init__(self, said):
        self.said = said  # prompt -> tokens

    def propose(self, tokens, max_nodes):
        for prompt, out in self.said.items():
            if tuple(tokens[:len(prompt)]) == prompt and list(tokens[len(prompt):]) == out[:len(tokens) - len(prompt)]:
                rest = out[len(tokens) - len(prompt):][:3]
                toks, par, cur = [], [], -1
                for t in rest:
                    toks += [(t + 1) % 500, t]
                    par += [cur, cur]
                    cur = len(toks) - 1
                return toks[:max_nodes], par[:max_nodes]
        return [], []


@pytest.mark.parametrize("drafter", ["oracle", "lookup"])
def test_scheduler_with_a_drafter_says_the_same(cuda_device, drafter):
    from stub_model import CFG, TorchStubModel, make_weights, prompts

    dev = cuda_device
    model = TorchStubModel(make_weights(), dev)

    def run(d):
        c = PagedKVCache(CFG["num_layers"], CFG["hkv"], CFG["head_dim"], 256, 8, 16, "fp16", device=dev)
        s = ContinuousBatchScheduler(model, c, max_batch_size=4, drafter=d)
        for i, p in enumerate(prompts()):
            s.submit_request(f"r{i}", p, max_new_tokens=9, stop_token_ids=set())
        steps = s.run_until_complete()
        c.check()
        assert c.n_live == 0 and c.pool.alloc_state()["allocated"] == 0
        return {r: list(q.generated_ids) for r, q in s.completed_requests.items()}, s, steps

    plain, _, plain_steps = run(None)
    said = {tuple(p): plain[f"r{i}"] for i, p in enumerate(prompts())}
    got, s, steps = run(Oracle(said) if drafter == "oracle" else PromptLookupDrafter())
    assert got == plain
    if drafter == "oracle":
        assert s.accepted_drafts > 0 and len(steps) < len(plain_steps)
    for rid in got:
        assert [t for st in steps for t in st["accepted_tokens"].get(rid, [])] == got[rid]


def test_scheduler_drafter_refusals(cuda_device):
    from stub_model import CFG, TorchStubModel, make_weights

    dev = cuda_device
    model = TorchStubModel(make_weights(), dev)
    c = PagedKVCache(CFG["num_layers"], CFG["hkv"], CFG["head_dim"], 64, 2, 8, "fp16", device=dev)
    with pytest.raises(ValueError):
        ContinuousBatchScheduler(model, c, drafter=PromptLookupDrafter(), capture_decode=True)

    class Bad:
        def propose(self, tokens, max_nodes):
            return [1, 2], [-1, 1]

    s = ContinuousBatchScheduler(model, c, drafter=Bad())
    s.submit_request("r", [1, 2, 3], max_new_tokens=5, stop_token_ids=set())
    s.step_batch()
    with pytest.raises(ValueError):
        s.step_batch()


# ----------------------------------------------------------- wider ranges
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hq,nodes", [(1, 1), (8, 5), (8, 64)])
def test_tree_attn_one_item_over_all_sms(cuda_device, kind, hq, nodes):
    """One K/V head of one sequence: a part of the sum in nearly every SM."""
    check_attn(cuda_device, kind, hq, 1, [16000], [nodes], seed=hq + nodes)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("seqs,ctx,hq,hkv", [(60, 700, 16, 2), (15, 1251, 64, 8), (40, 300, 48, 3)])
def test_tree_attn_row_groups_of_all_sizes_in_turn(cuda_device, kind, seqs, ctx, hq, hkv):
    """An SM takes items of two query tiles and of one, with one, two and four copies of its rows, in any order."""
    r = torch.Generator().manual_seed(seqs)
    nodes = torch.randint(1, 41, (seqs,), generator=r).tolist()
    nodes[0::4] = [35] * len(nodes[0::4])
    check_attn(cuda_device, kind, hq, hkv, [ctx - 3 * b for b in range(seqs)], nodes, seed=seqs)


def test_tree_attn_limits(cuda_device):
    dev = cuda_device
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    pool = KVPool(1, 1, D, 4, "fp16", device=dev)
    fill_pool(pool, gen(1, dev))
    for seqs, ok in ((2048, True), (2049, False)):
        bt = i32([[0]] * seqs)
        q = torch.randn(seqs, 2, D, generator=gen(2, dev), device=dev).half()
        mask = torch.ones(seqs, 1, dtype=torch.int64, device=dev)
        args = (0, q, i32(range(seqs + 1)), i32([i % 15 for i in range(seqs)]), bt, mask)
        if ok:
            out = pool.tree_attn(*args)
            ref, absum, big = reference(values(pool), 0, q[:40], list(range(41)), [i % 15 for i in range(40)], bt,
                                        mask[:40], D ** -0.5)
            tol = tolerance("fp16", q.dtype, q.dtype, ref, absum, big)
            assert ((out[:40].double() - ref).abs() <= tol).all()
        else:
            with pytest.raises(SCKVError):
                pool.tree_attn(*args)
    wide = torch.zeros(1, 4096, D, dtype=torch.float16, device=dev)
    one = torch.ones(1, 1, dtype=torch.int64, device=dev)
    with pytest.raises(SCKVError):
        pool.tree_attn(0, wide, i32([0, 1]), i32([3]), i32([[0]]), one)
    check_attn(dev, "fp16", 4095, 1, [20], [1], seed=3)
    pool.raise_on_status()


@pytest.mark.parametrize("src", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lens", [[2500], [4000, 1200], [7100, 1], [9000, 17, 1203]])
def test_append_rope_axes_of_long_prompts(cuda_device, src, lens):
    """Token counts that give a CTA one to four tokens; no sequence owns the last three."""
    dev, g = cuda_device, gen(len(lens), cuda_device)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    hq, hkv, T = 3, 2, sum(lens) + 3
    start = [5 + b for b in range(len(lens))]
    bt, pages = tables([a + n for a, n in zip(start, lens)], dev, 2)
    cu = [sum(lens[:b]) for b in range(len(lens) + 1)]
    kind = "bf16" if src == torch.bfloat16 else "fp16"
    pool = KVPool(1, hkv, D, pages, kind, device=dev)
    x = torch.randn(T, hq + 2 * hkv, D, generator=g, device=dev).to(src)
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    w = [(1 + 0.2 * torch.randn(D, generator=g, device=dev)).half() for _ in range(2)]
    pos = torch.randint(0, 10 ** 6, (2, T), generator=g, device=dev, dtype=torch.int32)
    axis, freq = rope_axis_map([40, 24], device=dev), rope_inv_freq(1e6, D, dev)
    q_out = torch.full((T, hq, D), 7.0, dtype=src, device=dev)
    pool.append_rope_axes(0, q, k, v, pos, axis, i32(cu), i32(start), bt, freq, q_norm_w=w[0], k_norm_w=w[1], eps=1e-5,
                          q_out=q_out)
    pool.raise_on_status()
    n = T - 3
    assert (q_out[n:] == 7).all()
    t = torch.arange(n, device=dev)
    b = torch.searchsorted(i32(cu), t.int(), right=True) - 1
    at = i32(start).long()[b] + t - i32(cu).long()[b]
    rows = pool.pool_view()[0][bt.long()[b, at // 16], :, :, at % 16]  # [n, 2, hkv, D]
    # (the same roundings as in test_append_rope_axes)
    for y, wx, got, out in ((q, w[0], q_out[:n], src), (k, w[1], rows[:, 0], TORCH[kind])):
        ref, size = rope_reference(y[:n], wx, 1e-5, pos[:, :n], axis, freq, 1.0)
        tol = size * 80 * 2.0 ** -24
        assert ((got.double() - ref).abs() <= tol + HALF[out] * (ref.abs() + tol) + 1e-7).all()
    assert torch.equal(rows[:, 1], v[:n].to(TORCH[kind]))


@pytest.mark.parametrize("kind", ["fp16", "int8"])
def test_compact_tree_long_paths(cuda_device, kind):
    """More moved rows than one batch of looked-up pages, over and past pages that they came from."""
    dev, g = cuda_device, gen(5, cuda_device)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    ctx = [5, 48]
    paths = [list(range(10)) + list(range(11, 611)), list(range(0, 900, 2))]
    bt, pages = tables([c + p[-1] + 1 for c, p in zip(ctx, paths)], dev, 2)
    pool = KVPool(2, 3, D, pages, kind, device=dev)
    fill_pool(pool, g)
    views = [pool.pool_view()] + ([pool.scale_view()] if kind == "int8" else [])
    want = [v.clone() for v in views]
    for b, path in enumerate(paths):
        src, dst = torch.tensor(path, device=dev) + ctx[b], torch.arange(len(path), device=dev) + ctx[b]
        ids = bt[b].long()
        for v, x in zip(views, want):
            x[:, ids[dst // 16], :, :, dst % 16] = v[:, ids[src // 16], :, :, src % 16]
    P = max(len(p) for p in paths)
    pool.compact_tree(bt, i32(ctx), i32([p + [-1] * (P - len(p)) for p in paths]), i32([len(p) for p in paths]))
    pool.raise_on_status()
    assert all(torch.equal(v, x) for v, x in zip(views, want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_verify_tree_rows_of_any_alignment(cuda_device, dtype):
    """Rows that begin and end anywhere in 16 bytes, their largest value (the first of equals, 0 and -0 among them) or
    NaN anywhere."""
    dev, g = cuda_device, gen(9, cuda_device)
    T = 64
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    pool = KVPool(1, 1, D, 1, "fp16", device=dev)
    zero, cu = torch.zeros(T, dtype=torch.int32, device=dev), i32(range(T + 1))
    for vocab in (1, 2, 5, 8, 13, 24, 31, 77, 2049, 4100):
        for off in range(0, 9, 1 if vocab < 40 else 3):
            full = torch.randint(-3, 4, (T, vocab + off + vocab % 5), generator=g, device=dev).to(dtype)
            full[full == 3] = -0.0
            x = full[:, off:off + vocab]
            full[:, :off] = 100
            full[:, off + vocab:] = 100
            x[:16].clamp_(max=0)
            where = torch.randint(0, vocab, (16,), generator=g, device=dev)
            x[torch.arange(16, 32, device=dev), where] = math.nan
            x[32:40] = -math.inf
            path, keep, nxt = pool.verify_tree(x, zero, zero - 1, cu, max_path=1)
            assert nxt.tolist() == walk(x, [0] * T, [-1] * T, list(range(T + 1)), 1)[2], (vocab, off)
    pool.raise_on_status()


@pytest.mark.parametrize("kind", KINDS)
def test_captured_tree_step_equals_the_calls(cuda_device, kind):
    """append, attend, verify and move as one captured graph, replayed on new inputs and lengths."""
    dev = cuda_device
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    trees = [[-1, 0, 0, 1, 1, 2, 2], [-1], [-1, 0, 1, 2, 0]]
    n = [len(t) for t in trees]
    cu = i32([0, n[0], n[0] + n[1], sum(n)])
    mask, depth = tree_mask(trees, dev)
    parents = i32([p for t in trees for p in t])
    T, hq, hkv = sum(n), 4, 2
    src = torch.bfloat16 if kind == "bf16" else torch.float16
    bt, pages = tables([200] * 3, dev, 4)
    pools = [KVPool(1, hkv, D, pages, kind, device=dev) for _ in range(2)]
    for p in pools:
        fill_pool(p, gen(6, dev))
    axis, freq = rope_axis_map([64], device=dev), rope_inv_freq(1e4, D, dev)

    def inputs(i):
        g = gen(20 + i, dev)
        x = torch.randn(T, hq + 2 * hkv, D, generator=g, device=dev).to(src)
        ctx = i32([17 + 31 * i, 1 + i, 100 - 7 * i])
        pos = (torch.repeat_interleave(ctx, i32(n).long()) + depth).to(torch.int32)
        logits = torch.randint(0, 2, (T, 50), generator=g, device=dev).float()
        tokens = torch.randint(0, 3, (T,), generator=g, device=dev, dtype=torch.int32)
        return [x, ctx, pos, logits, tokens]

    def step(pool, x, ctx, pos, logits, tokens):
        q = pool.append_rope_axes(0, x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:], pos, axis, cu, ctx, bt, freq)
        out = pool.tree_attn(0, q, cu, ctx, bt, mask)
        path, keep, nxt = pool.verify_tree(logits, tokens, parents, cu, max_path=8)
        pool.compact_tree(bt, ctx, path, keep)
        return q, out, path, keep, nxt

    held = inputs(0)
    step(pools[0], *held), step(pools[1], *held)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(pools[0], *held)
    for i in (1, 2):
        new = inputs(i)
        for a, b in zip(held, new):
            a.copy_(b)
        graph.replay()
        want = step(pools[1], *new)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert torch.equal(pools[0].pool_view(), pools[1].pool_view())
    for p in pools:
        p.raise_on_status()
