"""Workloads of the speculative-decoding operators over the paged KV cache.

One decoding step checks a tree of drafted tokens per sequence: the nodes'
q and k are normed, rotated at their own positions and appended
(`append_rope_axes`), every node attends over its sequence's cached tokens and
its own ancestors (`tree_attn`), the logits pick the accepted path
(`verify_tree`), and the accepted rows move next to the committed ones
(`compact_tree`). `append_rope_axes` also serves prompts whose tokens have
(time, height, width) positions.

Each case is one call. `run` computes it in elementary torch operations, or,
with `own` set, through `synapcore_b200.KVPool`.
"""
from __future__ import annotations

import math

import torch

own = False

PAGE = 16
DIM = 128
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# --------------------------------------------------------------------- cases
def listed():
    return [
        # one chat, a small tree over a short context: latency
        {"name": "attn_one_small", "op": "attn", "kv": "bf16", "q": "bf16", "seqs": 1, "ctx": 700, "spread": 0,
         "nodes": 8, "hq": 32, "hkv": 8},
        # a batch of a model without grouped heads
        {"name": "attn_mha_batch", "op": "attn", "kv": "fp16", "q": "fp16", "seqs": 32, "ctx": 4096, "spread": 1500,
         "nodes": 24, "hq": 16, "hkv": 16},
        # the largest: grouped heads over FP8 pages, long contexts of different lengths
        {"name": "attn_fp8_long", "op": "attn", "kv": "fp8_e4m3", "q": "bf16", "seqs": 64, "ctx": 16384,
         "spread": 4000, "nodes": 16, "hq": 32, "hkv": 8},
        # groups of 7 heads, int8 pages, odd lengths
        {"name": "attn_int8_odd", "op": "attn", "kv": "int8", "q": "bf16", "seqs": 23, "ctx": 5003, "spread": 3001,
         "nodes": 13, "hq": 28, "hkv": 4},
        # few sequences with very long contexts and wide trees
        {"name": "attn_bf16_wide", "op": "attn", "kv": "bf16", "q": "bf16", "seqs": 4, "ctx": 65536, "spread": 999,
         "nodes": 64, "hq": 32, "hkv": 8},
        # a prompt with images: (time, height, width) positions, per-head norms
        {"name": "rope_prompt_3axes", "op": "rope", "kv": "bf16", "seqs": 5, "tokens": 8192, "hq": 32, "hkv": 8,
         "axes": 3, "norm": True, "far": 200000},
        # the nodes of a batch's trees: one axis, positions by depth
        {"name": "rope_tree_1axis", "op": "rope", "kv": "fp16", "seqs": 64, "tokens": 771, "hq": 16, "hkv": 16,
         "axes": 1, "norm": False, "far": 30000},
        # one sequence's tree: latency
        {"name": "rope_one_small", "op": "rope", "kv": "bf16", "seqs": 1, "tokens": 9, "hq": 28, "hkv": 4,
         "axes": 3, "norm": True, "far": 4000},
        # accepted rows of a batch, every layer
        {"name": "compact_batch", "op": "compact", "kv": "bf16", "seqs": 64, "ctx": 100, "nodes": 48, "keep": 6,
         "layers": 36, "hkv": 8},
        # accepted rows of one sequence
        {"name": "compact_one", "op": "compact", "kv": "fp16", "seqs": 1, "ctx": 1001, "nodes": 16, "keep": 4,
         "layers": 16, "hkv": 16},
        # the vocabulary of a large model, a full batch of trees
        {"name": "verify_batch", "op": "verify", "logits": "bf16", "seqs": 48, "nodes": 24, "vocab": 151936},
        # one tree, fp32 logits, an odd vocabulary
        {"name": "verify_one", "op": "verify", "logits": "fp32", "seqs": 1, "nodes": 10, "vocab": 50281},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "rope", "compact", "verify"])
    if op == "attn":
        kv = rng.choice(["fp16", "bf16", "int8", "fp8_e4m3"])
        hq, hkv = rng.choice([(32, 8), (16, 16), (28, 4), (8, 1), (40, 8), (64, 8), (12, 6)])
        ctx = _log(rng, 1, 60000)
        nodes = _log(rng, 1, 64)
        # at most the largest listed case's cached tokens times heads, and the widest one's products
        most = min(64, max(1, 4_000_000 // ((ctx + nodes) * hkv)), max(1, 500_000_000 // ((ctx + nodes) * hq * nodes)))
        return {"op": "attn", "kv": kv, "q": "fp16" if kv == "fp16" else "bf16", "seqs": _log(rng, 1, most),
                "ctx": ctx, "spread": rng.randrange(0, max(1, ctx // 2)), "nodes": nodes, "hq": hq, "hkv": hkv}
    if op == "rope":
        tokens = _log(rng, 1, 8192)
        hq, hkv = rng.choice([(32, 8), (16, 16), (28, 4), (12, 6)])
        return {"op": "rope", "kv": rng.choice(["fp16", "bf16"]), "seqs": min(tokens, _log(rng, 1, 64)),
                "tokens": tokens, "hq": hq, "hkv": hkv, "axes": rng.choice([1, 2, 3]), "norm": rng.random() < 0.5,
                "far": _log(rng, 100, 200000)}
    if op == "compact":
        keep = _log(rng, 1, 12)
        return {"op": "compact", "kv": rng.choice(["fp16", "bf16"]), "seqs": _log(rng, 1, 64),
                "ctx": _log(rng, 1, 110), "nodes": min(64, keep * rng.randrange(2, 6)), "keep": keep,
                "layers": rng.randrange(1, 37), "hkv": rng.choice([1, 4, 8])}
    return {"op": "verify", "logits": rng.choice(["bf16", "fp16", "fp32"]), "seqs": _log(rng, 1, 24),
            "nodes": _log(rng, 1, 24), "vocab": _log(rng, 1000, 152000)}


# -------------------------------------------------------------------- inputs
def _tree(g, n):
    """Parents of n nodes in breadth-first order: node 0 is the root, a later
    one hangs on one of the few before it."""
    par = [-1]
    for i in range(1, n):
        lo = max(0, (i - 1) // 4 - 3)
        par.append(int(torch.randint(lo, (i - 1) // 2 + 1, (1,), generator=g)))
    return par


def _mask(par):
    """Bit j of entry i: node j is i or an ancestor of it (64-bit two's complement)."""
    out = []
    for i, p in enumerate(par):
        out.append((1 << i) | (out[p] if p >= 0 else 0))
    return [m - (1 << 64) if m >= 1 << 63 else m for m in out]


def _depth(par):
    out = []
    for p in par:
        out.append(out[p] + 1 if p >= 0 else 0)
    return out


def _table(g, lens, most, dev):
    """Pages of a pool in a shuffled order: block table [n, blocks] of sequences
    of `lens` tokens, and the pool's page count, with room for `most` tokens each."""
    blocks = [-(-n // PAGE) for n in lens]
    total = sum(-(-n // PAGE) for n in most) + 3
    ids = torch.randperm(total, generator=g).tolist()
    rows, at = [], 0
    for b in blocks:
        rows.append(ids[at:at + b] + [-1] * (max(blocks) - b))
        at += b
    return torch.tensor(rows, dtype=torch.int32).to(dev), total


def _store(kv, data, scales, layers, pages, hkv, dev):
    """The page pool that a serving program holds: KVPool's, or its bytes."""
    s = {"kv": kv, "data": data, "scales": scales, "pool": None}
    if own:
        from synapcore_b200 import KVPool

        pool = KVPool(layers, hkv, DIM, pages, kv, device=dev)
        pool.pool_view().copy_(data)
        if scales is not None:
            pool.scale_view().copy_(scales)
        s |= {"pool": pool, "data": pool.pool_view(), "scales": pool.scale_view()}
    return s


def _pages(kv, layers, pages, hkv, gd, dev):
    """K and V pages [layers, pages, 2, hkv, 16, D] with their scales."""
    shape = (layers, pages, 2, hkv, PAGE, DIM)
    if kv in DTYPES:
        return torch.randn(shape, generator=gd, device=dev, dtype=DTYPES[kv]), None
    x = torch.randn(shape, generator=gd, device=dev, dtype=torch.float16)
    # tokens of different sizes
    x *= torch.exp(0.3 * torch.randn(shape[:-1] + (1,), generator=gd, device=dev)).half()
    if kv == "int8":
        s = (x.abs().amax(-1, keepdim=True).float() / 127).clamp_min(1e-7)
        q = torch.empty(shape, dtype=torch.int8, device=dev)
        for i in range(layers):
            q[i] = torch.clamp(torch.round(x[i].float() / s[i]), -127, 127).to(torch.int8)
        return q, s[..., 0].half()
    s = x.abs().amax((-1, -2)).float() / 448
    q = torch.empty(shape, dtype=torch.uint8, device=dev)
    for i in range(layers):
        q[i] = (x[i].float() / s[i][..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    return q, s


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator().manual_seed(seed)
    gd = torch.Generator(device=dev).manual_seed(seed)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).to(dev)  # noqa: E731
    op, S = case["op"], case["seqs"]
    if op == "attn":
        n, hq, hkv = case["nodes"], case["hq"], case["hkv"]
        # the first sequence has the full length and tree, others are shorter
        ctx = [max(1, case["ctx"] - (int(torch.randint(0, case["spread"] + 1, (1,), generator=g)) if b else 0))
               for b in range(S)]
        nn = [max(1, n - (b % 3)) for b in range(S)]
        trees = [_tree(g, m) for m in nn]
        bt, pages = _table(g, [c + m for c, m in zip(ctx, nn)], [case["ctx"] + n] * S, dev)
        data, scales = _pages(case["kv"], 1, pages, hkv, gd, dev)
        s = _store(case["kv"], data, scales, 1, pages, hkv, dev)
        del data, scales
        cu = [0]
        for m in nn:
            cu.append(cu[-1] + m)
        s |= {"bt": bt, "ctx": i32(ctx), "cu": i32(cu), "nmax": max(nn),
              "mask": torch.tensor([m for t in trees for m in _mask(t)], dtype=torch.int64).to(dev)[:, None],
              "q": (2 * torch.randn(cu[-1], hq, DIM, generator=gd, device=dev)).to(DTYPES[case["q"]]),
              "hkv": hkv, "scale": DIM ** -0.5}
    elif op == "rope":
        T, hq, hkv, A = case["tokens"], case["hq"], case["hkv"], case["axes"]
        dt = DTYPES[case["kv"]]
        base, extra = divmod(T, S)
        lens = [base + (b < extra) for b in range(S)]
        start = [int(torch.randint(0, 40, (1,), generator=g)) for _ in range(S)]
        bt, pages = _table(g, [a + m for a, m in zip(start, lens)], [40 + m for m in lens], dev)
        s = _store(case["kv"], *_pages(case["kv"], 1, pages, hkv, gd, dev), 1, pages, hkv, dev)
        cu = [0]
        for m in lens:
            cu.append(cu[-1] + m)
        sections = {1: [64], 2: [32, 32], 3: [16, 24, 24]}[A]
        # q, k and v as the rows of one projection's output
        x = (1.5 * torch.randn(T, hq + 2 * hkv, DIM, generator=gd, device=dev)).to(dt)
        w = lambda: (1 + 0.1 * torch.randn(DIM, generator=gd, device=dev)).half()  # noqa: E731
        s |= {"bt": bt, "start": i32(start), "cu": i32(cu), "q": x[:, :hq], "k": x[:, hq:hq + hkv],
              "v": x[:, hq + hkv:],
              "pos": torch.randint(0, case["far"], (A, T), generator=g, dtype=torch.int32).to(dev),
              "axis": torch.repeat_interleave(torch.arange(A), torch.tensor(sections)).to(torch.int32).to(dev),
              "freq": (1000000.0 ** (-torch.arange(0, DIM, 2, dtype=torch.float64) / DIM)).float().to(dev),
              "qw": w() if case["norm"] else None, "kw": w() if case["norm"] else None, "eps": 1e-6}
    elif op == "compact":
        n, keep, L, hkv = case["nodes"], case["keep"], case["layers"], case["hkv"]
        ctx = [case["ctx"] + int(torch.randint(0, 16, (1,), generator=g)) for _ in range(S)]
        bt, pages = _table(g, [c + n for c in ctx], [case["ctx"] + 15 + n] * S, dev)
        s = _store(case["kv"], *_pages(case["kv"], L, pages, hkv, gd, dev), L, pages, hkv, dev)
        path, cnt = [], []
        for b in range(S):
            k = max(1, keep - b % 3)
            # the root, then one node of each later level: breadth-first numbers, wider than deep
            later = sorted((torch.randperm(n - k, generator=g)[:k - 1] + k).tolist()) if n > k else []
            path.append(([0] + later)[:k] + [-1] * (keep - 1 - len(later[:k - 1])))
            cnt.append(1 + len(later[:k - 1]))
        s |= {"bt": bt, "ctx": i32(ctx), "path": i32(path), "keep": i32(cnt)}
    else:
        n, V = case["nodes"], case["vocab"]
        dt = torch.float32 if case["logits"] == "fp32" else DTYPES[case["logits"]]
        trees = [_tree(g, n) for _ in range(S)]
        logits = 3 * torch.randn(S * n, V, generator=gd, device=dev, dtype=dt)
        best = logits.max(-1).indices.tolist()
        hit = torch.rand(S * n, generator=g).tolist()
        rnd = torch.randint(0, V, (S * n,), generator=g).tolist()
        # three of four drafted tokens are what the model says after their parent
        tok = [best[b * n + p] if p >= 0 and hit[b * n + i] < 0.75 else rnd[b * n + i]
               for b, t in enumerate(trees) for i, p in enumerate(t)]
        s = {"logits": logits, "tok": i32(tok), "par": i32([p for t in trees for p in t]),
             "cu": i32([b * n for b in range(S + 1)]), "n": n, "pool": None}
        if own:
            from synapcore_b200 import KVPool

            s["pool"] = KVPool(1, 1, DIM, 1, "fp16", device=dev)
    s["op"] = op
    return s


# --------------------------------------------------------------- plain forms
def _values(s):
    """K and V of every sequence's pages in 32 bits: two [S, hkv, blocks * 16, D]."""
    ids = s["bt"].long().clamp_min(0)
    x = s["data"][0][ids]  # [S, blocks, 2, hkv, 16, D]
    if s["kv"] == "int8":
        x = x.float() * s["scales"][0][ids].float()[..., None]
    elif s["kv"] == "fp8_e4m3":
        x = x.view(torch.float8_e4m3fn).float() * s["scales"][0][ids][..., None, None]
    else:
        x = x.float()
    S, nb, _, h, _, _ = x.shape
    x = x.permute(2, 0, 3, 1, 4, 5).reshape(2, S, h, nb * PAGE, DIM)
    return x[0], x[1]


def _attn(s):
    k, v = _values(s)
    S, hkv, L, _ = k.shape
    cu, ctx, nmax = s["cu"].long(), s["ctx"].long(), s["nmax"]
    dev = k.device
    node = torch.arange(nmax, device=dev)
    rows = cu[:-1, None] + node  # [S, nmax]
    live = node < (cu[1:] - cu[:-1])[:, None]
    rows = rows.clamp_max(s["q"].shape[0] - 1)
    hq = s["q"].shape[1]
    G = hq // hkv
    q = s["q"][rows].float().view(S, nmax, hkv, G, DIM).permute(0, 2, 1, 3, 4).reshape(S, hkv, nmax * G, DIM)
    sc = torch.matmul(q, k.transpose(-1, -2)) * s["scale"]
    at = torch.arange(L, device=dev) - ctx[:, None]  # [S, L]: the key's node, negative for cached tokens
    bits = s["mask"][rows][..., 0]  # [S, nmax]
    sees = (bits[..., None] >> at.clamp(0, 63)[:, None, :]) & 1
    sees = torch.where(at[:, None, :] < 0, torch.ones_like(sees), sees * (at[:, None, :] < nmax))  # [S, nmax, L]
    sees = (sees.bool() & (at < (cu[1:] - cu[:-1])[:, None])[:, None, :])[:, None, :, None, :]
    sc = sc.view(S, hkv, nmax, G, L).masked_fill_(~sees, float("-inf")).view(S, hkv, nmax * G, L)
    top = sc.amax(-1, keepdim=True).clamp_min(-3e38)
    p = sc.sub_(top).exp_()
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True).clamp_min(1e-38)
    o = o.view(S, hkv, nmax, G, DIM).permute(0, 2, 1, 3, 4).reshape(S, nmax, hq, DIM)
    return o[live].to(s["q"].dtype)


def _slots(s, n):
    """Page and in-page slot of n appended tokens."""
    t = torch.arange(n, device=s["cu"].device)
    b = torch.searchsorted(s["cu"].long(), t, right=True) - 1
    p = s["start"].long()[b] + t - s["cu"].long()[b]
    return s["bt"].long()[b, p // PAGE], p % PAGE


def _rotate(x, w, eps, cos, sin):
    x = x.float()
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w.float()
    a, b = x[..., :DIM // 2], x[..., DIM // 2:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _rope(s):
    ang = s["pos"].double()[s["axis"].long()].T * s["freq"].double()  # [T, D / 2]
    cos, sin = ang.cos().float()[:, None], ang.sin().float()[:, None]
    q = _rotate(s["q"], s["qw"], s["eps"], cos, sin).to(s["q"].dtype)
    k = _rotate(s["k"], s["kw"], s["eps"], cos, sin).to(s["data"].dtype)
    page, slot = _slots(s, q.shape[0])
    s["data"][0][page, 0, :, slot] = k
    s["data"][0][page, 1, :, slot] = s["v"].to(s["data"].dtype)
    return q, s["data"]


def _compact(s):
    path, ctx = s["path"].long(), s["ctx"].long()
    j = torch.arange(path.shape[1], device=path.device)
    b, j = torch.nonzero(j < s["keep"][:, None], as_tuple=True)
    src, dst, bt = ctx[b] + path[b, j], ctx[b] + j, s["bt"].long()
    rows = s["data"][:, bt[b, src // PAGE], :, :, src % PAGE]
    s["data"][:, bt[b, dst // PAGE], :, :, dst % PAGE] = rows
    return s["data"]


def _verify(s):
    x, n = s["logits"], s["n"]
    S = x.shape[0] // n
    top = x.amax(-1, keepdim=True)
    col = torch.arange(x.shape[1], device=x.device, dtype=torch.int32)
    best = torch.where(x == top, col, x.shape[1]).amin(-1).view(S, n)
    tok, par = s["tok"].view(S, n), s["par"].long().view(S, n)
    up = par.clamp_min(0)
    good = (tok == best.gather(1, up)) & (par >= 0)
    # of equal tokens under one parent the first counts
    twin = (par[:, :, None] == par[:, None, :]) & (tok[:, :, None] == tok[:, None, :])
    first = ~(twin & torch.ones(n, n, device=x.device, dtype=torch.bool).tril(-1)).any(-1)
    good = good & first
    good[:, 0] = True
    # accepted: the node and all its ancestors are good (pointer jumping over the parents)
    for _ in range(max(1, (n - 1).bit_length())):
        good = good & good.gather(1, up)
        up = up.gather(1, up)
    keep = good.sum(-1).to(torch.int32)
    node = torch.arange(n, device=x.device)
    path = torch.where(good, node, n).sort(-1).values
    last = path.gather(1, (keep.long() - 1)[:, None])
    return torch.where(path < n, path, -1).to(torch.int32), keep, best.gather(1, last)[:, 0].to(torch.int32)


def run(state):
    s = state
    p = s["pool"]
    if s["op"] == "attn":
        if own:
            return p.tree_attn(0, s["q"], s["cu"], s["ctx"], s["bt"], s["mask"], scale=s["scale"])
        return _attn(s)
    if s["op"] == "rope":
        if own:
            q = p.append_rope_axes(0, s["q"], s["k"], s["v"], s["pos"], s["axis"], s["cu"], s["start"], s["bt"],
                                   s["freq"], q_norm_w=s["qw"], k_norm_w=s["kw"], eps=s["eps"])
            return q, s["data"]
        return _rope(s)
    if s["op"] == "compact":
        if own:
            p.compact_tree(s["bt"], s["ctx"], s["path"], s["keep"])
            return s["data"]
        return _compact(s)
    if own:
        return p.verify_tree(s["logits"], s["tok"], s["par"], s["cu"], max_path=s["n"])
    return _verify(s)


# ------------------------------------------------------------ work and truth
def work(case):
    S = case["seqs"]
    if case["op"] == "attn":
        el = {"fp16": 2, "bf16": 2, "int8": 1, "fp8_e4m3": 1}[case["kv"]]
        keys = nodes = prod = 0
        for b in range(S):
            c = max(1, case["ctx"] - (case["spread"] // 2 if b else 0))
            m = max(1, case["nodes"] - b % 3)
            keys += c + m
            nodes += m
            prod += m * (c + m)
        per = 2 * case["hkv"] * (DIM * el + {"int8": 2, "fp8_e4m3": 0.25}.get(case["kv"], 0))
        return {"bytes": keys * per + 2 * nodes * case["hq"] * DIM * 2 + keys / 4 + nodes * 8,
                "flops": 4 * prod * case["hq"] * DIM}
    if case["op"] == "rope":
        rows = case["hq"] + 2 * case["hkv"]
        return {"bytes": case["tokens"] * (rows * DIM * 2 * 2 + 4 * case["axes"]),
                "flops": case["tokens"] * (case["hq"] + case["hkv"]) * DIM * (3 + 4 * case["norm"])}
    if case["op"] == "compact":
        # the root stays where it is
        rows = sum(max(1, case["keep"] - b % 3) - 1 for b in range(S))
        return {"bytes": 2 * max(1, rows) * case["layers"] * 2 * case["hkv"] * DIM * 2, "flops": 0}
    el = 4 if case["logits"] == "fp32" else 2
    n = S * case["nodes"]
    return {"bytes": n * (case["vocab"] * el + 16), "flops": n * case["vocab"]}


def exact(case, seed):
    if case["op"] in ("compact", "verify"):
        return None  # moved rows and whole numbers: nothing that is rounded
    s = prepare(case, seed)
    if case["op"] == "rope":
        cu, start = s["cu"].tolist(), s["start"].tolist()
        half = DIM // 2
        turn = torch.empty(s["q"].shape[0], half, dtype=torch.complex128, device=s["q"].device)
        for i, a in enumerate(s["axis"].tolist()):
            turn[:, i] = torch.polar(torch.ones((), dtype=torch.float64, device=turn.device),
                                     s["pos"][a].double() * s["freq"][i].double())

        def rot(x, w):
            x = x.double()
            if w is not None:
                x = x / (x.square().sum(-1, keepdim=True) / DIM + s["eps"]).sqrt() * w.double()
            z = torch.complex(x[..., :half], x[..., half:]) * turn[:, None]
            return torch.cat([z.real, z.imag], -1)

        q, k, data = rot(s["q"], s["qw"]), rot(s["k"], s["kw"]), s["data"].double()
        for b in range(len(start)):
            for t in range(cu[b], cu[b + 1]):
                at = start[b] + t - cu[b]
                page = int(s["bt"][b, at // PAGE]) if t == cu[b] or at % PAGE == 0 else page
                data[0, page, 0, :, at % PAGE] = k[t]
                data[0, page, 1, :, at % PAGE] = s["v"][t].double()
        return q, data
    cu, ctx, bt = s["cu"].tolist(), s["ctx"].tolist(), s["bt"].tolist()
    words = s["mask"][:, 0].tolist()
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    G = case["hq"] // case["hkv"]
    for b, c in enumerate(ctx):
        n = cu[b + 1] - cu[b]
        L = c + n
        ids = bt[b][:-(-L // PAGE)]
        raw = s["data"][0, ids]
        if case["kv"] == "fp8_e4m3":
            raw = raw.view(torch.float8_e4m3fn).double() * s["scales"][0, ids].double()[..., None, None]
        elif case["kv"] == "int8":
            raw = raw.double() * s["scales"][0, ids].double()[..., None]
        raw = raw.double()
        sees = torch.ones(n, L, dtype=torch.bool)
        for i in range(n):
            for j in range(n):
                sees[i, c + j] = bool((words[cu[b] + i] >> j) & 1)
        sees = sees.to(raw.device).repeat_interleave(G, 0)
        for h in range(case["hkv"]):
            K = raw[:, 0, h].reshape(-1, DIM)[:L]
            Vh = raw[:, 1, h].reshape(-1, DIM)[:L]
            q = s["q"][cu[b]:cu[b + 1], h * G:(h + 1) * G].double().reshape(n * G, DIM)
            z = (q @ K.T * s["scale"]).masked_fill(~sees, -math.inf)
            out[cu[b]:cu[b + 1], h * G:(h + 1) * G] = (torch.softmax(z, -1) @ Vh).view(n, G, DIM)
    return out
